// The paged KV cache's write and read.
//
// paged_rope_kv: token n of qkv [N, (H + 2 Hkv) D] is rotated as rope_kv does it (interleaved pairs, each product and
// the difference rounded separately in fp32, then rounded to the model's type), q goes to q_out, k and v to slot
// slots[n] = page * page_size + offset of the pages. With an 8-bit cache each vector x (one token of one kv head,
// after the rounding to the model's type) is held as e4m3 codes of x * 2^-e and the byte e + 127:
//   e = the smallest integer with max|x| <= 448 * 2^e, held to [-40, 40].
// A power of two loses nothing over an arbitrary scale in a floating-point code (e4m3 keeps its 4 significant bits
// whatever the exponent), is exact to apply and to undo, and takes one byte. The range keeps every product of a scale
// with a softmax weight inside fp32; finite values past 448 * 2^40, infinities and NaN are held as NaN and do not
// count for the scale. paged_kv_read gives the values code * 2^e (exact in fp32, rounded to the output's type).
//
// Both move each byte once and compute next to nothing: HBM for prompts, latency for single tokens.

#include <math.h>

#include <cuda_fp8.h>

#include <type_traits>

#include "attention.cuh"
#include "common.cuh"
#include "paged.cuh"
#include "rope_kv.cuh"

namespace omni {
namespace {

// The scale exponent of a vector whose largest finite magnitude has these bits.
OMNI_DEV int scale_exponent(uint32_t amax_bits) {
  const int e = (int)(amax_bits >> 23) - 135 + ((amax_bits & 0x7fffffu) > 0x600000u ? 1 : 0);
  return e < -40 ? -40 : (e > 40 ? 40 : e);
}

OMNI_DEV float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// Four e4m3 codes of x * inv.
OMNI_DEV uint32_t codes4(const float* x, float inv) {
  float y[4];
  bool bad[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    y[i] = x[i] * inv;
    bad[i] = !(fabsf(y[i]) <= 448.f);
  }
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(y[0], y[1]), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(y[2], y[3]), __NV_SATFINITE, __NV_E4M3);
  uint32_t r = lo | (hi << 16);
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (bad[i]) r |= 0x7fu << (8 * i);
  return r;
}

// Two e4m3 codes as floats.
OMNI_DEV float2 values2(uint32_t codes) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(codes & 0xffffu), __NV_E4M3);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

constexpr int kRopeThreads = 256;

// One CTA: the vectors [item0, item0 + per) of one token (heads of q, then k, then v). A vector is taken by L lanes,
// 16 bytes per lane and step, so a thread keeps the same dims for all its vectors and loads their cos / sin once.
// IL vectors per thread are in flight together.
// (Prompts of 32 + 2 x 8 heads of 128, 291 MB: 61 us with four vectors per thread of which the fourth had nothing to do,
// 53 us, 5470 GB/s, with three and registers for six CTAs per SM; a CTA that walks tokens with the next one's loads in
// flight needs twice the registers: 93 us.)
template <typename T, int D, bool FP8, int IL>
__global__ void __launch_bounds__(kRopeThreads, D * sizeof(T) <= 512 ? (IL == 4 ? 5 : 6) : 2) paged_rope_kernel(const PagedRopeArgs a, int per) {
  constexpr int kVec = Elem<T>::kVec;
  constexpr int VPV = D / kVec;            // 16-byte words per vector
  constexpr int L = VPV < 32 ? VPV : 32;   // lanes per vector
  constexpr int NV = VPV / L;              // words per lane
  constexpr int TEAMS = kRopeThreads / L;
  grid_launch_dependents();
  grid_dependency_wait();
  const int64_t n = blockIdx.x;
  const int kvh = a.c.kv_heads;
  const int items = a.heads + 2 * kvh;
  const int i0 = blockIdx.y * per, i1 = min(items, i0 + per);
  const int lane = threadIdx.x % L, team = threadIdx.x / L;
  const T* src = reinterpret_cast<const T*>(a.qkv) + n * a.qkv_stride;
  uint4 u[IL][NV];
  auto load = [&](int base) {
#pragma unroll
    for (int j = 0; j < IL; ++j) {
      const int it = base + j * TEAMS + team;
#pragma unroll
      for (int v = 0; v < NV; ++v)
        u[j][v] = it < i1 ? __ldg(reinterpret_cast<const uint4*>(src + (int64_t)it * D) + v * L + lane)
                          : make_uint4(0u, 0u, 0u, 0u);
    }
  };
  load(i0);  // before the position is waited for
  const int64_t p = a.pos[n];
  const int64_t slot = a.slots[n];
  const bool pos_ok = p >= 0 && p < a.cs_positions;
  const bool slot_ok = slot >= 0 && slot < a.c.pages * a.c.page;
  if (threadIdx.x == 0 && (!pos_ok || slot >= a.c.pages * a.c.page)) raise_status(a.status, kStatusIndex);
  const int64_t pg = slot_ok ? slot / a.c.page : 0;
  const int off = slot_ok ? (int)(slot - pg * a.c.page) : 0;

  float cs[NV][kVec];
#pragma unroll
  for (int v = 0; v < NV; ++v)
#pragma unroll
    for (int i = 0; i < kVec / 4; ++i) {
      const float4 f = pos_ok ? __ldg(reinterpret_cast<const float4*>(a.cs + p * D + (v * L + lane) * kVec) + i)
                              : make_float4(0.f, 0.f, 0.f, 0.f);
      cs[v][4 * i] = f.x;
      cs[v][4 * i + 1] = f.y;
      cs[v][4 * i + 2] = f.z;
      cs[v][4 * i + 3] = f.w;
    }
  // Every team of a warp takes the same number of rounds (the scale's shuffles need the whole warp).
  for (int base = i0; base < i1; base += TEAMS * IL) {
    if (base > i0) load(base);
#pragma unroll
    for (int j = 0; j < IL; ++j) {
      const int it = base + j * TEAMS + team;
      const bool turn = it < a.heads + kvh;
      const bool live = it < i1;
      float y[NV][kVec];
      uint4 r[NV];
      if (turn) {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
          float x[kVec];
          Elem<T>::unpack(u[j][v], x);
#pragma unroll
          for (int i = 0; i < kVec / 2; ++i) {
            const float re = x[2 * i], im = x[2 * i + 1], co = cs[v][2 * i], si = cs[v][2 * i + 1];
            y[v][2 * i] = __fsub_rn(__fmul_rn(re, co), __fmul_rn(im, si));
            y[v][2 * i + 1] = __fadd_rn(__fmul_rn(re, si), __fmul_rn(im, co));
          }
          r[v] = pos_ok ? Pack<T>::pack(y[v]) : make_uint4(0u, 0u, 0u, 0u);
        }
      } else {
#pragma unroll
        for (int v = 0; v < NV; ++v) r[v] = u[j][v];
      }
      if (live && it < a.heads) {
#pragma unroll
        for (int v = 0; v < NV; ++v)
          reinterpret_cast<uint4*>(reinterpret_cast<T*>(a.q_out) + (n * a.heads + it) * D)[v * L + lane] = r[v];
      }
      const bool is_k = it < a.heads + kvh;
      const int h = it - a.heads - (is_k ? 0 : kvh);
      const bool write = live && it >= a.heads && slot_ok && (pos_ok || !is_k);
      const int64_t dst = pg * a.c.s_page + (int64_t)h * a.c.s_head + (int64_t)off * a.c.s_pos;
      if constexpr (FP8) {
        if (__all_sync(0xffffffffu, it < a.heads)) continue;  // a warp of query heads (the same for all its lanes)
        uint32_t amax = 0u;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
          Elem<T>::unpack(r[v], y[v]);  // the vector as the model's type holds it
#pragma unroll
          for (int i = 0; i < kVec; ++i) {
            const uint32_t b = __float_as_uint(y[v][i]) & 0x7fffffffu;
            amax = max(amax, b < 0x7f800000u ? b : 0u);
          }
        }
#pragma unroll
        for (int o = L / 2; o > 0; o >>= 1) amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        if (write) {
          const int e = scale_exponent(amax);
          const float inv = pow2(-e);
          uint8_t* row = reinterpret_cast<uint8_t*>(is_k ? a.c.k : a.c.v) + dst;
#pragma unroll
          for (int v = 0; v < NV; ++v) {
            if constexpr (kVec == 8)
              reinterpret_cast<uint2*>(row)[v * L + lane] = make_uint2(codes4(y[v], inv), codes4(y[v] + 4, inv));
            else
              reinterpret_cast<uint32_t*>(row)[v * L + lane] = codes4(y[v], inv);
          }
          if (lane == 0) (is_k ? a.c.k_scale : a.c.v_scale)[(pg * kvh + h) * a.c.page + off] = (uint8_t)(e + 127);
        }
      } else if (write) {
        T* row = reinterpret_cast<T*>(is_k ? a.c.k : a.c.v) + dst;
#pragma unroll
        for (int v = 0; v < NV; ++v) reinterpret_cast<uint4*>(row)[v * L + lane] = r[v];
      }
    }
  }
}

constexpr int kReadThreads = 256;

// One CTA: consecutive output tokens of one head (a page's positions of a head lie together), R rounds of TP tokens with
// 16 bytes of the output per thread and round. Threads find the tokens' places first (the sequence by bisection in the
// offsets, the page in its table row); then all rounds' loads are in flight together, and every store of a warp covers
// whole lines: 195 MB of an fp8 context 34 us (5741 GB/s); 44 us with 16-byte loads (two half-line stores each), token-major.
template <typename T, int D, bool FP8, int R>
__global__ void __launch_bounds__(kReadThreads) paged_read_kernel(const PagedReadArgs a) {
  constexpr int kOut = 16 / sizeof(T);       // elements per thread and round
  constexpr int W = D / kOut;                // threads per vector
  constexpr int TP = kReadThreads / W;       // tokens per round
  constexpr int TB = TP * R;
  grid_launch_dependents();
  grid_dependency_wait();
  __shared__ int64_t s_page[TB];
  __shared__ int s_off[TB];
  const int kvh = a.c.kv_heads;
  const int64_t t0 = (int64_t)(blockIdx.x / (unsigned)kvh) * TB;
  const int h = blockIdx.x % (unsigned)kvh;
  for (int i = threadIdx.x; i < TB; i += kReadThreads) {
    const int64_t tok = t0 + i;
    int64_t page = -1;
    int off = 0;
    if (tok < a.tokens && tok >= a.offsets[0] && tok < a.offsets[a.rows]) {
      int lo = 0, hi = a.rows - 1;  // the last row that starts at or before the token
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (a.offsets[mid] <= tok) lo = mid;
        else hi = mid - 1;
      }
      const int64_t j = tok - a.offsets[lo];
      const int64_t pi = j / a.c.page;
      off = (int)(j - pi * a.c.page);
      const int64_t id = j >= 0 && pi < a.table_width ? a.table[lo * a.table_stride + pi] : -1;
      if (id >= 0 && id < a.c.pages) page = id;
      else if (h == 0) raise_status(a.status, kStatusIndex);
    }
    s_page[i] = page;
    s_off[i] = off;
  }
  __syncthreads();
  const int c = threadIdx.x % W;
  using In = std::conditional_t<!FP8, uint4, std::conditional_t<kOut == 8, uint2, uint32_t>>;
  In ku[R], vu[R];
  float ks[R], vs[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int i = r * TP + threadIdx.x / W;
    const int64_t page = s_page[i];
    ku[r] = In{};
    vu[r] = In{};
    ks[r] = vs[r] = 0.f;
    if (page >= 0) {
      const int64_t at = page * a.c.s_page + (int64_t)h * a.c.s_head + (int64_t)s_off[i] * a.c.s_pos + c * kOut;
      constexpr int es = FP8 ? 1 : sizeof(T);
      ku[r] = __ldcs(reinterpret_cast<const In*>(reinterpret_cast<const char*>(a.c.k) + at * es));
      vu[r] = __ldcs(reinterpret_cast<const In*>(reinterpret_cast<const char*>(a.c.v) + at * es));
      if (FP8) {
        const int64_t si = (page * kvh + h) * a.c.page + s_off[i];
        ks[r] = __uint_as_float((uint32_t)__ldg(a.c.k_scale + si) << 23);
        vs[r] = __uint_as_float((uint32_t)__ldg(a.c.v_scale + si) << 23);
      }
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int64_t tok = t0 + r * TP + threadIdx.x / W;
    if (tok >= a.tokens) break;
    const int64_t dst = (tok * kvh + h) * D + c * kOut;
    uint4* ko = reinterpret_cast<uint4*>(reinterpret_cast<T*>(a.k_out) + dst);
    uint4* vo = reinterpret_cast<uint4*>(reinterpret_cast<T*>(a.v_out) + dst);
    if constexpr (FP8) {
      uint32_t kw[2], vw[2];
      if constexpr (kOut == 8) {
        kw[0] = ku[r].x, kw[1] = ku[r].y, vw[0] = vu[r].x, vw[1] = vu[r].y;
      } else {
        kw[0] = ku[r], vw[0] = vu[r];
      }
      float kf[kOut], vf[kOut];
#pragma unroll
      for (int i = 0; i < kOut / 2; ++i) {
        const float2 kk = values2(kw[i >> 1] >> (16 * (i & 1))), vv = values2(vw[i >> 1] >> (16 * (i & 1)));
        kf[2 * i] = kk.x * ks[r];
        kf[2 * i + 1] = kk.y * ks[r];
        vf[2 * i] = vv.x * vs[r];
        vf[2 * i + 1] = vv.y * vs[r];
      }
      __stcs(ko, Pack<T>::pack(kf));
      __stcs(vo, Pack<T>::pack(vf));
    } else {
      __stcs(ko, ku[r]);
      __stcs(vo, vu[r]);
    }
  }
}

template <typename T, int D, bool FP8>
cudaError_t rope_launch(const PagedRopeArgs& a, cudaStream_t s) {
  constexpr int VPV = D / Elem<T>::kVec;
  constexpr int TEAMS = kRopeThreads / (VPV < 32 ? VPV : 32);
  const int items = a.heads + 2 * a.c.kv_heads;
  // A token's vectors go to several CTAs while the tokens alone leave SMs idle (a decode step).
  const int want = 2 * device_sm_count();
  int parts = (want + a.n - 1) / a.n;
  const int most = (items + TEAMS - 1) / TEAMS;
  parts = parts < 1 ? 1 : (parts > most ? most : parts);
  const int per = (items + parts - 1) / parts;
  const dim3 grid((unsigned)a.n, (unsigned)((items + per - 1) / per));
  // Vectors per thread in flight: of 4, 3 and 2, the one that leaves the fewest without work.
  const int rounds = (per + TEAMS - 1) / TEAMS;
  int il = 1;
  if (rounds > 1) {
    int idle = 1 << 30;
    for (int k = 4; k >= 2; --k) {
      const int w = (rounds + k - 1) / k * k - rounds;
      if (w < idle) {
        idle = w;
        il = k;
      }
    }
  }
  switch (il) {
    case 1: return launch_dependent(paged_rope_kernel<T, D, FP8, 1>, grid, dim3(kRopeThreads), 0, s, a, per);
    case 2: return launch_dependent(paged_rope_kernel<T, D, FP8, 2>, grid, dim3(kRopeThreads), 0, s, a, per);
    case 3: return launch_dependent(paged_rope_kernel<T, D, FP8, 3>, grid, dim3(kRopeThreads), 0, s, a, per);
    default: return launch_dependent(paged_rope_kernel<T, D, FP8, 4>, grid, dim3(kRopeThreads), 0, s, a, per);
  }
}

template <typename T, int D, bool FP8>
cudaError_t read_launch(const PagedReadArgs& a, cudaStream_t s) {
  constexpr int TP = kReadThreads / (D / (16 / (int)sizeof(T)));
  // Four rounds per CTA, one where four would leave SMs without work.
  const int64_t four = (a.tokens + 4 * TP - 1) / (4 * TP) * a.c.kv_heads;
  const int64_t one = (a.tokens + TP - 1) / TP * a.c.kv_heads;
  if (four >= 2 * device_sm_count())
    return launch_dependent(paged_read_kernel<T, D, FP8, 4>, dim3((unsigned)four), dim3(kReadThreads), 0, s, a);
  return launch_dependent(paged_read_kernel<T, D, FP8, 1>, dim3((unsigned)one), dim3(kReadThreads), 0, s, a);
}

#define OMNI_DIM_SWITCH(DIM, CALL)      \
  switch (DIM) {                        \
    case 16: return CALL(16);           \
    case 32: return CALL(32);           \
    case 64: return CALL(64);           \
    case 128: return CALL(128);         \
    case 256: return CALL(256);         \
    case 512: return CALL(512);         \
    default: return cudaErrorInvalidValue; \
  }

template <typename T, bool FP8>
cudaError_t rope_dim(const PagedRopeArgs& a, cudaStream_t s) {
#define CALL(D) rope_launch<T, D, FP8>(a, s)
  OMNI_DIM_SWITCH(a.c.dim, CALL)
#undef CALL
}

template <typename T, bool FP8>
cudaError_t read_dim(const PagedReadArgs& a, cudaStream_t s) {
#define CALL(D) read_launch<T, D, FP8>(a, s)
  OMNI_DIM_SWITCH(a.c.dim, CALL)
#undef CALL
}

}  // namespace

cudaError_t launch_paged_rope_kv(int dtype, const PagedRopeArgs& a, cudaStream_t stream) {
  if (a.n <= 0) return cudaSuccess;
  if (dtype == kBF16) return a.c.type == kFp8 ? rope_dim<__nv_bfloat16, true>(a, stream) : rope_dim<__nv_bfloat16, false>(a, stream);
  return a.c.type == kFp8 ? rope_dim<float, true>(a, stream) : rope_dim<float, false>(a, stream);
}

cudaError_t launch_paged_kv_read(int dtype, const PagedReadArgs& a, cudaStream_t stream) {
  if (a.tokens <= 0) return cudaSuccess;
  if (dtype == kBF16) return a.c.type == kFp8 ? read_dim<__nv_bfloat16, true>(a, stream) : read_dim<__nv_bfloat16, false>(a, stream);
  return a.c.type == kFp8 ? read_dim<float, true>(a, stream) : read_dim<float, false>(a, stream);
}

}  // namespace omni
