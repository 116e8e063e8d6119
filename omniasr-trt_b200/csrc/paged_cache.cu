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
// count for the scale. paged_kv_read gives the values code * 2^e (exact in fp32, rounded to the output's type). With a 4-bit cache a
// group of 32 dims is held as 4-bit codes and a bf16 scale (int4.cuh); read back, s (c - 8), exact in fp32 too.
//
// Both move each byte once and compute next to nothing: HBM for prompts, latency for single tokens.

#include <math.h>

#include <cuda_fp8.h>

#include <type_traits>

#include "paged_rope.cuh"

namespace omni {
namespace {

// Two e4m3 codes as floats.
OMNI_DEV float2 values2(uint32_t codes) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(codes & 0xffffu), __NV_E4M3);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

constexpr int kReadThreads = 256;

// One CTA: consecutive output tokens of one head (a page's positions of a head lie together), R rounds of TP tokens with
// 16 bytes of the output per thread and round. Threads find the tokens' places first (the sequence by bisection in the
// offsets, the page in its table row); then all rounds' loads are in flight together, and every store of a warp covers
// whole lines: 195 MB of an fp8 context 34 us (5741 GB/s); 44 us with 16-byte loads (two half-line stores each), token-major.
template <typename T, int D, int KIND, int R>
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
  using In = std::conditional_t<KIND == kOwnType, uint4, std::conditional_t<KIND == kFp8 && kOut == 8, uint2, uint32_t>>;
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
      const int64_t row = page * a.c.s_page + (int64_t)h * a.c.s_head + (int64_t)s_off[i] * a.c.s_pos, at = row + c * kOut;
      constexpr int es = KIND == kFp8 ? 1 : sizeof(T);
      const int64_t si = (page * kvh + h) * a.c.page + s_off[i];
      if constexpr (KIND == kInt4) {
        const uint16_t* kr = reinterpret_cast<const uint16_t*>(reinterpret_cast<const char*>(a.c.k) + row);
        const uint16_t* vr = reinterpret_cast<const uint16_t*>(reinterpret_cast<const char*>(a.c.v) + row);
#pragma unroll
        for (int q = 0; q < kOut / 4; ++q) {
          ku[r] |= (uint32_t)__ldcs(kr + quad_at<D, true>(c * (kOut / 4) + q)) << (16 * q);
          vu[r] |= (uint32_t)__ldcs(vr + quad_at<D, false>(c * (kOut / 4) + q)) << (16 * q);
        }
        const int64_t g = si * (D / 32) + c * kOut / 32;
        ks[r] = bf16_value(reinterpret_cast<const uint16_t*>(a.c.k_scale)[g]);
        vs[r] = bf16_value(reinterpret_cast<const uint16_t*>(a.c.v_scale)[g]);
      } else {
        ku[r] = __ldcs(reinterpret_cast<const In*>(reinterpret_cast<const char*>(a.c.k) + at * es));
        vu[r] = __ldcs(reinterpret_cast<const In*>(reinterpret_cast<const char*>(a.c.v) + at * es));
      }
      if constexpr (KIND == kFp8) {
        ks[r] = __uint_as_float((uint32_t)a.c.k_scale[si] << 23);
        vs[r] = __uint_as_float((uint32_t)a.c.v_scale[si] << 23);
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
    if constexpr (KIND == kInt4 && kOut == 8) {
      const uint32_t k2 = __float_as_uint(ks[r]) >> 16, v2 = __float_as_uint(vs[r]) >> 16;
      const uint2 k0 = int4_values_bf16(ku[r] & 0xffffu, k2 | k2 << 16), k1 = int4_values_bf16(ku[r] >> 16, k2 | k2 << 16);
      const uint2 v0 = int4_values_bf16(vu[r] & 0xffffu, v2 | v2 << 16), v1 = int4_values_bf16(vu[r] >> 16, v2 | v2 << 16);
      __stcs(ko, make_uint4(k0.x, k0.y, k1.x, k1.y));
      __stcs(vo, make_uint4(v0.x, v0.y, v1.x, v1.y));
    } else if constexpr (KIND == kInt4) {
      float kf[kOut], vf[kOut];
#pragma unroll
      for (int q = 0; q < kOut / 4; ++q) {
        int4_values(ku[r] >> (16 * q), ks[r], kf + 4 * q);
        int4_values(vu[r] >> (16 * q), vs[r], vf + 4 * q);
      }
      __stcs(ko, Pack<T>::pack(kf));
      __stcs(vo, Pack<T>::pack(vf));
    } else if constexpr (KIND == kFp8) {
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

template <typename T, int D, int KIND>
cudaError_t read_launch(const PagedReadArgs& a, cudaStream_t s) {
  constexpr int TP = kReadThreads / (D / (16 / (int)sizeof(T)));
  // Four rounds per CTA, one where four would leave SMs without work.
  const int64_t four = (a.tokens + 4 * TP - 1) / (4 * TP) * a.c.kv_heads;
  const int64_t one = (a.tokens + TP - 1) / TP * a.c.kv_heads;
  if (four >= 2 * device_sm_count())
    return launch_dependent(paged_read_kernel<T, D, KIND, 4>, dim3((unsigned)four), dim3(kReadThreads), 0, s, a);
  return launch_dependent(paged_read_kernel<T, D, KIND, 1>, dim3((unsigned)one), dim3(kReadThreads), 0, s, a);
}

template <typename T, int KIND>
cudaError_t read_dim(const PagedReadArgs& a, cudaStream_t s) {
#define CALL(D) read_launch<T, D, KIND == kInt4 && D < 32 ? -1 : KIND>(a, s)
  if (KIND == kInt4 && a.c.dim < 32) return cudaErrorInvalidValue;
  OMNI_DIM_SWITCH(a.c.dim, CALL)
#undef CALL
}

template <typename T>
cudaError_t read_kind(const PagedReadArgs& a, cudaStream_t s) {
  if (a.c.type == kFp8) return read_dim<T, kFp8>(a, s);
  if (a.c.type == kInt4) return read_dim<T, kInt4>(a, s);
  return read_dim<T, kOwnType>(a, s);
}

}  // namespace

cudaError_t launch_paged_rope_kv(int dtype, const PagedRopeArgs& a, cudaStream_t stream) {
  if (a.n <= 0) return cudaSuccess;
  return dtype == kBF16 ? rope_kind<__nv_bfloat16, false>(a, stream) : rope_kind<float, false>(a, stream);
}

cudaError_t launch_paged_kv_read(int dtype, const PagedReadArgs& a, cudaStream_t stream) {
  if (a.tokens <= 0) return cudaSuccess;
  return dtype == kBF16 ? read_kind<__nv_bfloat16>(a, stream) : read_kind<float>(a, stream);
}

}  // namespace omni
