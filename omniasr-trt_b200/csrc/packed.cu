// Causal attention of packed sequences with grouped heads: entry, and the CUDA-core kernel for what the tensor-core
// kernels (prefill.cu, prefill_wide.cu) do not take (fp32, head dims under 64, scales that are not positive).
//
// Sequence s has queries q_offsets[s] .. q_offsets[s+1] - 1 and keys k_offsets[s] .. k_offsets[s+1] - 1; its last query
// sees its last key (a chunk of a prompt attends to the keys before it), so query i sees i + 1 + lk - lq keys, none
// where that is not positive. q [Tq, H, D], k and v [Tk, Hkv, D], head h reads kv head h / (H / Hkv).
//
// One CTA: BM queries of one head; K and V tiles of BN keys go through shared memory as fp32; S = Q K^T and O += P V
// in registers (16 lanes across keys and head dims: thread (y, x) holds rows y + YR i, keys x + 16 j and groups of four dims,
// so a row's softmax statistics are a shuffle over half a warp). Bound by shared-memory reads and FMA; fp32 throughout, as an
// fp32 model needs. BM is 64 (32 for head dims of 256 and more, whose tiles fill the shared memory), or 16, of 128 threads,
// while larger tiles leave SMs idle: three prompts of 17 to 131 tokens, 8 heads of 64, take 11 us; 22
// with 256 threads of one row each (a value read from shared memory then serves one product, not two) and no copy of the
// next tile in flight.

#include <math.h>

#include <algorithm>
#include <type_traits>

#include "attention.cuh"
#include "common.cuh"
#include "paged.cuh"

namespace omni {
namespace packed {

template <typename T, int D, int BM_>
struct Shape {
  static constexpr int BM = BM_;
  static constexpr int THREADS = BM == 16 ? 128 : 256, YR = THREADS / 16;
  static constexpr int BN = D <= 128 ? 64 : 32;
  static constexpr int VW = D >= 64 ? 4 : D / 16;  // consecutive head dims of O per thread
  static constexpr int LD = D + 4;  // row stride in shared memory (floats): 16-byte aligned, rows on different banks
  static constexpr int LP = BN + 4;
  static constexpr int KV = 2 * BN * LD;  // floats of a K and a V tile
  // fp32 tiles are copied asynchronously, for small tiles (which wait for nothing else) the next one during this one's work.
  static constexpr bool ASYNC = sizeof(T) == 4;
  static constexpr int STAGES = ASYNC && BM == 16 && (BM * (LD + LP) + 2 * KV) * 4 <= 232448 - 1024 ? 2 : 1;
  static constexpr int BYTES = (BM * (LD + LP) + STAGES * KV) * 4;
};

OMNI_DEV bool offsets_ok(const PackedArgs& a, int s) {
  const int64_t qa = a.q_offsets[s], qb = a.q_offsets[s + 1], ka = a.k_offsets[s], kb = a.k_offsets[s + 1];
  return qa >= 0 && qb >= qa && qb <= a.q_tokens && ka >= 0 && kb >= ka && kb <= a.k_tokens;
}

// Tile `slot` of the packed queries -> sequence and first query: the sequences' tile counts, summed 32 at a time by one
// warp. Returns the sequence, or -1 past the last tile.
OMNI_DEV int find_tile(const int64_t* offsets, int seqs, int bm, int slot, int lane, int* tile) {
  int before = 0;
  for (int s0 = 0; s0 < seqs; s0 += 32) {
    const int s = s0 + lane;
    const int64_t n = s < seqs ? offsets[s + 1] - offsets[s] : 0;
    const int mine = n > 0 ? (int)((n + bm - 1) / bm) : 0;
    int incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += y;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, slot < before + incl);
    if (hit) {
      const int w = __ffs(hit) - 1;
      *tile = slot - before - __shfl_sync(0xffffffffu, incl - mine, w);
      return s0 + w;
    }
    before += __shfl_sync(0xffffffffu, incl, 31);
  }
  return -1;
}

template <typename T>
OMNI_DEV void load4(const T* p, float* f);
template <>
OMNI_DEV void load4<float>(const float* p, float* f) {
  const float4 v = __ldg(reinterpret_cast<const float4*>(p));
  f[0] = v.x, f[1] = v.y, f[2] = v.z, f[3] = v.w;
}
template <>
OMNI_DEV void load4<__nv_bfloat16>(const __nv_bfloat16* p, float* f) {
  const uint2 v = __ldg(reinterpret_cast<const uint2*>(p));
  f[0] = __uint_as_float(v.x << 16), f[1] = __uint_as_float(v.x & 0xffff0000u);
  f[2] = __uint_as_float(v.y << 16), f[3] = __uint_as_float(v.y & 0xffff0000u);
}

// ROWS rows of 4-element groups from global (row stride st) into shared memory, all loads in flight together; rows at or
// past `valid` are zeros.
template <typename T, int D, int LD, int ROWS, int kThreads>
OMNI_DEV void load_tile(float* dst, const T* src, int64_t st, int valid) {
  constexpr int TOTAL = ROWS * (D / 4), N = (TOTAL + kThreads - 1) / kThreads, B = N < 8 ? N : 8;
  if constexpr (sizeof(T) == 4) {  // asynchronously: the caller waits (nothing is read for the rows of zeros)
#pragma unroll 4
    for (int i = threadIdx.x; i < TOTAL; i += kThreads) {
      const int r = i / (D / 4), c = (i - r * (D / 4)) * 4;
      const int size = r < valid ? 16 : 0;
      const T* from = size ? src + (int64_t)r * st + c : src;
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_addr(dst + r * LD + c)), "l"(from), "r"(size) : "memory");
    }
    return;
  }
#pragma unroll 1
  for (int i0 = 0; i0 < N; i0 += B) {
    float f[B][4];
#pragma unroll
    for (int b = 0; b < B; ++b) {
      const int i = (i0 + b) * kThreads + threadIdx.x;
      const int r = i / (D / 4), c = (i - r * (D / 4)) * 4;
      f[b][0] = f[b][1] = f[b][2] = f[b][3] = 0.f;
      if (r < valid && i < TOTAL) load4(src + (int64_t)r * st + c, f[b]);
    }
#pragma unroll
    for (int b = 0; b < B; ++b) {
      const int i = (i0 + b) * kThreads + threadIdx.x;
      const int r = i / (D / 4), c = (i - r * (D / 4)) * 4;
      if (i < TOTAL) *reinterpret_cast<float4*>(dst + r * LD + c) = make_float4(f[b][0], f[b][1], f[b][2], f[b][3]);
    }
  }
}

// Parts of a query tile's keys for the calls of few tiles over many keys (part z of them: blockIdx.z); each leaves its rows'
// maxima, sums and unnormalised outputs, and join_kernel adds them up in the order of the keys.
struct Parts {
  int n;
  float* ml;  // [row * heads + head][part][2]
  float* o;   // ... [D]
};
constexpr int kMostParts = 32;

// At most this many parts: two CTAs per SM.
int most_parts(int dtype, int64_t q_tokens, int heads, int kv_heads, int dim) {
  if (dtype == kBF16 && dim >= 64 && heads / kv_heads <= 128) return 1;  // the tensor-core kernels' calls
  const int64_t units = heads * ((q_tokens + 15) / 16);
  return (int)std::max<int64_t>(1, std::min<int64_t>(kMostParts, units > 0 ? 2 * device_sm_count() / units : 1));
}

template <typename T, int D, int BM_>
__global__ void __launch_bounds__(Shape<T, D, BM_>::THREADS) packed_kernel(const PackedArgs a, const Parts parts) {
  using S = Shape<T, D, BM_>;
  constexpr int BM = S::BM, BN = S::BN, LD = S::LD, LP = S::LP, VW = S::VW, YR = S::YR;
  constexpr int MR = BM / YR, NR = BN / 16, DR = D / 16, DG = DR / VW;
  extern __shared__ __align__(16) float sm[];
  float* qs = sm;
  float* ps = qs + BM * LD;
  float* ring = ps + BM * LP;  // [stage][K, V]
  __shared__ int s_seq, s_tile;
  grid_launch_dependents();
  grid_dependency_wait();
  if (blockIdx.x == gridDim.x - 1 && blockIdx.y == 0 && blockIdx.z == 0) {  // one CTA looks all offsets over
    for (int s = threadIdx.x; s < a.seqs; s += S::THREADS)
      if (!offsets_ok(a, s)) raise_status(a.status, kStatusIndex);
  }
  if (threadIdx.x < 32) {
    int tile = 0;
    const int seq = find_tile(a.q_offsets, a.seqs, BM, blockIdx.x, threadIdx.x, &tile);
    if (threadIdx.x == 0) {
      s_seq = seq;
      s_tile = tile;
    }
  }
  __syncthreads();
  if (s_seq < 0) return;
  const int h = blockIdx.y, kvh = h / (a.heads / a.kv_heads);
  const int64_t qa = a.q_offsets[s_seq], qb = a.q_offsets[s_seq + 1];
  const int64_t ka = a.k_offsets[s_seq], kb = a.k_offsets[s_seq + 1];
  if (!offsets_ok(a, s_seq)) return;
  const int64_t q0 = qa + (int64_t)s_tile * BM;
  const int rows = (int)min((int64_t)BM, qb - q0);
  // Row r of the tile sees keys [0, lim0 + r) of the sequence.
  const int64_t lim0 = (q0 - qa) + 1 + (kb - ka) - (qb - qa);
  int64_t keys = max((int64_t)0, lim0 + rows - 1), first = 0;
  if (BM == 16 && parts.n > 1) {
    const int64_t each = ((keys + BN - 1) / BN + parts.n - 1) / parts.n * BN;
    first = min(keys, blockIdx.z * each);
    keys = min(keys, first + each);
  }
  const int x = threadIdx.x & 15, y = threadIdx.x >> 4;
  load_tile<T, D, LD, BM, S::THREADS>(qs, reinterpret_cast<const T*>(a.q) + q0 * a.q_st + (int64_t)h * a.q_sh, a.q_st, rows);
  const T* kg = reinterpret_cast<const T*>(a.k) + ka * a.k_st + (int64_t)kvh * a.k_sh;
  const T* vg = reinterpret_cast<const T*>(a.v) + ka * a.v_st + (int64_t)kvh * a.v_sh;
  const float qscale = a.scale * kLog2e;
  auto fetch = [&](float* to, int64_t j0) {  // the K and V tile of keys j0 ..
    const int valid = (int)min((int64_t)BN, keys - j0);
    load_tile<T, D, LD, BN, S::THREADS>(to, kg + j0 * a.k_st, a.k_st, valid);
    load_tile<T, D, LD, BN, S::THREADS>(to + BN * LD, vg + j0 * a.v_st, a.v_st, valid);
  };
  float m[MR], l[MR], o[MR][DR];
#pragma unroll
  for (int i = 0; i < MR; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.f;
#pragma unroll
    for (int d = 0; d < DR; ++d) o[i][d] = 0.f;
  }
  for (int64_t j0 = first; j0 < keys; j0 += BN) {
    const int valid = (int)min((int64_t)BN, keys - j0);
    float* ks = ring + (S::STAGES == 2 && (j0 / BN & 1) ? S::KV : 0);
    const float* vs = ks + BN * LD;
    __syncthreads();  // the tile before is used up
    if (S::STAGES == 1 || j0 == first) {
      fetch(ks, j0);
      if (S::ASYNC) asm volatile("cp.async.commit_group;" ::: "memory");
    }
    if (S::STAGES == 2) {
      if (j0 + BN < keys) fetch(ring + (j0 / BN & 1 ? 0 : S::KV), j0 + BN);
      asm volatile("cp.async.commit_group;" ::: "memory");
    }
    if (S::ASYNC) asm volatile("cp.async.wait_group %0;" ::"n"(S::STAGES - 1) : "memory");
    __syncthreads();
    float s[MR][NR];
#pragma unroll
    for (int i = 0; i < MR; ++i)
#pragma unroll
      for (int j = 0; j < NR; ++j) s[i][j] = 0.f;
#pragma unroll 4
    for (int d = 0; d < D; d += 4) {
      float4 qv[MR], kv[NR];
#pragma unroll
      for (int i = 0; i < MR; ++i) qv[i] = *reinterpret_cast<const float4*>(qs + (y + YR * i) * LD + d);
#pragma unroll
      for (int j = 0; j < NR; ++j) kv[j] = *reinterpret_cast<const float4*>(ks + (x + 16 * j) * LD + d);
#pragma unroll
      for (int i = 0; i < MR; ++i)
#pragma unroll
        for (int j = 0; j < NR; ++j)
          s[i][j] = fmaf(qv[i].w, kv[j].w, fmaf(qv[i].z, kv[j].z, fmaf(qv[i].y, kv[j].y, fmaf(qv[i].x, kv[j].x, s[i][j]))));
    }
    const bool edge = j0 + BN > lim0;  // some row does not see all of the tile
#pragma unroll
    for (int i = 0; i < MR; ++i) {
      const int64_t lim = lim0 + y + YR * i - j0;
      float top = -INFINITY;
#pragma unroll
      for (int j = 0; j < NR; ++j) {
        s[i][j] = x + 16 * j < lim ? s[i][j] * qscale : -INFINITY;
        top = fmaxf(top, s[i][j]);
      }
#pragma unroll
      for (int w = 8; w > 0; w >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
      const float mn = fmaxf(m[i], top);
      const float base = mn == -INFINITY ? 0.f : mn;
      const float f = ex2(m[i] - base);
      m[i] = mn;
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < NR; ++j) {
        const float p = ex2(s[i][j] - base);  // a NaN score gives NaN: the row is NaN, as the formula is
        sum += p;
        ps[(y + YR * i) * LP + x + 16 * j] = p;
      }
      l[i] = fmaf(l[i], f, sum);
#pragma unroll
      for (int d = 0; d < DR; ++d) o[i][d] *= f;
    }
    __syncwarp();  // a row's probabilities are written and read by the same half-warp
    // Four keys at a time (rows past the valid ones hold zeros, their probabilities are zeros or hidden).
    auto values = [&](auto masked) {
#pragma unroll 2
      for (int k = 0; k < valid; k += 4) {
        float p[MR][4];
#pragma unroll
        for (int i = 0; i < MR; ++i) {
          const float4 f = *reinterpret_cast<const float4*>(ps + (y + YR * i) * LP + k);
          p[i][0] = f.x, p[i][1] = f.y, p[i][2] = f.z, p[i][3] = f.w;
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) {
#pragma unroll
          for (int d = 0; d < DG; ++d) {
            const float* src = vs + (k + c) * LD + (x + 16 * d) * VW;
            float v[VW];
            if constexpr (VW == 4) {
              const float4 f = *reinterpret_cast<const float4*>(src);
              v[0] = f.x, v[1] = f.y, v[2] = f.z, v[3] = f.w;
            } else if constexpr (VW == 2) {
              const float2 f = *reinterpret_cast<const float2*>(src);
              v[0] = f.x, v[1] = f.y;
            } else {
              v[0] = src[0];
            }
#pragma unroll
            for (int i = 0; i < MR; ++i) {
              // A key past the row's does not enter, whatever its value holds.
              if (!decltype(masked)::value || j0 + k + c < lim0 + y + YR * i) {
#pragma unroll
                for (int e = 0; e < VW; ++e) o[i][d * VW + e] = fmaf(p[i][c], v[e], o[i][d * VW + e]);
              }
            }
          }
        }
      }
    };
    if (edge) values(std::true_type{});
    else values(std::false_type{});
  }
  if (S::ASYNC) asm volatile("cp.async.wait_all;" ::: "memory");  // (a sequence without keys: the queries')
#pragma unroll
  for (int i = 0; i < MR; ++i) {
#pragma unroll
    for (int w = 8; w > 0; w >>= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], w);
    const int r = y + YR * i;
    if (BM == 16 && parts.n > 1) {
      if (r < rows) {
        const int64_t at = ((q0 + r) * a.heads + h) * parts.n + blockIdx.z;
        if (x == 0) reinterpret_cast<float2*>(parts.ml)[at] = make_float2(m[i], l[i]);
#pragma unroll
        for (int d = 0; d < DG; ++d)
#pragma unroll
          for (int e = 0; e < VW; ++e) parts.o[at * D + (x + 16 * d) * VW + e] = o[i][d * VW + e];
      }
      continue;
    }
    if (r < rows) {
      const float inv = l[i] != 0.f ? 1.f / l[i] : (lim0 + r > 0 ? NAN : 0.f);  // (keys that all score -inf: no softmax)
      T* dst = reinterpret_cast<T*>(a.out) + ((q0 + r) * a.heads + h) * D;
#pragma unroll
      for (int d = 0; d < DG; ++d)
#pragma unroll
        for (int e = 0; e < VW; ++e) dst[(x + 16 * d) * VW + e] = Elem<T>::from_float(o[i][d * VW + e] * inv);
    }
  }
}

// One warp per query and head: o = sum 2^(m_p - m) o_p / sum 2^(m_p - m) l_p over its parts. Rows of no sequence (or of one
// whose offsets are bad) have no parts and are not written.
template <typename T>
__global__ void __launch_bounds__(256) join_kernel(const PackedArgs a, const Parts parts) {
  grid_launch_dependents();
  grid_dependency_wait();
  const int lane = threadIdx.x & 31;
  const int64_t at = blockIdx.x * 8ll + (threadIdx.x >> 5), row = at / a.heads;
  if (row >= a.q_tokens) return;
  int64_t lim = -1;  // keys the query sees
  bool mine = false;
  for (int s0 = 0; s0 < a.seqs && !mine; s0 += 32) {
    const int s = s0 + lane;
    bool hit = false;
    if (s < a.seqs) {
      const int64_t qa = a.q_offsets[s], qb = a.q_offsets[s + 1], ka = a.k_offsets[s], kb = a.k_offsets[s + 1];
      hit = qa <= row && row < qb && offsets_ok(a, s);
      if (hit) lim = row - qa + 1 + (kb - ka) - (qb - qa);
    }
    const unsigned who = __ballot_sync(0xffffffffu, hit);
    if (who) {
      mine = true;
      lim = __shfl_sync(0xffffffffu, lim, __ffs(who) - 1);
    }
  }
  if (!mine) return;
  const float2* ml = reinterpret_cast<const float2*>(parts.ml) + at * parts.n;
  const float2 own = lane < parts.n ? ml[lane] : make_float2(-INFINITY, 0.f);  // (at most 32 parts)
  float top = own.x;
#pragma unroll
  for (int w = 16; w > 0; w >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
  const float weight = ex2(own.x - (top == -INFINITY ? 0.f : top));
  float sum = weight * own.y;
#pragma unroll
  for (int w = 16; w > 0; w >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
  const float inv = sum != 0.f ? 1.f / sum : (lim > 0 ? NAN : 0.f);
  for (int d0 = 0; d0 < a.dim; d0 += 32) {
    const int d = d0 + lane;
    float o = 0.f;
    for (int p = 0; p < parts.n; ++p) {
      const float w = __shfl_sync(0xffffffffu, weight, p);
      if (d < a.dim) o = fmaf(w, parts.o[(at * parts.n + p) * a.dim + d], o);
    }
    if (d < a.dim) reinterpret_cast<T*>(a.out)[at * a.dim + d] = Elem<T>::from_float(o * inv);
  }
}

template <typename T, int D, int BM>
cudaError_t launch_t(const PackedArgs& a, const Parts& parts, cudaStream_t s) {
  using S = Shape<T, D, BM>;
  static PerDevice configured;
  if (const cudaError_t e = allow_smem(packed_kernel<T, D, BM>, S::BYTES, configured)) return e;
  // At most this many tiles: a sequence's last tile may be partly filled.
  const int64_t tiles = a.q_tokens / BM + a.seqs;
  const cudaError_t e = launch_dependent(packed_kernel<T, D, BM>, dim3((unsigned)tiles, (unsigned)a.heads, (unsigned)parts.n),
                                         dim3(S::THREADS), (size_t)S::BYTES, s, a, parts);
  if (e != cudaSuccess || parts.n == 1) return e;
  return launch_dependent(join_kernel<T>, dim3((unsigned)((a.q_tokens * a.heads + 7) / 8)), dim3(256), 0, s, a, parts);
}

template <typename T, int D>
cudaError_t launch_bm(const PackedArgs& a, cudaStream_t s) {
  constexpr int BM = D <= 128 ? 64 : 32;
  Parts parts{1, nullptr, nullptr};
  if (a.q_tokens * a.heads >= (int64_t)BM * 2 * device_sm_count()) return launch_t<T, D, BM>(a, parts, s);
  // Parts of 128 keys at least, in the mean: 16 queries of 8 heads of 64 over 1516 keys take 22 us in 11 parts, 64 whole.
  const int dtype = sizeof(T) == 4 ? kF32 : kBF16;
  parts.n = (int)std::max<int64_t>(1, std::min<int64_t>(most_parts(dtype, a.q_tokens, a.heads, a.kv_heads, D), a.k_tokens / a.seqs / 128));
  parts.ml = reinterpret_cast<float*>(reinterpret_cast<char*>(a.counters) + kCounterBytes);
  parts.o = parts.ml + (a.q_tokens * a.heads * parts.n * 2 + 3) / 4 * 4;
  return launch_t<T, D, 16>(a, parts, s);
}

template <typename T>
cudaError_t launch_dim(const PackedArgs& a, cudaStream_t s) {
  switch (a.dim) {
    case 16: return launch_bm<T, 16>(a, s);
    case 32: return launch_bm<T, 32>(a, s);
    case 64: return launch_bm<T, 64>(a, s);
    case 128: return launch_bm<T, 128>(a, s);
    case 256: return launch_bm<T, 256>(a, s);
    case 512: return launch_bm<T, 512>(a, s);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace packed

size_t packed_parts_bytes(int dtype, int64_t q_tokens, int heads, int kv_heads, int dim) {
  const int n = packed::most_parts(dtype, q_tokens, heads, kv_heads, dim);
  return n > 1 ? sizeof(float) * ((size_t)q_tokens * heads * n * (dim + 2) + 4) : 0;
}

cudaError_t launch_packed(int dtype, const PackedArgs& a, cudaStream_t stream) {
  // (The tensor-core kernels take the maximum of a row's products before they scale them.)
  if (dtype == kBF16 && a.dim >= 64 && a.heads / a.kv_heads <= 128 && a.k_tokens > 0 && a.scale > 0.f) {
    const cudaError_t e = a.dim <= 128 ? launch_packed_tc(a, stream) : launch_packed_tc_wide(a, stream);
    if (e != cudaErrorNotSupported) return e;
  }
  return dtype == kBF16 ? packed::launch_dim<__nv_bfloat16>(a, stream) : packed::launch_dim<float>(a, stream);
}

}  // namespace omni
