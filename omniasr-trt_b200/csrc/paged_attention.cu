// Attention of each row's newest tokens over a paged KV cache: entry, and the CUDA-core kernels for what the
// tensor-core pass (paged_attention_tc.cu) does not take (fp32, small head dims, odd page sizes).
//
// Query i < T of row b sees keys [0, lengths[b] + i); key j of the row is offset j % page of page table[b, j / page].
// A unit is (row, kv head, chunk of query columns): its T * G query vectors (G = heads / kv_heads, column c = token
// c / G, head kv * G + c % G) share every key read. Keys are cut into splits; each keeps a running maximum and sum
// (log2 units, fp32) and its unnormalised output, and a second kernel joins the splits:
//   o = sum_s 2^(m_s - m) o_s / sum_s 2^(m_s - m) l_s.
// A team of lanes owns a key at a time, 8 dims per lane and step, so that a key's K and V rows are read as whole
// 32-byte sectors; a key that a column does not see takes no part in it, whatever its row holds.

#include <math.h>

#include <cuda_fp8.h>

#include <algorithm>

#include "attention.cuh"
#include "common.cuh"
#include "paged.cuh"

namespace omni {
namespace paged {

constexpr int kThreads = 128;

template <typename T>
struct Row8;  // eight consecutive elements of a cache row as floats

template <>
struct Row8<__nv_bfloat16> {
  uint4 u;
  OMNI_DEV void load(const void* base, int64_t at) { u = __ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const __nv_bfloat16*>(base) + at)); }
  OMNI_DEV void get(float* f) const { Elem<__nv_bfloat16>::unpack(u, f); }
};
template <>
struct Row8<float> {
  float4 a, b;
  OMNI_DEV void load(const void* base, int64_t at) {
    a = __ldg(reinterpret_cast<const float4*>(reinterpret_cast<const float*>(base) + at));
    b = __ldg(reinterpret_cast<const float4*>(reinterpret_cast<const float*>(base) + at) + 1);
  }
  OMNI_DEV void get(float* f) const {
    f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
  }
};
template <>
struct Row8<__nv_fp8_e4m3> {
  uint2 u;
  OMNI_DEV void load(const void* base, int64_t at) { u = __ldg(reinterpret_cast<const uint2*>(reinterpret_cast<const uint8_t*>(base) + at)); }
  OMNI_DEV void get(float* f) const {
    const uint32_t w[2] = {u.x, u.y};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)((w[i >> 1] >> (16 * (i & 1))) & 0xffffu), __NV_E4M3);
      const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&h));
      f[2 * i] = v.x;
      f[2 * i + 1] = v.y;
    }
  }
};

struct Split {
  int splits, chunks, cols;  // key splits per unit, column chunks per (row, kv head), columns per chunk
  float* part_o;             // [row * T * heads + column's query][split][D]
  float* part_ml;            // ... [split][2]
};

// The result of query vector `row` where nothing was summed: zeros if it sees no key, else all its keys score -inf and it
// has no softmax.
OMNI_DEV float nothing(const int64_t* lengths, int tokens, int heads, int64_t row) {
  const int64_t t = row / heads;
  return lengths[t / tokens] + t % tokens > 0 ? NAN : 0.f;
}

// TQ: the queries' and output's type; TC: the cache's; NC: columns per unit.
template <typename TQ, typename TC, int D, int NC>
__global__ void __launch_bounds__(kThreads) split_kernel(const PagedAttnArgs a, const Split sp) {
  constexpr int L = D / 8 < 32 ? D / 8 : 32;  // lanes per key
  constexpr int NV = D / 8 / L;               // steps of 8 dims per lane
  constexpr int TEAMS = kThreads / L;
  constexpr bool FP8 = sizeof(TC) == 1;
  grid_launch_dependents();
  grid_dependency_wait();
  const int split = blockIdx.x;
  const int kvh = blockIdx.y / sp.chunks, chunk = blockIdx.y - kvh * sp.chunks;
  const int64_t b = blockIdx.z;
  const int group = a.heads / a.c.kv_heads;
  const int cols = a.tokens * group;
  const int c0 = chunk * sp.cols;
  const int lane = threadIdx.x % L, team = threadIdx.x / L;
  const int64_t cap = (int64_t)a.table_width * a.c.page;
  const int64_t given = a.lengths[b], len = min(given, cap);  // (past the table: reported, and no key past it)
  if (threadIdx.x == 0 && blockIdx.x == 0 && blockIdx.y == 0 && (given < 0 || given > cap - (a.tokens - 1)))
    raise_status(a.status, kStatusIndex);
  const int64_t need = max((int64_t)0, min(cap, len + a.tokens - 1));

  float q[NC][NV][8];
  int64_t lim[NC];  // keys column c sees
  int64_t qrow[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int col = c0 + c;
    const int t = col / group;
    const bool on = c < sp.cols && col < cols;
    qrow[c] = on ? (b * a.tokens + t) * a.heads + kvh * group + (col - t * group) : -1;
    int64_t l = len + t;
    lim[c] = on ? (l < 0 ? 0 : (l > need ? need : l)) : 0;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      if (on) {
        Row8<TQ> r;
        r.load(a.q, qrow[c] * D + (v * L + lane) * 8);
        r.get(q[c][v]);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) q[c][v][i] = 0.f;
      }
    }
  }
  const float qscale = a.scale * kLog2e;
  float m[NC], l[NC], o[NC][NV][8];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    m[c] = -INFINITY;
    l[c] = 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int i = 0; i < 8; ++i) o[c][v][i] = 0.f;
  }
  const int64_t per = (need + sp.splits - 1) / sp.splits;
  const int64_t j0 = split * per, j1 = min(need, j0 + per);
  // Every lane of a warp goes through the same rounds (its teams' sums are shuffles of the whole warp).
  for (int64_t jj = j0; jj < j1; jj += TEAMS) {
    const int64_t j = jj + team;
    const bool on = j < j1;
    int64_t at = 0, si = 0;
    bool page_ok = false;
    if (on) {
      const int64_t pi = j / a.c.page;
      const int off = (int)(j - pi * a.c.page);
      const int64_t id = a.table[b * a.table_stride + pi];
      page_ok = id >= 0 && id < a.c.pages;
      if (page_ok) {
        at = id * a.c.s_page + (int64_t)kvh * a.c.s_head + (int64_t)off * a.c.s_pos;
        si = (id * a.c.kv_heads + kvh) * a.c.page + off;
      } else if (lane == 0) {
        raise_status(a.status, kStatusIndex);
      }
    }
    float s[NC];
    Row8<TC> kr[NV], vr[NV];
#pragma unroll
    for (int c = 0; c < NC; ++c) s[c] = 0.f;
    float ks = 1.f, vs = 1.f;
    if (page_ok) {
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        kr[v].load(a.c.k, at + (v * L + lane) * 8);
        vr[v].load(a.c.v, at + (v * L + lane) * 8);
      }
      if (FP8) {
        ks = __uint_as_float((uint32_t)a.c.k_scale[si] << 23);
        vs = __uint_as_float((uint32_t)a.c.v_scale[si] << 23);
      }
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        float kf[8];
        kr[v].get(kf);
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
          for (int i = 0; i < 8; ++i) s[c] = fmaf(q[c][v][i], kf[i], s[c]);
      }
    }
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int w = L / 2; w > 0; w >>= 1) s[c] += __shfl_xor_sync(0xffffffffu, s[c], w);
    if (page_ok) {
      float p[NC];
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        p[c] = 0.f;
        if (j < lim[c]) {
          const float x = s[c] * (qscale * ks);
          // A NaN score makes the row NaN, as the formula does; -inf scores of every key so far leave m at -inf.
          const float mn = x > m[c] ? x : m[c];
          const float base = mn == -INFINITY ? 0.f : mn;
          const float f = ex2(m[c] - base);
          p[c] = ex2(x - base);
          l[c] = fmaf(l[c], f, p[c]);
          m[c] = mn;
#pragma unroll
          for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int i = 0; i < 8; ++i) o[c][v][i] *= f;
        }
      }
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        float vf[8];
        vr[v].get(vf);
#pragma unroll
        for (int c = 0; c < NC; ++c)
          if (j < lim[c]) {
            const float pv = p[c] * vs;
#pragma unroll
            for (int i = 0; i < 8; ++i) o[c][v][i] = fmaf(pv, vf[i], o[c][v][i]);
          }
      }
    }
  }

  // Join the teams in a fixed order through shared memory, one column at a time.
  __shared__ float s_m[TEAMS], s_l[TEAMS], s_o[TEAMS][D];
#pragma unroll 1
  for (int c = 0; c < NC; ++c) {
    if (qrow[c] < 0) break;
    // The state's registers must keep constant indexes: picked by unrolled compares.
    float mc = 0.f, lc = 0.f;
#pragma unroll
    for (int k = 0; k < NC; ++k)
      if (k == c) {
        mc = m[k];
        lc = l[k];
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
          for (int i = 0; i < 8; ++i) s_o[team][(v * L + lane) * 8 + i] = o[k][v][i];
      }
    if (lane == 0) {
      s_m[team] = mc;
      s_l[team] = lc;
    }
    __syncthreads();
    float top = -INFINITY;
    for (int t = 0; t < TEAMS; ++t) top = fmaxf(top, s_m[t]);
    const float base = top == -INFINITY ? 0.f : top;
    float sum = 0.f;
    for (int t = 0; t < TEAMS; ++t) sum = fmaf(s_l[t], ex2(s_m[t] - base), sum);
    for (int d = threadIdx.x; d < D; d += kThreads) {
      float acc = 0.f;
      for (int t = 0; t < TEAMS; ++t) acc = fmaf(s_o[t][d], ex2(s_m[t] - base), acc);
      if (sp.splits == 1) {
        const float r = sum != 0.f ? acc / sum : nothing(a.lengths, a.tokens, a.heads, qrow[c]);
        reinterpret_cast<TQ*>(a.out)[qrow[c] * D + d] = Elem<TQ>::from_float(r);
      } else {
        sp.part_o[(qrow[c] * sp.splits + split) * D + d] = acc;
      }
    }
    if (sp.splits > 1 && threadIdx.x == 0)
      reinterpret_cast<float2*>(sp.part_ml)[qrow[c] * sp.splits + split] = make_float2(top, sum);
    __syncthreads();
  }
}

template <typename TQ>
__global__ void __launch_bounds__(kThreads) join_kernel(const Split sp, int dim, const int64_t* lengths, int tokens, int heads,
                                                        TQ* __restrict__ out) {
  grid_launch_dependents();
  grid_dependency_wait();
  const int64_t row = blockIdx.x;
  const float2* ml = reinterpret_cast<const float2*>(sp.part_ml) + row * sp.splits;
  float top = -INFINITY;
  for (int s = 0; s < sp.splits; ++s) top = fmaxf(top, ml[s].x);
  const float base = top == -INFINITY ? 0.f : top;
  float sum = 0.f;
  for (int s = 0; s < sp.splits; ++s) sum = fmaf(ml[s].y, ex2(ml[s].x - base), sum);
  for (int d = threadIdx.x; d < dim; d += kThreads) {
    float acc = 0.f;
    for (int s = 0; s < sp.splits; ++s) acc = fmaf(sp.part_o[(row * sp.splits + s) * dim + d], ex2(ml[s].x - base), acc);
    out[row * dim + d] = Elem<TQ>::from_float(sum != 0.f ? acc / sum : nothing(lengths, tokens, heads, row));
  }
}

// Columns per unit: as many as share the keys, while the queries and accumulators stay in registers.
int columns(int dim, int cols) {
  const int most = dim == 512 ? 2 : dim == 256 ? 4 : 4;
  return cols >= most ? most : (cols >= 2 ? 2 : 1);
}

Split plan(int rows, int tokens, int heads, int kv_heads, int dim, int page, int table_width) {
  Split s{};
  const int cols = tokens * (heads / kv_heads);
  s.cols = columns(dim, cols);
  s.chunks = (cols + s.cols - 1) / s.cols;
  // About 8 CTAs per SM, and no split under 64 keys.
  const int64_t units = (int64_t)rows * kv_heads * s.chunks;
  const int64_t keys = (int64_t)page * table_width;
  int64_t want = (8 * device_sm_count() + units - 1) / units;
  want = std::min(want, (keys + 63) / 64);
  s.splits = (int)std::max<int64_t>(1, std::min<int64_t>(want, 256));
  return s;
}

template <typename TQ, typename TC, int D>
cudaError_t launch_cols(const PagedAttnArgs& a, const Split& sp, cudaStream_t s) {
  const dim3 grid((unsigned)sp.splits, (unsigned)(a.c.kv_heads * sp.chunks), (unsigned)a.rows);
  if (sp.cols == 1) return launch_dependent(split_kernel<TQ, TC, D, 1>, grid, dim3(kThreads), 0, s, a, sp);
  if (sp.cols == 2) return launch_dependent(split_kernel<TQ, TC, D, 2>, grid, dim3(kThreads), 0, s, a, sp);
  if constexpr (D <= 256) return launch_dependent(split_kernel<TQ, TC, D, 4>, grid, dim3(kThreads), 0, s, a, sp);
  return cudaErrorInvalidValue;
}

template <typename TQ, typename TC>
cudaError_t launch_dim(const PagedAttnArgs& a, const Split& sp, cudaStream_t s) {
  switch (a.c.dim) {
    case 16: return launch_cols<TQ, TC, 16>(a, sp, s);
    case 32: return launch_cols<TQ, TC, 32>(a, sp, s);
    case 64: return launch_cols<TQ, TC, 64>(a, sp, s);
    case 128: return launch_cols<TQ, TC, 128>(a, sp, s);
    case 256: return launch_cols<TQ, TC, 256>(a, sp, s);
    case 512: return launch_cols<TQ, TC, 512>(a, sp, s);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace paged

size_t paged_attention_workspace(int, int, int rows, int tokens, int heads, int kv_heads, int dim, int page,
                                 int table_width) {
  const paged::Split s = paged::plan(rows, tokens, heads, kv_heads, dim, page, table_width);
  if (s.splits == 1) return kCounterBytes;
  return kCounterBytes + (size_t)rows * tokens * heads * s.splits * (dim + 2) * sizeof(float);
}

cudaError_t launch_paged_attention(int dtype, const PagedAttnArgs& a, cudaStream_t stream) {
  paged::Split sp = paged::plan(a.rows, a.tokens, a.heads, a.c.kv_heads, a.c.dim, a.c.page, a.table_width);
  const int64_t qrows = (int64_t)a.rows * a.tokens * a.heads;
  sp.part_o = reinterpret_cast<float*>(reinterpret_cast<char*>(a.workspace) + kCounterBytes);
  sp.part_ml = sp.part_o + qrows * sp.splits * a.c.dim;
  cudaError_t e;
  if (dtype == kBF16)
    e = a.c.type == kFp8 ? paged::launch_dim<__nv_bfloat16, __nv_fp8_e4m3>(a, sp, stream)
                         : paged::launch_dim<__nv_bfloat16, __nv_bfloat16>(a, sp, stream);
  else
    e = a.c.type == kFp8 ? paged::launch_dim<float, __nv_fp8_e4m3>(a, sp, stream)
                         : paged::launch_dim<float, float>(a, sp, stream);
  if (e != cudaSuccess || sp.splits == 1) return e;
  if (dtype == kBF16)
    return launch_dependent(paged::join_kernel<__nv_bfloat16>, dim3((unsigned)qrows), dim3(paged::kThreads), 0, stream, sp,
                            a.c.dim, a.lengths, a.tokens, a.heads, reinterpret_cast<__nv_bfloat16*>(a.out));
  return launch_dependent(paged::join_kernel<float>, dim3((unsigned)qrows), dim3(paged::kThreads), 0, stream, sp, a.c.dim,
                          a.lengths, a.tokens, a.heads, reinterpret_cast<float*>(a.out));
}

}  // namespace omni
