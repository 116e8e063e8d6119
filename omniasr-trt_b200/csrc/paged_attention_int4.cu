// Attention of each row's newest tokens over a paged cache held in 4 bits (bf16 queries, head_dim 64 to 512).
//
// Query column c < T G of a unit (row, kv head; G = heads / kv_heads, column c = token c / G, head kv G + c % G) sees keys
// [0, lengths[b] + c / G). A key costs 2 (D / 2 + D / 16) bytes and nothing else is read more than once, so the bound is HBM, and next
// to it the instructions that make operands of the codes: 2 D codes a key, about 0.17 keys a clock and SM at HBM's rate, with 64
// integer lanes a clock. Hence:
//
// * The codes never become a tile in shared memory (for tcgen05 they would be written and read there in four times their bytes,
//   more than its 128 bytes a clock): each lane dequantises in registers what it feeds to mma.m16n8k16 itself, whose rate
//   (one per two clocks and SM) is more than twice what is needed. The cache's order of codes (int4.cuh) makes a lane's share of a
//   vector one run of 16 bytes (K) or 8 (V).
// * S^T = K Q^T, 16 keys x 8 columns. A code masked out of its word is, read as fp16, the subnormal c 2^-24 (16 c 2^-24 four bits
//   up), exact, so a word of 8 codes takes four ands and a shift; the queries (fp16, scaled by a power of two per column so that the
//   largest is 2^14 and more: exact but for values 2^-28 of it) carry the factors. The sums start from -8 sum q, which is the
//   codes' offset, and every group's sum is scaled in fp32.
// * O^T = V^T P^T: two keys' codes of a dim are the halves of a word after one byte permutation; 128 + c - 8 is exact in
//   bf16. The scales go onto the probabilities: P^T is turned by movmatrix and multiplied per group, so that no value needs one.
// * Warps are independent: each takes blocks of 16 or 32 keys of the CTA's share with a maximum, a sum and an accumulator of
//   its own, and copies its next blocks asynchronously into a ring of its own; no barrier in the loop. A column's maximum is raised
//   only when a score passes it by 2^8. At a unit's end the CTA's warps join through shared memory.
// * All blocks of all units are cut evenly between the CTAs. A unit that is cut leaves parts in the workspace; the CTA that
//   publishes last joins them in the order of the keys, so a call repeats its bits.
//
// What a column does not see has weight zero: its score is masked before the exponential, and its group scales (which may be
// NaN) are masked out of the products; keys past the row's last are not read.

#include <math.h>

#include <algorithm>

#include "attention.cuh"
#include "common.cuh"
#include "int4.cuh"
#include "paged.cuh"

namespace omni {
namespace paged4 {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr float kLazy = 8.f;  // log2 of how far a score may pass its column's maximum

template <int DIM, int NT>  // NT: tiles of 8 columns
struct Cfg {
  static constexpr int kMt = DIM <= 128 ? 2 : 1;  // tiles of 16 keys per block
  static constexpr int kKeys = 16 * kMt;
  static constexpr int kRow = DIM / 2;      // bytes of a vector's codes
  static constexpr int kScale = DIM / 16;   // and of its scales
  static constexpr int kBlocks = DIM < 128 ? 1 : DIM / 128;
  static constexpr int kGroups = DIM < 128 ? DIM / 32 : 4;  // per block of 128 dims
  static constexpr int kStage = 2 * kKeys * (kRow + kScale);
  static constexpr int kStages = DIM == 64 ? 4 : 2;
  static constexpr int kCols = 8 * NT;
  static constexpr int kPitch = 132;  // floats between columns of the joining buffer: a quarter warp's float4 meet all banks
  // shared memory
  static constexpr int kRing = 0;
  static constexpr int kQ = kRing + kWarps * kStages * kStage;
  static constexpr int kInit = kQ + DIM / 16 * NT * 256;
  static constexpr int kMl = kInit + DIM / 32 * kCols * 4;
  static constexpr int kLim = kMl + kWarps * kCols * 8;
  static constexpr int kJoin = (kLim + kCols * 8 + 15) / 16 * 16;
  static constexpr int kBytes = kJoin + kWarps * 8 * kPitch * 4;
  static constexpr int kCtas = DIM == 512 || NT * DIM >= 384 || NT * DIM == 256 && DIM == 64 ? 2 : NT * DIM > 128 ? 3 : 4;  // per SM, for the registers
};

struct Params {
  PagedAttnArgs a;
  int cols, chunks;  // columns of a (row, kv head); units per (row, kv head)
  int grid;
  unsigned* counters;  // [grid], zero on entry and left zero
  float* part_o;       // [2 grid][cols of a unit][dim]
  float2* part_ml;     // [2 grid][cols of a unit]
};

OMNI_DEV void copy_async(uint32_t dst, const void* src, bool on, int bytes) {
  const int n = on ? bytes : 0;  // the rest is zeros
  if (bytes == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
  else if (bytes == 8)
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
OMNI_DEV void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
OMNI_DEV void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

template <int WORDS>
OMNI_DEV void load_words(uint32_t* w, uint32_t addr) {
  if constexpr (WORDS == 4)
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(addr));
  else if constexpr (WORDS == 2)
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(addr));
  else
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[0]) : "r"(addr));
}

OMNI_DEV void mma_f16(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, const uint32_t* b) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b[0]), "r"(b[1]));
}
OMNI_DEV void mma_bf16(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
OMNI_DEV uint32_t turned(uint32_t x) {  // an 8 x 8 tile of 16-bit values across the warp, transposed
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
OMNI_DEV uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// Nibble n of each half of z as bf16 c - 8.
OMNI_DEV uint32_t centred(uint32_t z, int n) {
  const uint32_t v = ((z >> (4 * n)) & 0x000f000fu) | 0x43004300u;  // 128 + c
  uint32_t r;
  asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(v), "r"(0x43084308u));
  return r;
}

// Where the 16-byte word c of key r's codes lies in a tile: so that a quarter warp's reads (K: 16 bytes of 2 keys x 4 lanes; V, 8
// bytes: 4 keys x 4 lanes) meet all banks. Keys of V lie in the order of its operand, so that a lane's four are 4 apart.
template <int DIM>
OMNI_DEV int k_place(int r, int c) {
  return r * (DIM / 32) + (DIM >= 256 ? c ^ ((r & 1) << 2) : c);
}
OMNI_DEV int v_slot(int r) { return (r & 24) | ((r & 1) << 2) | ((r >> 1) & 3); }
template <int DIM>
OMNI_DEV int v_place(int slot, int c) {
  return slot * (DIM / 32) + (DIM >= 256 ? c ^ ((slot & 3) << 1) : DIM == 128 ? c ^ (slot & 2) : c);
}

// A walk over the units in order: unit (row, hc) has the blocks [u0, u0 + nb).
struct Walk {
  int64_t u0;
  int row, hc, nb;
  int len, need;  // keys the row's first query sees (at least 0), and its last
};

template <int KEYS>
struct Rows {
  const Params& p;
  int64_t cap;
  OMNI_DEV explicit Rows(const Params& q) : p(q), cap((int64_t)q.a.table_width * q.a.c.page) {}
  OMNI_DEV void look(int row, Walk& w) const {
    const int64_t len = min(p.a.lengths[row], cap);
    w.need = (int)max((int64_t)0, min(cap, len + p.a.tokens - 1));
    w.len = (int)max(len, (int64_t)-p.a.tokens);
    w.nb = (w.need + KEYS - 1) / KEYS;
  }
  OMNI_DEV void next(Walk& w) const {
    w.u0 += w.nb;
    if (++w.hc == p.a.c.kv_heads * p.chunks) {
      w.hc = 0;
      while (++w.row < p.a.rows) {
        look(w.row, w);
        if (w.nb) break;
      }
    }
  }
};

OMNI_DEV int64_t block_sum(int64_t v, int64_t* s) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  int64_t t = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) t += s[w];
  return t;
}

template <int DIM, int NT>
struct Kernel {
  using C = Cfg<DIM, NT>;
  static constexpr int W2 = C::kGroups / 2;  // 32-bit words of a block's scales, of a lane's V codes

  const Params& p;
  char* smem;
  uint32_t ring;  // this warp's
  int lane, warp, g, t;
  uint32_t q_at, init_at;

  float o[C::kBlocks * C::kGroups][2][NT][4];
  float m[NT][2], l[NT][2], qs[NT][2];

  OMNI_DEV Kernel(const Params& q, char* s) : p(q), smem(s) {
    lane = threadIdx.x & 31;
    warp = threadIdx.x >> 5;
    g = lane >> 2;
    t = lane & 3;
    ring = smem_addr(smem) + C::kRing + warp * C::kStages * C::kStage;
    q_at = smem_addr(smem) + C::kQ + lane * 8;
    init_at = smem_addr(smem) + C::kInit + t * 8;
  }

  // ---- loads: block n (of the walk's unit) into a stage of the ring

  OMNI_DEV void fetch(const Walk& w, int64_t n, int stage) {
    const PagedAttnArgs& a = p.a;
    const int j0 = (int)(n - w.u0) * C::kKeys;
    const int h = w.hc / p.chunks;
    const uint32_t kd = ring + stage * C::kStage, vd = kd + C::kKeys * C::kRow, ksd = vd + C::kKeys * C::kRow,
                   vsd = ksd + C::kKeys * C::kScale;
    // The page of each key: lane r's.
    const int jr = j0 + (lane < C::kKeys ? lane : 0);
    int id = -1, off = 0;
    if (jr < w.need) {
      const int pi = jr / a.c.page;
      off = jr - pi * a.c.page;
      id = a.table[w.row * a.table_stride + pi];
      if (id < 0 || id >= a.c.pages) {
        if (lane < C::kKeys) raise_status(a.status, kStatusIndex);
        id = -1;
      }
    }
    constexpr int CPR = C::kRow / 16;              // 16-byte words per key
    constexpr int N = C::kKeys * CPR / 32;         // per lane
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int r = (lane + 32 * i) / CPR, c = lane % CPR;
      const int rid = __shfl_sync(0xffffffffu, id, r), roff = __shfl_sync(0xffffffffu, off, r);
      const bool on = rid >= 0;
      const int64_t at = on ? rid * a.c.s_page + h * a.c.s_head + roff * a.c.s_pos + c * 16 : 0;
      const int tile = r >> 4, rr = r & 15;
      copy_async(kd + (tile * 16 * CPR + k_place<DIM>(rr, c)) * 16, reinterpret_cast<const char*>(a.c.k) + at, on, 16);
      copy_async(vd + (tile * 16 * CPR + v_place<DIM>(v_slot(rr), c)) * 16, reinterpret_cast<const char*>(a.c.v) + at, on, 16);
    }
    constexpr int CS = C::kScale < 16 ? C::kScale : 16, SPR = C::kScale / CS;  // bytes of a copy, copies per key
    static_assert(C::kKeys * SPR <= 32, "a copy per lane");
    const int r = lane / SPR % C::kKeys, c = lane % SPR;
    const int rid = __shfl_sync(0xffffffffu, id, r), roff = __shfl_sync(0xffffffffu, off, r);
    if (C::kKeys * SPR == 32 || lane < C::kKeys * SPR) {
      const bool on = rid >= 0;
      const int64_t at = on ? (((int64_t)rid * a.c.kv_heads + h) * a.c.page + roff) * C::kScale + c * CS : 0;
      copy_async(ksd + r * C::kScale + c * CS, reinterpret_cast<const char*>(a.c.k_scale) + at, on, CS);
      copy_async(vsd + v_slot(r) * C::kScale + c * CS, reinterpret_cast<const char*>(a.c.v_scale) + at, on, CS);
    }
  }

  // ---- a unit's queries

  OMNI_DEV int limit(const Walk& w, int col) const {  // keys a column sees; -1: no such column
    const int gr = p.a.heads / p.a.c.kv_heads;
    return col < p.cols ? max(0, min(w.need, w.len + col / gr)) : -1;
  }
  OMNI_DEV int64_t query_row(const Walk& w, int col) const {
    const int gr = p.a.heads / p.a.c.kv_heads, tok = col / gr;
    return ((int64_t)w.row * p.a.tokens + tok) * p.a.heads + w.hc / p.chunks * gr + (col - tok * gr);
  }

  // Warp by warp a column: fp16 operands in the order of the codes, the sums' start per group, the factor of its scores.
  OMNI_DEV void load_queries(const Walk& w) {
    const int c0 = w.hc % p.chunks * C::kCols;
    float* init = reinterpret_cast<float*>(smem + C::kInit);
    float* factor = reinterpret_cast<float*>(smem + C::kLim);
    int* lims = reinterpret_cast<int*>(smem + C::kLim) + C::kCols;
    constexpr int V = DIM > 256 ? 2 : 1;  // words of 8 dims per lane
    for (int col = warp; col < C::kCols; col += kWarps) {
      const int lim = limit(w, c0 + col);
      float x[V][8];
      uint32_t top = 0u;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const int word = v * 32 + lane;
        uint4 u = make_uint4(0u, 0u, 0u, 0u);
        if (lim >= 0 && word * 8 < DIM)
          u = __ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const __nv_bfloat16*>(p.a.q) + query_row(w, c0 + col) * DIM) + word);
        Elem<__nv_bfloat16>::unpack(u, x[v]);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint32_t b = __float_as_uint(x[v][i]) & 0x7fffffffu;
          top = max(top, b < 0x7f800000u ? b : 0u);
        }
      }
      top = __reduce_max_sync(0xffffffffu, top);
      const int e = top == 0u ? 0 : max(-112, (int)(top >> 23) - 127);
      const float up = __uint_as_float((uint32_t)(14 - e + 127) << 23);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const int word = v * 32 + lane;
        uint32_t b[4];
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {  // nibbles i and i + 4 of the word; odd ones stand for 16 c
          const float f = (i & 1) ? up * 0.0625f : up;
          const __half2 h = __floats2half2_rn(x[v][i] * f, x[v][i + 4] * f);
          b[i] = *reinterpret_cast<const uint32_t*>(&h);
          const float2 back = __half22float2(h);
          sum += (back.x + back.y) * ((i & 1) ? 16.f : 1.f);
        }
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        if (word * 8 < DIM) {
          const int group = word >> 2;
          uint2* dst = reinterpret_cast<uint2*>(smem + C::kQ) + ((group * 2) * NT + (col >> 3)) * 32 + (col & 7) * 4 + (word & 3);
          dst[0] = make_uint2(b[0], b[1]);
          dst[NT * 32] = make_uint2(b[2], b[3]);
          if ((word & 3) == 0) init[group * C::kCols + col] = sum * (-8.f * 0x1p-24f);
        }
      }
      if (lane == 0) {
        factor[col] = p.a.scale * kLog2e * 0x1p10f * __uint_as_float((uint32_t)(e + 127) << 23);
        lims[col] = lim;
      }
    }
  }

  OMNI_DEV void start_unit() {
    const float* factor = reinterpret_cast<const float*>(smem + C::kLim);
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        m[n][i] = -INFINITY;
        l[n][i] = 0.f;
        qs[n][i] = factor[n * 8 + 2 * t + i];
      }
#pragma unroll
    for (int b = 0; b < C::kBlocks * C::kGroups; ++b)
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) o[b][j][n][i] = 0.f;
  }

  // ---- one block. TAIL: some column does not see all of it.

  template <bool TAIL>
  OMNI_DEV void block(int stage, int j0) {
    const uint32_t kd = ring + stage * C::kStage, vd = kd + C::kKeys * C::kRow, ksd = vd + C::kKeys * C::kRow,
                   vsd = ksd + C::kKeys * C::kScale;
    const int* lims = reinterpret_cast<const int*>(smem + C::kLim) + C::kCols;
    float s[C::kMt][NT][4];
#pragma unroll
    for (int k = 0; k < C::kMt; ++k)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[k][n][i] = 0.f;
#pragma unroll
    for (int b = 0; b < C::kBlocks; ++b) {
      uint32_t kw[C::kMt][2][C::kGroups], ks[C::kMt][2][W2];
#pragma unroll
      for (int k = 0; k < C::kMt; ++k)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int r = g + 8 * e;
          if constexpr (C::kGroups == 4)
            load_words<4>(kw[k][e], kd + k * 16 * C::kRow + k_place<DIM>(r, b * 4 + t) * 16);
          else
            load_words<2>(kw[k][e], kd + k * 16 * C::kRow + r * C::kRow + t * 8);
          load_words<W2>(ks[k][e], ksd + (k * 16 + r) * C::kScale + b * 8);
        }
#pragma unroll
      for (int gr = 0; gr < C::kGroups; ++gr) {
        const int group = b * C::kGroups + gr;
        uint32_t lo[C::kMt][4], hi[C::kMt][4];  // the operands of keys g and g + 8: nibbles (0, 4), (1, 5), (2, 6), (3, 7)
#pragma unroll
        for (int k = 0; k < C::kMt; ++k) {
          const uint32_t x = kw[k][0][gr], y = kw[k][1][gr];
          lo[k][0] = x & 0x000f000fu, lo[k][1] = x & 0x00f000f0u, lo[k][2] = (x >> 8) & 0x000f000fu, lo[k][3] = (x >> 8) & 0x00f000f0u;
          hi[k][0] = y & 0x000f000fu, hi[k][1] = y & 0x00f000f0u, hi[k][2] = (y >> 8) & 0x000f000fu, hi[k][3] = (y >> 8) & 0x00f000f0u;
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          uint32_t q0[2], q1[2], start[2];
          load_words<2>(q0, q_at + ((group * 2) * NT + n) * 256);
          load_words<2>(q1, q_at + ((group * 2 + 1) * NT + n) * 256);
          load_words<2>(start, init_at + (group * C::kCols + n * 8) * 4);
#pragma unroll
          for (int k = 0; k < C::kMt; ++k) {
            float c[4] = {__uint_as_float(start[0]), __uint_as_float(start[1]), __uint_as_float(start[0]), __uint_as_float(start[1])};
            mma_f16(c, lo[k][0], hi[k][0], lo[k][1], hi[k][1], q0);
            mma_f16(c, lo[k][2], hi[k][2], lo[k][3], hi[k][3], q1);
            const uint32_t w0 = ks[k][0][gr >> 1], w1 = ks[k][1][gr >> 1];
            const float s0 = __uint_as_float((gr & 1) ? w0 & 0xffff0000u : w0 << 16), s1 = __uint_as_float((gr & 1) ? w1 & 0xffff0000u : w1 << 16);
            s[k][n][0] = fmaf(s0, c[0], s[k][n][0]);
            s[k][n][1] = fmaf(s0, c[1], s[k][n][1]);
            s[k][n][2] = fmaf(s1, c[2], s[k][n][2]);
            s[k][n][3] = fmaf(s1, c[3], s[k][n][3]);
          }
        }
      }
    }
    // Scores, masks, the maxima.
    bool raise = false;
#pragma unroll
    for (int k = 0; k < C::kMt; ++k)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float& x = s[k][n][i];
          x *= qs[n][i & 1];
          if (TAIL && j0 + k * 16 + g + (i & 2) * 4 >= lims[n * 8 + 2 * t + (i & 1)]) x = -INFINITY;
          raise |= x > m[n][i & 1] + kLazy;
        }
    if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float top = m[n][i];
#pragma unroll
          for (int k = 0; k < C::kMt; ++k) top = fmaxf(top, fmaxf(s[k][n][i], s[k][n][i + 2]));
#pragma unroll
          for (int w = 4; w < 32; w <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
          const float f = m[n][i] == top ? 1.f : ex2(m[n][i] - top);
          m[n][i] = top;
          l[n][i] *= f;
#pragma unroll
          for (int b = 0; b < C::kBlocks * C::kGroups; ++b)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              o[b][j][n][i] *= f;
              o[b][j][n][i + 2] *= f;
            }
        }
    }
#pragma unroll
    for (int k = 0; k < C::kMt; ++k) {
      uint32_t pt[NT][2], seen[NT][2];  // P^T's operand: column g, keys (2 t, 2 t + 1) and those + 8
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float e[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float base = m[n][i & 1] == -INFINITY ? 0.f : m[n][i & 1];
          e[i] = ex2(s[k][n][i] - base);
          l[n][i & 1] += e[i];
        }
        const __nv_bfloat162 a = __floats2bfloat162_rn(e[0], e[1]), b = __floats2bfloat162_rn(e[2], e[3]);
        pt[n][0] = turned(*reinterpret_cast<const uint32_t*>(&a));
        pt[n][1] = turned(*reinterpret_cast<const uint32_t*>(&b));
        if (TAIL) {
          const int lim = lims[n * 8 + g], j = j0 + k * 16 + 2 * t;
#pragma unroll
          for (int i = 0; i < 2; ++i)
            seen[n][i] = (j + 8 * i < lim ? 0xffffu : 0u) | (j + 8 * i + 1 < lim ? 0xffff0000u : 0u);
        }
      }
#pragma unroll
      for (int b = 0; b < C::kBlocks; ++b) {
        uint32_t vw[4][W2], vs[4][W2];  // keys 2 t, 2 t + 1, 2 t + 8, 2 t + 9: the slots t, t + 4, t + 8, t + 12
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int slot = t + 4 * i;
          if constexpr (W2 == 2)
            load_words<2>(vw[i], vd + k * 16 * C::kRow + v_place<DIM>(slot, b * 4 + (g >> 1)) * 16 + (g & 1) * 8);
          else
            load_words<1>(vw[i], vd + k * 16 * C::kRow + slot * C::kRow + g * 4);
          load_words<W2>(vs[i], vsd + (k * 16 + slot) * C::kScale + b * 8);
        }
#pragma unroll
        for (int gr = 0; gr < C::kGroups; ++gr) {
          const uint32_t sel = (gr & 1) ? 0x7632u : 0x5410u;
          const uint32_t za = __byte_perm(vw[0][gr >> 1], vw[1][gr >> 1], sel), zb = __byte_perm(vw[2][gr >> 1], vw[3][gr >> 1], sel);
          const uint32_t sa = __byte_perm(vs[0][gr >> 1], vs[1][gr >> 1], sel), sb = __byte_perm(vs[2][gr >> 1], vs[3][gr >> 1], sel);
          const uint32_t a0[4] = {centred(za, 0), centred(za, 1), centred(zb, 0), centred(zb, 1)};
          const uint32_t a1[4] = {centred(za, 2), centred(za, 3), centred(zb, 2), centred(zb, 3)};
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            uint32_t b0 = mul_bf16x2(pt[n][0], sa), b1 = mul_bf16x2(pt[n][1], sb);
            if (TAIL) {
              b0 &= seen[n][0];
              b1 &= seen[n][1];
            }
            mma_bf16(o[b * C::kGroups + gr][0][n], a0, b0, b1);
            mma_bf16(o[b * C::kGroups + gr][1][n], a1, b0, b1);
          }
        }
      }
    }
  }

  // ---- a unit's end: the warps' states joined, the CTA's part written (to `part` of the workspace, or out)

  OMNI_DEV void write_out(const Walk& w, int col, int d, float4 x, float sum) {
    const int64_t row = query_row(w, col);
    const float none = w.len + col / (p.a.heads / p.a.c.kv_heads) > 0 ? NAN : 0.f;  // (its keys all score -inf, or it sees none)
    const float inv = 1.f / sum;
    const bool any = sum != 0.f;
    const __nv_bfloat162 a = __floats2bfloat162_rn(any ? x.x * inv : none, any ? x.y * inv : none),
                         b = __floats2bfloat162_rn(any ? x.z * inv : none, any ? x.w * inv : none);
    uint2 u;
    u.x = *reinterpret_cast<const uint32_t*>(&a);
    u.y = *reinterpret_cast<const uint32_t*>(&b);
    *reinterpret_cast<uint2*>(reinterpret_cast<__nv_bfloat16*>(p.a.out) + row * DIM + d) = u;
  }

  OMNI_DEV void end_unit(const Walk& w, int part) {
    float2* ml = reinterpret_cast<float2*>(smem + C::kMl);
    float* join = reinterpret_cast<float*>(smem + C::kJoin);
    const int c0 = w.hc % p.chunks * C::kCols;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int k = 4; k < 32; k <<= 1) l[n][i] += __shfl_xor_sync(0xffffffffu, l[n][i], k);
        if (g == 0) ml[warp * C::kCols + n * 8 + 2 * t + i] = make_float2(m[n][i], l[n][i]);
      }
    __syncthreads();
    auto joined = [&](int col, float& top, float& sum) {
      top = -INFINITY;
      for (int k = 0; k < kWarps; ++k) top = fmaxf(top, ml[k * C::kCols + col].x);
      const float base = top == -INFINITY ? 0.f : top;
      sum = 0.f;
      for (int k = 0; k < kWarps; ++k) sum = fmaf(ml[k * C::kCols + col].y, ex2(ml[k * C::kCols + col].x - base), sum);
    };
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      if (c0 + n * 8 >= p.cols) break;
      float f[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float top, sum;
        joined(n * 8 + 2 * t + i, top, sum);
        f[i] = ex2(m[n][i] - (top == -INFINITY ? 0.f : top));
      }
#pragma unroll
      for (int b = 0; b < C::kBlocks; ++b) {
#pragma unroll
        for (int gr = 0; gr < C::kGroups; ++gr)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float(&x)[2][NT][4] = o[b * C::kGroups + gr];
            *reinterpret_cast<float4*>(join + (warp * 8 + 2 * t + i) * C::kPitch + gr * 32 + g * 4) =
                make_float4(x[0][n][i] * f[i], x[0][n][i + 2] * f[i], x[1][n][i] * f[i], x[1][n][i + 2] * f[i]);
          }
        __syncthreads();
        constexpr int Q4 = C::kGroups * 8;  // float4 of a column
        for (int e = threadIdx.x; e < 8 * Q4; e += kThreads) {
          const int col = e / Q4, d = e % Q4 * 4;
          if (c0 + n * 8 + col < p.cols) {
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int k = 0; k < kWarps; ++k) {
              const float4 y = *reinterpret_cast<const float4*>(join + (k * 8 + col) * C::kPitch + d);
              x.x += y.x, x.y += y.y, x.z += y.z, x.w += y.w;
            }
            float top, sum;
            joined(n * 8 + col, top, sum);
            if (part < 0) {
              write_out(w, c0 + n * 8 + col, b * 128 + d, x, sum);
            } else {
              const int64_t at = (int64_t)part * C::kCols + n * 8 + col;
              *reinterpret_cast<float4*>(p.part_o + at * DIM + b * 128 + d) = x;
              if (b == 0 && d == 0) p.part_ml[at] = make_float2(top, sum);
            }
          }
        }
        __syncthreads();
      }
    }
  }

  // The parts of a unit cut between the CTAs first .. last, in their order. A CTA's part of a unit that starts before its share is
  // its slot 0, of one that starts in it slot 1.
  OMNI_DEV void join_parts(const Walk& w, int first, int last) {
    const int c0 = w.hc % p.chunks * C::kCols;
    constexpr int Q4 = DIM / 4;
    for (int e = threadIdx.x; e < C::kCols * Q4; e += kThreads) {
      const int col = e / Q4, d = e % Q4 * 4;
      if (c0 + col >= p.cols) break;
      auto at = [&](int c) { return (int64_t)(2 * c + (c == first)) * C::kCols + col; };
      float top = -INFINITY;
      for (int c = first; c <= last; ++c) top = fmaxf(top, __ldcg(p.part_ml + at(c)).x);
      const float base = top == -INFINITY ? 0.f : top;
      float sum = 0.f;
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int c = first; c <= last; ++c) {
        const float2 s = __ldcg(p.part_ml + at(c));
        const float4 y = __ldcg(reinterpret_cast<const float4*>(p.part_o + at(c) * DIM + d));
        const float f = ex2(s.x - base);
        sum = fmaf(s.y, f, sum);
        x.x = fmaf(y.x, f, x.x), x.y = fmaf(y.y, f, x.y), x.z = fmaf(y.z, f, x.z), x.w = fmaf(y.w, f, x.w);
      }
      write_out(w, c0 + col, d, x, sum);
    }
  }
};

template <int DIM, int NT>
__global__ void __launch_bounds__(kThreads, Cfg<DIM, NT>::kCtas) int4_kernel(const __grid_constant__ Params p) {
  using C = Cfg<DIM, NT>;
  extern __shared__ __align__(16) char smem[];
  __shared__ int64_t s_sum[kWarps];
  __shared__ int64_t s_u0;
  __shared__ int s_row, s_last;
  Kernel<DIM, NT> k(p, smem);
  grid_launch_dependents();
  grid_dependency_wait();
  const Rows<C::kKeys> rows(p);
  const int hcs = p.a.c.kv_heads * p.chunks, cta = blockIdx.x;

  // The shares: all units' blocks cut evenly.
  int64_t mine = 0;
  for (int r = threadIdx.x; r < p.a.rows; r += kThreads) {
    Walk w;
    rows.look(r, w);
    mine += w.nb;
    const int64_t given = p.a.lengths[r];
    if (cta == 0 && (given < 0 || given > rows.cap - (p.a.tokens - 1))) raise_status(p.a.status, kStatusIndex);
  }
  const int64_t total = block_sum(mine, s_sum) * hcs;
  const int64_t per = max((total + p.grid - 1) / p.grid, (int64_t)kWarps);
  const int64_t b0 = min(total, per * cta), b1 = min(total, b0 + per);
  // Rows without keys: zeros.
  for (int r = cta; r < p.a.rows; r += p.grid) {
    Walk w;
    rows.look(r, w);
    if (w.nb == 0) {
      const int64_t n = (int64_t)p.a.tokens * p.a.heads * DIM / 8;
      uint4* dst = reinterpret_cast<uint4*>(reinterpret_cast<__nv_bfloat16*>(p.a.out) + (int64_t)r * p.a.tokens * p.a.heads * DIM);
      for (int64_t i = threadIdx.x; i < n; i += kThreads) dst[i] = make_uint4(0u, 0u, 0u, 0u);
    }
  }
  if (b0 >= b1) return;
  // The row that b0 lies in: sums of kThreads rows at a time, then one after another within.
  {
    int64_t before = 0;
    for (int r0 = 0;; r0 += kThreads) {
      Walk w;
      w.nb = 0;
      if (r0 + (int)threadIdx.x < p.a.rows) rows.look(r0 + threadIdx.x, w);
      const int64_t n = (int64_t)w.nb * hcs;
      int64_t x = n;  // the sum up to this thread's row
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
        if (k.lane >= o) x += y;
      }
      __syncthreads();
      if (k.lane == 31) s_sum[k.warp] = x;
      __syncthreads();
      int64_t all = 0;
#pragma unroll
      for (int i = 0; i < kWarps; ++i) {
        if (i < k.warp) x += s_sum[i];
        all += s_sum[i];
      }
      x += before;
      if (b0 < x && b0 >= x - n) {
        s_row = r0 + threadIdx.x;
        s_u0 = x - n;
      }
      before += all;
      if (b0 < before) break;
    }
    __syncthreads();
  }
  Walk use;
  use.row = s_row;
  rows.look(use.row, use);
  use.hc = (int)((b0 - s_u0) / use.nb);
  use.u0 = s_u0 + (int64_t)use.hc * use.nb;

  // This warp's blocks: b0 + warp, and every kWarps-th from there.
  Walk get = use;
  int64_t next = b0 + k.warp;  // the next block to copy
  int put = 0;                 // its stage
  auto fetch = [&]() {
    if (next < b1) {
      while (next >= get.u0 + get.nb) rows.next(get);
      k.fetch(get, next, put);
      next += kWarps;
    }
    copy_commit();
    put = put + 1 == C::kStages ? 0 : put + 1;
  };
#pragma unroll 1
  for (int i = 0; i < C::kStages - 1; ++i) fetch();

  int64_t n = b0 + k.warp;
  int take = 0;
  while (true) {
    k.load_queries(use);
    __syncthreads();
    k.start_unit();
    const int64_t end = min(b1, use.u0 + use.nb);
    const int full = max(0, use.len);  // keys that every column sees
#pragma unroll 1
    for (; n < end; n += kWarps) {
      fetch();  // into the stage that the block before has left
      copy_wait<C::kStages - 1>();
      __syncwarp();
      const int j0 = (int)(n - use.u0) * C::kKeys;
      if (j0 + C::kKeys <= full) k.template block<false>(take, j0);
      else k.template block<true>(take, j0);
      __syncwarp();
      take = take + 1 == C::kStages ? 0 : take + 1;
    }
    const int first = (int)(use.u0 / per), last = (int)((use.u0 + use.nb - 1) / per);
    const bool cut = first != last;
    k.end_unit(use, cut ? 2 * cta + (cta == first) : -1);
    if (cut) {
      __threadfence();
      __syncthreads();
      if (threadIdx.x == 0) {
        s_last = atomicAdd(p.counters + first, 1u) == (unsigned)(last - first);
        if (s_last) p.counters[first] = 0u;
        __threadfence();
      }
      __syncthreads();
      if (s_last) k.join_parts(use, first, last);
    }
    if (end == b1) break;
    rows.next(use);
  }
  copy_wait<0>();
}

// Tiles of 8 columns of a unit: as many as share the keys while the accumulators stay in registers.
int most_tiles(int dim) { return dim <= 128 ? 4 : dim == 256 ? 2 : 1; }

int tiles_of(int dim, int cols) {
  const int tiles = (cols + 7) / 8, most = most_tiles(dim);
  const int chunks = (tiles + most - 1) / most;
  return (tiles + chunks - 1) / chunks;
}

template <int DIM, int NT>
int grid_of() {
  return device_sm_count() * std::min(Cfg<DIM, NT>::kCtas, (227 << 10) / (Cfg<DIM, NT>::kBytes + 1024 + 256));
}

template <int DIM, int NT>
cudaError_t launch(const PagedAttnArgs& a, cudaStream_t s) {
  using C = Cfg<DIM, NT>;
  static PerDevice done;
  if (cudaError_t e = allow_smem(int4_kernel<DIM, NT>, C::kBytes, done)) return e;
  Params p;
  p.a = a;
  p.cols = a.tokens * (a.heads / a.c.kv_heads);
  p.chunks = (p.cols + C::kCols - 1) / C::kCols;
  p.grid = grid_of<DIM, NT>();
  p.counters = reinterpret_cast<unsigned*>(a.workspace);
  p.part_o = reinterpret_cast<float*>(reinterpret_cast<char*>(a.workspace) + kCounterBytes);
  p.part_ml = reinterpret_cast<float2*>(p.part_o + (int64_t)2 * p.grid * C::kCols * DIM);
  return launch_dependent(int4_kernel<DIM, NT>, dim3((unsigned)p.grid), dim3(kThreads), C::kBytes, s, p);
}

}  // namespace paged4

bool paged_int4_supported(int dtype, int type, int dim) { return dtype == kBF16 && type == kInt4 && dim >= 64; }

size_t paged_int4_workspace(int dim) {
  // Two parts a CTA, of all the columns a unit can have.
  return kCounterBytes + (size_t)2 * 4 * device_sm_count() * paged4::most_tiles(dim) * 8 * (dim * sizeof(float) + sizeof(float2));
}

cudaError_t launch_paged_attention_int4(const PagedAttnArgs& a, cudaStream_t s) {
  using namespace paged4;
  const int nt = tiles_of(a.c.dim, a.tokens * (a.heads / a.c.kv_heads));
  switch (a.c.dim * 8 + nt) {
    case 64 * 8 + 1: return launch<64, 1>(a, s);
    case 64 * 8 + 2: return launch<64, 2>(a, s);
    case 64 * 8 + 3: return launch<64, 3>(a, s);
    case 64 * 8 + 4: return launch<64, 4>(a, s);
    case 128 * 8 + 1: return launch<128, 1>(a, s);
    case 128 * 8 + 2: return launch<128, 2>(a, s);
    case 128 * 8 + 3: return launch<128, 3>(a, s);
    case 128 * 8 + 4: return launch<128, 4>(a, s);
    case 256 * 8 + 1: return launch<256, 1>(a, s);
    case 256 * 8 + 2: return launch<256, 2>(a, s);
    case 512 * 8 + 1: return launch<512, 1>(a, s);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace omni
