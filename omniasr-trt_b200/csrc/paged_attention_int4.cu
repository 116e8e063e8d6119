// Attention of each row's newest tokens over a paged cache held in 4 bits (bf16 queries, head_dim 64 to 512).
//
// Query column c < T G of a unit (row, kv head; G = heads / kv_heads, column c = token c / G, head kv G + c % G) sees keys
// [0, lengths[b] + c / G). A key costs 2 (D / 2 + D / 16) bytes and nothing else is read more than once, so the bound is HBM, and next
// to it the instructions that make operands of the codes: 2 D codes a key, about 0.17 keys a clock and SM at HBM's rate, with 64
// integer lanes a clock. Hence:
//
// * The codes never become a tile in shared memory (for tcgen05 they would be written and read there in two or four times their
//   bytes, with 128 bytes a clock): each lane dequantises in registers what it feeds to mma.sync itself, whose rate (a
//   product of 16 x 8 x 16 in two clocks) is more than twice what is needed. The cache's order of codes
//   (int4.cuh) makes a lane's share of a vector one run of 16 bytes (K) or 8 (V).
// * S^T = K Q^T in fp16, 16 keys x 8 columns a step: a code masked out of its word is, read as fp16, the subnormal c 2^-24 (16 c 2^-24
//   four bits up), exact, so a word of 8 codes takes four ands and a shift. The queries, scaled by a power of two per column
//   (largest value 2^14 and more; exact but for values under 2^-27 of it), carry the factors. The sums start from -8 sum q, which is the
//   codes' offset, and every group's sum is scaled in fp32.
// * O^T = V^T P^T in fp16: two keys' codes of a dim are the halves of a word after one byte permutation, and a code masked out of it
//   is the subnormal c 2^-24 (16 c 2^-24 four bits up), exact; the offset is a second product, with constants. The scales go onto
//   the probabilities in fp32, before these are rounded, once, to fp16 and turned by movmatrix. Two things keep them in fp16's range.
//   A column's weights 2^(x - m) may grow to 2^14, then m is raised so that the largest is 2^12. And every group of 32 dims has a unit, a
//   power of two that a warp's accumulators of the group count in, which the scales of a block lie between 2^-11 and 2^2 of; a block
//   whose scales do not moves the unit (and the accumulators with it), and one with scales too far apart for any unit is summed in
//   fp32 on the CUDA cores (four to six times as long). So a weight is rounded by 2^-11 of itself or, if that is more, by 2^-26 of the
//   row's largest (half of fp16's smallest step, 2^-25, is 2^-37 of the largest weight in units of at most 2^11 times the key's own
//   scale), whatever the scales are.
// * Warps are independent: each takes blocks of 16 or 32 keys of the CTA's share with a maximum, a sum and an accumulator of
//   its own, and copies its next blocks asynchronously into a ring of its own; no barrier in the loop. At a unit's end the CTA's
//   warps join through shared memory.
// * All blocks of all units are cut evenly between the CTAs. A unit that is cut leaves parts in the workspace; the CTA that
//   publishes last joins them in the order of the keys, so a call repeats its bits.
//
// Measured (graph of five calls, L2 flushed before): 48 rows of 61 to 4093 keys, 32 heads on 8 of 128, 50 us (e4m3 pages 65); 48 rows of
// 4096 keys 75 us (e4m3 79); 32 rows of 1400 to 1600 keys, 8 heads of 512, 88 us (e4m3 79: eight warps an SM are too few there).
//
// What a column does not see has weight zero: its score is masked before the exponential, and its group scales (which may be
// NaN) are masked out of the products; keys past the row's last are not read.

#include <math.h>

#include <cuda_fp16.h>

#include <algorithm>

#include "attention.cuh"
#include "common.cuh"
#include "int4.cuh"
#include "paged.cuh"

namespace omni {
namespace paged4 {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr float kMost = 14.f, kGoal = 12.f;  // log2 of a weight: the most, and the largest when m is raised
// Units: a block's scales have exponents from unit - kBelow to unit + kAbove, so that a product is at most 2^kMost (4 - 2^-6) = 65,280
// (a bf16 number under 4), which fp16 holds.
// Units stay from kUnitLeast to kUnitMost (2^-unit and what the join multiplies by are fp32 numbers), and at most kFall below the highest
// that the warp's unit had (an accumulator, under 2^50 with 2^31 keys, is scaled up by no more). They start where groups whose largest
// values are 2^-6 to 2^7 need no other (32 rows of 1400 to 1600 keys, 8 heads of 512, keys' sizes spread by a factor of 2: from 2^0 97 us, from 2^2 82).
constexpr int kAbove = 1, kBelow = 11, kUnitFirst = 2, kUnitLeast = -100, kUnitMost = 110, kFall = 64;
constexpr float kNone = -3e38f;  // a maximum before any score: below what a score can be, and a number, so that nothing needs a case for it
// A unit's start and end (queries, the join of the warps), about 3 us of a CTA, counted as so many blocks in the shares.
constexpr int kStart = 8;

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
  static constexpr int kCtas = DIM == 512 || NT * DIM >= 384 || NT * DIM == 256 && DIM == 64 ? 2 : NT * DIM > 64 ? 3 : 4;  // per SM, for the registers
};

struct Params {
  PagedAttnArgs a;
  int cols, chunks;  // columns of a (row, kv head); units per (row, kv head)
  int grid;
  int page_shift;        // pages of 2^page_shift positions, 16 and more, one behind another in a head's part of under 2^31 bytes; else -1
  uint32_t page_scales;  // bytes of a page's scales
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

// d = a b + c.
OMNI_DEV void mma_f16(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, const uint32_t* b, float c0, float c1, float c2, float c3) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b[0]), "r"(b[1]), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}
// c += a b.
OMNI_DEV void mma_f16(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
OMNI_DEV uint32_t turned(uint32_t x) {  // an 8 x 8 tile of 16-bit values across the warp, transposed
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
OMNI_DEV uint32_t max_abs_bf16x2(uint32_t a, uint32_t b) {  // (of a NaN and a number the number)
  uint32_t r;
  asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a & 0x7fff7fffu), "r"(b & 0x7fff7fffu));
  return r;
}
// Two fp32 as fp16 (lo, hi).
OMNI_DEV uint32_t half2_of(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
OMNI_DEV uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// Whether one of two scales (bf16, relative to their units) is not 0 and outside [2^-kBelow, 2^(kAbove + 1)); of a NaN no.
OMNI_DEV bool outside(uint32_t scales) {
  const uint32_t x = scales & 0x7fff7fffu;
  constexpr uint32_t lo = (127u - kBelow) << 7, hi = (127u + kAbove + 1) << 7;
  auto pair = [](uint32_t u) { return *reinterpret_cast<const __nv_bfloat162*>(&u); };
  return (__hge2_mask(pair(x), pair(hi | hi << 16)) | (__hlt2_mask(pair(x), pair(lo | lo << 16)) & __hgt2_mask(pair(x), pair(0u)))) != 0u;
}

// Where the 16-byte word c of key r's codes lies in a tile: so that a quarter warp's reads (K: 16 bytes of 2 keys x 4 lanes; V, 8
// bytes: 4 keys x 4 lanes) meet all banks. Keys of V lie in the order of its operand, so that a lane's four are 4 apart.
template <int DIM>
OMNI_DEV int k_place(int r, int c) {
  return r * (DIM / 32) + (DIM >= 256 ? c ^ ((r & 1) << 2) : c);
}
OMNI_DEV int v_slot(int r) { return (r & 8) | ((r & 1) << 2) | ((r >> 1) & 3); }
template <int DIM>
OMNI_DEV int v_place(int slot, int c) {
  return slot * (DIM / 32) + (DIM >= 256 ? c ^ ((slot & 3) << 1) : DIM == 128 ? c ^ (slot & 2) : c);
}

// A walk over the units in order. The shares are cut along a line on which a unit takes kStart places and then one per block: the
// blocks of unit (row, head, chunk of columns) are the places [u0, u0 + nb).
struct Walk {
  int64_t u0;
  int row, head, chunk, nb;
  int len, need;  // keys the row's first query sees (at least 0), and its last
};

template <int KEYS>
struct Rows {
  const Params& p;
  int64_t cap;
  OMNI_DEV explicit Rows(const Params& q) : p(q), cap((int64_t)q.a.table_width * q.a.c.page) {}
  OMNI_DEV int64_t look(int row, Walk& w) const {
    const int64_t given = p.a.lengths[row], len = min(given, cap);
    w.need = (int)max((int64_t)0, min(cap, len + p.a.tokens - 1));
    w.len = (int)max(len, (int64_t)-p.a.tokens);
    w.nb = (w.need + KEYS - 1) / KEYS;
    return given;
  }
  OMNI_DEV static int places(int nb) { return nb ? nb + kStart : 0; }
  OMNI_DEV void next(Walk& w) const {
    w.u0 += w.nb + kStart;
    if (++w.chunk < p.chunks) return;
    w.chunk = 0;
    if (++w.head < p.a.c.kv_heads) return;
    w.head = 0;
    while (++w.row < p.a.rows) {
      look(w.row, w);
      if (w.nb) break;
    }
  }
};

// a / b of numbers that are mostly small (a >= 0, b > 0).
OMNI_DEV int64_t quotient(int64_t a, int64_t b) {
  return ((a | b) >> 32) == 0 ? (int64_t)((uint32_t)a / (uint32_t)b) : a / b;
}

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
  int k_lane, v_lane;  // this lane's words in a tile: of key g in K, of slot t in V (block b's: ^ 64 b)

  float o[C::kBlocks * C::kGroups][2][NT][4];
  float m[NT][2], l[NT][2], qs[NT][2];  // what is taken off the scores, sums of weights, the scores' factors
  static constexpr int kWordsS = DIM / 64;  // 32-bit words of a vector's scales
  uint32_t down[kWordsS];                   // 2^-unit of each group (bf16, as the scales lie)
  int highest;                              // of the units so far

  OMNI_DEV Kernel(const Params& q, char* s) : p(q), smem(s) {
    lane = threadIdx.x & 31;
    warp = threadIdx.x >> 5;
    g = lane >> 2;
    t = lane & 3;
    ring = smem_addr(smem) + C::kRing + warp * C::kStages * C::kStage;
    q_at = smem_addr(smem) + C::kQ + lane * 16;
    init_at = smem_addr(smem) + C::kInit + t * 8;
    k_lane = DIM == 64 ? g * C::kRow + t * 8 : k_place<DIM>(g, t) * 16;
    v_lane = DIM == 64 ? t * C::kRow + g * 4 : v_place<DIM>(t, g >> 1) * 16 + (g & 1) * 8;
  }

  // ---- loads: block n (of the walk's unit) into a stage of the ring

  // Pages of whole tiles of 16 keys whose positions lie one behind another (p.page_shift >= 0): a tile is one run of bytes of K,
  // V and their scales each. What a lane needs of a unit to copy its part of any tile, and the pages of the next block:
  struct Source {
    const char *k, *v, *scale;  // where the head's part of page 0 starts, this lane's bytes of it (scales: V's in the upper half warp)
    const int32_t* table;
    int id[C::kMt];
  };
  static constexpr int kCopy = C::kScale < 16 ? C::kScale : 16;  // bytes of scales per copy

  OMNI_DEV void look_up(Source& f, const Walk& w, int block) const {  // (past the row's end: its last page)
    const int last = (w.need - 1) >> p.page_shift;
#pragma unroll
    for (int tile = 0; tile < C::kMt; ++tile) f.id[tile] = *(f.table + min((block * C::kKeys + tile * 16) >> p.page_shift, last));
  }
  OMNI_DEV void open(Source& f, const Walk& w, int block) const {
    if (p.page_shift < 0) return;
    const PagedAttnArgs& a = p.a;
    f.k = reinterpret_cast<const char*>(a.c.k) + w.head * a.c.s_head + lane * 16;
    f.v = reinterpret_cast<const char*>(a.c.v) + w.head * a.c.s_head + lane * 16;
    const bool upper = C::kScale <= 16 && lane >= 16;
    f.scale = reinterpret_cast<const char*>(upper ? a.c.v_scale : a.c.k_scale) + ((int64_t)w.head << p.page_shift) * C::kScale +
              (C::kScale <= 16 ? lane & 15 : lane) * kCopy;
    f.table = a.table + w.row * a.table_stride;
    look_up(f, w, block);
  }

  // A block of whole tiles; false (and nothing done) where a tile is not whole or its page number is none.
  OMNI_DEV bool fetch_whole(Source& f, const Walk& w, int block, int stage) const {
    bool ok = (block + 1) * C::kKeys <= w.need;
#pragma unroll
    for (int tile = 0; tile < C::kMt; ++tile) ok = ok && (unsigned)f.id[tile] < (unsigned)p.a.c.pages;
    if (!ok) return false;
    const uint32_t kd = ring + stage * C::kStage, vd = kd + C::kKeys * C::kRow, ksd = vd + C::kKeys * C::kRow;
    const PagedAttnArgs& a = p.a;
    constexpr int N = 16 * C::kRow / 512;  // copies of 16 bytes per lane and tile
    constexpr int CPR = C::kRow / 16;
#pragma unroll
    for (int tile = 0; tile < C::kMt; ++tile) {
      const uint32_t off = (block * C::kKeys + tile * 16) & ((1 << p.page_shift) - 1);
      const uint64_t at = (uint64_t)(uint32_t)f.id[tile] * (uint32_t)a.c.s_page + off * C::kRow;
      const char *k = f.k + at, *v = f.v + at;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int r = (lane + 32 * i) / CPR, c = lane % CPR;
        copy_async(kd + (tile * 16 * CPR + k_place<DIM>(r, c)) * 16, k + i * 512, true, 16);
        copy_async(vd + (tile * 16 * CPR + v_place<DIM>(v_slot(r), c)) * 16, v + i * 512, true, 16);
      }
      const char* scale = f.scale + ((uint64_t)(uint32_t)f.id[tile] * p.page_scales + off * C::kScale);
      if constexpr (C::kScale <= 16) {
        copy_async(ksd + (lane >= 16 ? C::kKeys * C::kScale : 0) + (tile * 16 + (lane & 15)) * C::kScale, scale, true, kCopy);
      } else {
        const int64_t apart = reinterpret_cast<const char*>(a.c.v_scale) - reinterpret_cast<const char*>(a.c.k_scale);
        copy_async(ksd + tile * 16 * C::kScale + lane * 16, scale, true, 16);
        copy_async(ksd + (C::kKeys + tile * 16) * C::kScale + lane * 16, scale + apart, true, 16);
      }
    }
    return true;
  }

  // Any page size: each key's page number by a lane of its own.
  OMNI_DEV void fetch_keys(const Walk& w, int j0, int stage) {
    const PagedAttnArgs& a = p.a;
    const int h = w.head;
    const uint32_t kd = ring + stage * C::kStage, vd = kd + C::kKeys * C::kRow, ksd = vd + C::kKeys * C::kRow,
                   vsd = ksd + C::kKeys * C::kScale;
    const int jr = j0 + (lane < C::kKeys ? lane : 0);
    bool live = false;
    int64_t at = 0, sat = 0;
    if (jr < w.need) {
      const int pi = (int)((uint32_t)jr / (uint32_t)a.c.page), off = jr - pi * a.c.page;
      const int id = a.table[w.row * a.table_stride + pi];
      live = (unsigned)id < (unsigned)a.c.pages;
      if (live) {
        at = (int64_t)id * a.c.s_page + h * a.c.s_head + off * a.c.s_pos;
        sat = (((int64_t)id * a.c.kv_heads + h) * a.c.page + off) * C::kScale;
      } else if (lane < C::kKeys) {
        raise_status(a.status, kStatusIndex);
      }
    }
    constexpr int CPR = C::kRow / 16, N = C::kKeys * CPR / 32;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int r = (lane + 32 * i) / CPR, c = lane % CPR, rr = r & 15;
      const bool on = __shfl_sync(0xffffffffu, live, r);
      const int64_t in = __shfl_sync(0xffffffffu, at, r) + (on ? c * 16 : 0);
      copy_async(kd + ((r & ~15) * CPR + k_place<DIM>(rr, c)) * 16, reinterpret_cast<const char*>(a.c.k) + in, on, 16);
      copy_async(vd + ((r & ~15) * CPR + v_place<DIM>(v_slot(rr), c)) * 16, reinterpret_cast<const char*>(a.c.v) + in, on, 16);
    }
    constexpr int CS = C::kScale < 16 ? C::kScale : 16, SPR = C::kScale / CS;
    static_assert(C::kKeys * SPR <= 32, "a copy per lane");
    const int r = lane / SPR % C::kKeys, c = lane % SPR;
    const bool on = __shfl_sync(0xffffffffu, live, r);
    const int64_t in = __shfl_sync(0xffffffffu, sat, r) + (on ? c * CS : 0);
    if (lane < C::kKeys * SPR) {
      copy_async(ksd + r * C::kScale + c * CS, reinterpret_cast<const char*>(a.c.k_scale) + in, on, CS);
      copy_async(vsd + r * C::kScale + c * CS, reinterpret_cast<const char*>(a.c.v_scale) + in, on, CS);
    }
  }

  // Block `block` of the unit into a stage; `then`: the one that comes next, if it is the unit's.
  OMNI_DEV void fetch(Source& f, const Walk& w, int block, int then, int stage) {
    if (p.page_shift < 0 || !fetch_whole(f, w, block, stage)) fetch_keys(w, block * C::kKeys, stage);
    if (p.page_shift >= 0) look_up(f, w, then);
  }

  // ---- a unit's queries

  OMNI_DEV int limit(const Walk& w, int col) const {  // keys a column sees; -1: no such column
    const int gr = p.a.heads / p.a.c.kv_heads;
    return col < p.cols ? max(0, min(w.need, w.len + col / gr)) : -1;
  }
  OMNI_DEV int64_t query_row(const Walk& w, int col) const {
    const int gr = p.a.heads / p.a.c.kv_heads, tok = col / gr;
    return ((int64_t)w.row * p.a.tokens + tok) * p.a.heads + w.head * gr + (col - tok * gr);
  }

  // A warp's columns of a unit: their words in flight ...
  static constexpr int kPer = C::kCols / kWarps, kWords = DIM > 256 ? 2 : 1;  // columns per warp, words of 8 dims per lane
  OMNI_DEV void read_queries(const Walk& w, uint4 (&u)[kPer][kWords]) const {
    const int c0 = w.chunk * C::kCols;
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      const int col = c0 + warp + k * kWarps;
      const bool on = col < p.cols;
      const uint4* src = reinterpret_cast<const uint4*>(reinterpret_cast<const __nv_bfloat16*>(p.a.q) + (on ? query_row(w, col) * DIM : 0));
#pragma unroll
      for (int v = 0; v < kWords; ++v) {
        const int word = v * 32 + lane;
        u[k][v] = on && word * 8 < DIM ? src[word] : make_uint4(0u, 0u, 0u, 0u);
      }
    }
  }

  // ... and as fp16 operands in the order of the codes, with the sums' start per group and the factor of the scores. (A column with
  // an infinity or a NaN comes out NaN through its sums' start.)
  OMNI_DEV void store_queries(const Walk& w, const uint4 (&u)[kPer][kWords]) {
    const int c0 = w.chunk * C::kCols;
    float* init = reinterpret_cast<float*>(smem + C::kInit);
    float* factor = reinterpret_cast<float*>(smem + C::kLim);
    int* lims = reinterpret_cast<int*>(smem + C::kLim) + C::kCols;
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      const int col = warp + k * kWarps;
      uint32_t top2 = 0u;
#pragma unroll
      for (int v = 0; v < kWords; ++v)
        top2 = max_abs_bf16x2(top2, max_abs_bf16x2(max_abs_bf16x2(u[k][v].x, u[k][v].y), max_abs_bf16x2(u[k][v].z, u[k][v].w)));
      const uint32_t top = __reduce_max_sync(0xffffffffu, max(top2 & 0xffffu, top2 >> 16));
      const int e = top == 0u ? 0 : max(-112, (int)(top >> 7) - 127);
      const float up = __uint_as_float((uint32_t)(14 - e + 127) << 23);
#pragma unroll
      for (int v = 0; v < kWords; ++v) {
        const int word = v * 32 + lane;
        float x[8];
        Elem<__nv_bfloat16>::unpack(u[k][v], x);
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          x[i] *= up;
          sum += x[i];
        }
        uint32_t b[4];  // nibbles i and i + 4 of the word; odd ones stand for 16 c
#pragma unroll
        for (int i = 0; i < 4; ++i) b[i] = (i & 1) ? half2_of(x[i] * 0.0625f, x[i + 4] * 0.0625f) : half2_of(x[i], x[i + 4]);
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        if (word * 8 < DIM) {
          const int group = word >> 2;
          reinterpret_cast<uint4*>(smem + C::kQ)[(group * NT + (col >> 3)) * 32 + (col & 7) * 4 + (word & 3)] = make_uint4(b[0], b[1], b[2], b[3]);
          if ((word & 3) == 0) init[group * C::kCols + col] = sum * (-8.f * 0x1p-24f);
        }
      }
      if (lane == 0) {
        factor[col] = p.a.scale * kLog2e * 0x1p10f * __uint_as_float((uint32_t)(e + 127) << 23);
        lims[col] = limit(w, c0 + col);
      }
    }
  }

  OMNI_DEV void start_unit() {
    highest = kUnitFirst;
#pragma unroll
    for (int i = 0; i < kWordsS; ++i) down[i] = (uint32_t)(127 - kUnitFirst) << 7 | (uint32_t)(127 - kUnitFirst) << 23;
    const float* factor = reinterpret_cast<const float*>(smem + C::kLim);
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        m[n][i] = kNone;
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

  // ---- the groups' units, and blocks that have none

  static constexpr int kLook = C::kKeys * C::kScale / 128;  // words of a block's scales per lane: a key's, half a key's from 256 dims on

  // Whether a block's scales (a lane's words of them) lie within reach of the units.
  OMNI_DEV bool in_units(const uint32_t (&w)[kLook]) const {
    bool off = false;
#pragma unroll
    for (int i = 0; i < kLook; ++i) off |= outside(mul_bf16x2(w[i], DIM >= 256 && (lane & 1) ? down[(kWordsS - kLook) + i] : down[i]));
    return !__any_sync(0xffffffffu, off);
  }
  OMNI_DEV bool in_units(int stage) const {
    uint32_t w[kLook];
    load_words<kLook>(w, ring + stage * C::kStage + 2 * C::kKeys * C::kRow + C::kKeys * C::kScale + lane * kLook * 4);
    return in_units(w);
  }

  // Units that a block with the scales w (a lane's words of them) can be counted in, the nearest to those so far; the accumulators go
  // along. True: there are none, some group's scales are too far apart.
  OMNI_DEV bool set_units(const uint32_t (&w)[kLook]) {
    uint32_t top[kLook], least[kLook];  // bits of the largest and of the least number that is not 0; halves are groups
#pragma unroll
    for (int i = 0; i < kLook; ++i) {
      top[i] = 0u;
      least[i] = 0u;
#pragma unroll
      for (int sh = 0; sh < 32; sh += 16) {
        const uint32_t x = (w[i] >> sh) & 0x7fffu;
        const bool number = x != 0u && x < 0x7f80u;
        top[i] |= (number ? x : 0u) << sh;
        least[i] |= (number ? x : 0x7f80u) << sh;
      }
#pragma unroll
      for (int o = DIM >= 256 ? 2 : 1; o < 32; o <<= 1) {
        top[i] = __vmaxu2(top[i], __shfl_xor_sync(0xffffffffu, top[i], o));
        least[i] = __vminu2(least[i], __shfl_xor_sync(0xffffffffu, least[i], o));
      }
    }
    bool wild = false;
    int up = highest;
#pragma unroll
    for (int j = 0; j < kWordsS; ++j) {
      const uint32_t tw = __shfl_sync(0xffffffffu, top[j % kLook], j / kLook), lw = __shfl_sync(0xffffffffu, least[j % kLook], j / kLook);
      uint32_t next = 0u;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int t = (int)((tw >> (16 * half)) & 0xffffu) >> 7, s = (int)((lw >> (16 * half)) & 0xffffu) >> 7;  // exponents + 127
        const int now = 127 - (int)(((down[j] >> (16 * half)) & 0xffffu) >> 7);
        int unit = now;
        if (t != 0) {  // (else no scale but zeros and numbers too small for one)
          const int lo = t - 127 - kAbove, hi = s - 127 + kBelow;  // units that the block can be counted in
          if (unit < lo) unit = max(lo, min(lo + 1, hi));  // (with room for scales twice as large)
          else if (unit > hi && hi >= lo) unit = hi;
          unit = min(max(max(unit, highest - kFall), kUnitLeast), kUnitMost);
          wild |= unit < lo || unit > hi;
          up = max(up, unit);
        } else if ((tw >> (16 * half)) & 0xffffu) {
          wild = true;
        }
        next |= (uint32_t)(127 - unit) << (7 + 16 * half);
        const float f = ex2((float)(now - unit));
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int c = 0; c < 4; ++c) o[2 * j + half][i][n][c] *= f;
      }
      down[j] = next;
    }
    highest = up;
    return wild;
  }

  // What the 16 keys from `key` of a block on add, in fp32: e[n][2 h + i] is the weight of key g + 8 h for column 2 t + i of tile n.
  OMNI_DEV void add_values(const float (&e)[NT][4], int key, int j0, uint32_t vd, uint32_t vsd) {
    const int* lims = reinterpret_cast<const int*>(smem + C::kLim) + C::kCols;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll 1
      for (int r = 0; r < 8; ++r) {
        const int at = key + 8 * h + r, slot = v_slot(8 * h + r);
        float p[NT][2];
        bool hidden[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            p[n][i] = __shfl_sync(0xffffffffu, e[n][2 * h + i], r * 4 + t);
            hidden[n][i] = j0 + at >= lims[n * 8 + 2 * t + i];
          }
#pragma unroll
        for (int b = 0; b < C::kBlocks; ++b) {
          uint32_t vw[W2], vs[W2];  // dims 4 g .. of each group, and the groups' scales
          load_words<W2>(vw, vd + key * C::kRow + (DIM == 64 ? slot * C::kRow + g * 4 : v_place<DIM>(slot, b * 4 + (g >> 1)) * 16 + (g & 1) * 8));
          load_words<W2>(vs, vsd + at * C::kScale + b * 8);
#pragma unroll
          for (int gr = 0; gr < C::kGroups; ++gr) {
            const int sh = 16 * (gr & 1);
            const float s = bf16_value((vs[gr >> 1] >> sh) & 0xffffu) * bf16_value((down[b * W2 + (gr >> 1)] >> sh) & 0xffffu);
            float c[4];
            int4_values(vw[gr >> 1] >> sh, 1.f, c);
            float(&x)[2][NT][4] = o[b * C::kGroups + gr];
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                const float y = hidden[n][i] ? 0.f : p[n][i] * s;
                x[0][n][i] = fmaf(y, c[0] * 0x1p-24f, x[0][n][i]);
                x[0][n][i + 2] = fmaf(y, c[1] * 0x1p-20f, x[0][n][i + 2]);
                x[1][n][i] = fmaf(y, c[2] * 0x1p-24f, x[1][n][i]);
                x[1][n][i + 2] = fmaf(y, c[3] * 0x1p-20f, x[1][n][i + 2]);
              }
          }
        }
      }
  }

  // ---- one block. TAIL: some column does not see all of it, or its scales do not fit the units.

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
          if constexpr (C::kGroups == 4)
            load_words<4>(kw[k][e], kd + k * 16 * C::kRow + 8 * e * C::kRow + (k_lane ^ (b * 64)));
          else
            load_words<2>(kw[k][e], kd + k * 16 * C::kRow + 8 * e * C::kRow + k_lane);
          load_words<W2>(ks[k][e], ksd + g * C::kScale + (k * 16 + 8 * e) * C::kScale + b * 8);
        }
#pragma unroll
      for (int gr = 0; gr < C::kGroups; ++gr) {
        const int group = b * C::kGroups + gr;
        uint32_t lo[C::kMt][4], hi[C::kMt][4];  // of keys g and g + 8 the nibbles (0, 4), (1, 5), (2, 6), (3, 7)
#pragma unroll
        for (int k = 0; k < C::kMt; ++k) {
          const uint32_t x = kw[k][0][gr], y = kw[k][1][gr];
          lo[k][0] = x & 0x000f000fu, lo[k][1] = x & 0x00f000f0u, lo[k][2] = (x >> 8) & 0x000f000fu, lo[k][3] = (x >> 8) & 0x00f000f0u;
          hi[k][0] = y & 0x000f000fu, hi[k][1] = y & 0x00f000f0u, hi[k][2] = (y >> 8) & 0x000f000fu, hi[k][3] = (y >> 8) & 0x00f000f0u;
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          uint32_t q[4], start[2];
          load_words<4>(q, q_at + (group * NT + n) * 512);
          load_words<2>(start, init_at + (group * C::kCols + n * 8) * 4);
          const float i0 = __uint_as_float(start[0]), i1 = __uint_as_float(start[1]);
#pragma unroll
          for (int k = 0; k < C::kMt; ++k) {
            float h[4], c[4];
            mma_f16(h, lo[k][0], hi[k][0], lo[k][1], hi[k][1], q, i0, i1, i0, i1);
            mma_f16(c, lo[k][2], hi[k][2], lo[k][3], hi[k][3], q + 2, h[0], h[1], h[2], h[3]);
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
    auto masked = [&](int k, int n, int i) {
      return TAIL && j0 + k * 16 + g + (i & 2) * 4 >= lims[n * 8 + 2 * t + (i & 1)];
    };
    bool wild = false;
    if constexpr (TAIL) {
      uint32_t w[kLook];
      load_words<kLook>(w, vsd + lane * kLook * 4);
      if (!in_units(w)) wild = set_units(w);
    }
    // Scores less m, masked.
    bool raise = false;
    float d[C::kMt][NT][4];
#pragma unroll
    for (int k = 0; k < C::kMt; ++k)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          d[k][n][i] = masked(k, n, i) ? -INFINITY : fmaf(s[k][n][i], qs[n][i & 1], -m[n][i & 1]);
          raise |= d[k][n][i] > kMost;
        }
    if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float top = -INFINITY;
#pragma unroll
          for (int k = 0; k < C::kMt; ++k)
#pragma unroll
            for (int e = i; e < 4; e += 2)
              if (!masked(k, n, e)) top = fmaxf(top, s[k][n][e] * qs[n][i]);
#pragma unroll
          for (int w = 4; w < 32; w <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
          top = fmaxf(m[n][i], top - kGoal);
          const float f = ex2(m[n][i] - top);
          m[n][i] = top;
#pragma unroll
          for (int k = 0; k < C::kMt; ++k)
#pragma unroll
            for (int e = i; e < 4; e += 2)
              if (!masked(k, n, e)) d[k][n][e] = fmaf(s[k][n][e], qs[n][i], -top);
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
      float e[NT][4];
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          e[n][i] = ex2(d[k][n][i]);
          l[n][i & 1] += e[n][i];
        }
      if (TAIL && wild) {
        add_values(e, k * 16, j0, vd, vsd);
        continue;
      }
#pragma unroll
      for (int b = 0; b < C::kBlocks; ++b) {
        uint32_t vw[4][W2], vs[2][W2];  // codes of keys 2 t, 2 t + 1, 2 t + 8, 2 t + 9 (slots t, t + 4, ...); scales of keys g, g + 8
#pragma unroll
        for (int i = 0; i < 4; ++i) load_words<W2>(vw[i], vd + k * 16 * C::kRow + 4 * i * C::kRow + (v_lane ^ (b * 64)));
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          load_words<W2>(vs[i], vsd + g * C::kScale + (k * 16 + 8 * i) * C::kScale + b * 8);
#pragma unroll
          for (int j = 0; j < W2; ++j) vs[i][j] = mul_bf16x2(vs[i][j], down[b * W2 + j]);  // (exact)
        }
#pragma unroll
        for (int gr = 0; gr < C::kGroups; ++gr) {
          const uint32_t sel = (gr & 1) ? 0x7632u : 0x5410u;
          const uint32_t za = __byte_perm(vw[0][gr >> 1], vw[1][gr >> 1], sel), zb = __byte_perm(vw[2][gr >> 1], vw[3][gr >> 1], sel);
          const uint32_t a0[4] = {za & 0x000f000fu, za & 0x00f000f0u, zb & 0x000f000fu, zb & 0x00f000f0u};
          const uint32_t a1[4] = {(za >> 8) & 0x000f000fu, (za >> 8) & 0x00f000f0u, (zb >> 8) & 0x000f000fu, (zb >> 8) & 0x00f000f0u};
          const uint32_t eight[4] = {0x80088008u, 0x80808080u, 0x80088008u, 0x80808080u};  // -8 in each place
          const uint32_t w0 = vs[0][gr >> 1], w1 = vs[1][gr >> 1];
          const float s0 = __uint_as_float((gr & 1) ? w0 & 0xffff0000u : w0 << 16), s1 = __uint_as_float((gr & 1) ? w1 & 0xffff0000u : w1 << 16);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            auto weight = [&](int i) { return masked(k, n, i) ? 0.f : e[n][i] * ((i & 2) ? s1 : s0); };  // (a hidden scale may be NaN)
            const uint32_t b0 = turned(half2_of(weight(0), weight(1))), b1 = turned(half2_of(weight(2), weight(3)));
            float(&x)[2][NT][4] = o[b * C::kGroups + gr];
            mma_f16(x[0][n], a0, b0, b1);
            mma_f16(x[1][n], a1, b0, b1);
            mma_f16(x[0][n], eight, b0, b1);
            mma_f16(x[1][n], eight, b0, b1);
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
    const int c0 = w.chunk * C::kCols;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int k = 4; k < 32; k <<= 1) l[n][i] += __shfl_xor_sync(0xffffffffu, l[n][i], k);
        if (g == 0) ml[warp * C::kCols + n * 8 + 2 * t + i] = make_float2(m[n][i], l[n][i]);
      }
    __syncthreads();
    if (threadIdx.x < C::kCols) {  // a column's maximum and sum; ml becomes (the warps' factors, the sum)
      const int col = threadIdx.x;
      float2 s[kWarps];
      float top = kNone, sum = 0.f;
#pragma unroll
      for (int k = 0; k < kWarps; ++k) {
        s[k] = ml[k * C::kCols + col];
        top = fmaxf(top, s[k].x);
      }
      top += kMost;  // (weights of at most 1, so that values up to the type's largest do not pass fp32's)
#pragma unroll
      for (int k = 0; k < kWarps; ++k) {
        s[k].x = ex2(s[k].x - top);
        sum = fmaf(s[k].y, s[k].x, sum);
      }
#pragma unroll
      for (int k = 0; k < kWarps; ++k) ml[k * C::kCols + col] = make_float2(s[k].x, sum);
      if (part >= 0 && c0 + col < p.cols) p.part_ml[(int64_t)part * C::kCols + col] = make_float2(top, sum);
    }
    __syncthreads();
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      if (c0 + n * 8 >= p.cols) break;
      constexpr float kHigh = 0x1p-14f;  // 2^-kMost; more only in a column whose scores are all -inf, where a unit's 2^110 would make it infinite
      const float f[2] = {fminf(ml[warp * C::kCols + n * 8 + 2 * t].x, kHigh), fminf(ml[warp * C::kCols + n * 8 + 2 * t + 1].x, kHigh)};
      const float low[2] = {f[0] * 0x1p24f, f[1] * 0x1p24f}, high[2] = {f[0] * 0x1p20f, f[1] * 0x1p20f};  // (by the dim's nibble)
#pragma unroll
      for (int b = 0; b < C::kBlocks; ++b) {
#pragma unroll
        for (int gr = 0; gr < C::kGroups; ++gr) {
          const uint32_t exp = ((down[b * W2 + (gr >> 1)] >> (16 * (gr & 1))) & 0xffffu) >> 7;  // 127 - unit
          const float unit = __uint_as_float((254u - exp) << 23);
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float(&x)[2][NT][4] = o[b * C::kGroups + gr];
            const float lo = low[i] * unit, hi = high[i] * unit;
            *reinterpret_cast<float4*>(join + (warp * 8 + 2 * t + i) * C::kPitch + gr * 32 + g * 4) =
                make_float4(x[0][n][i] * lo, x[0][n][i + 2] * hi, x[1][n][i] * lo, x[1][n][i + 2] * hi);
          }
        }
        __syncthreads();
        constexpr int Q4 = C::kGroups * 8;  // float4 of a column
#pragma unroll
        for (int e = threadIdx.x; e < 8 * Q4; e += kThreads) {
          const int col = e / Q4, d = e % Q4 * 4;
          if (c0 + n * 8 + col < p.cols) {
            float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int k = 0; k < kWarps; ++k) {
              const float4 y = *reinterpret_cast<const float4*>(join + (k * 8 + col) * C::kPitch + d);
              x.x += y.x, x.y += y.y, x.z += y.z, x.w += y.w;
            }
            if (part < 0)
              write_out(w, c0 + n * 8 + col, b * 128 + d, x, ml[n * 8 + col].y);
            else
              *reinterpret_cast<float4*>(p.part_o + ((int64_t)part * C::kCols + n * 8 + col) * DIM + b * 128 + d) = x;
          }
        }
        __syncthreads();
      }
    }
  }

  // The parts of a unit cut between the CTAs first .. last, in their order. A CTA's part of a unit that starts before its share is
  // its slot 0, of one that starts in it slot 1.
  OMNI_DEV void join_parts(const Walk& w, int first, int last) {
    const int c0 = w.chunk * C::kCols, cols = min(C::kCols, p.cols - c0);
    float2* ml = reinterpret_cast<float2*>(smem + C::kMl);  // per column the maximum and the sum
    auto at = [&](int c, int col) { return (int64_t)(2 * c + (c == first)) * C::kCols + col; };
    for (int col = warp; col < cols; col += kWarps) {
      float top = kNone, sum = 0.f;
      for (int c = first + lane; c <= last; c += 32) top = fmaxf(top, __ldcg(p.part_ml + at(c, col)).x);
#pragma unroll
      for (int k = 16; k > 0; k >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, k));
      for (int c = first + lane; c <= last; c += 32) {
        const float2 s = __ldcg(p.part_ml + at(c, col));
        sum = fmaf(s.y, ex2(s.x - top), sum);
      }
#pragma unroll
      for (int k = 16; k > 0; k >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, k);
      if (lane == 0) ml[col] = make_float2(top, sum);
    }
    __syncthreads();
    constexpr int Q4 = DIM / 4;
    for (int e = threadIdx.x; e < cols * Q4; e += kThreads) {
      const int col = e / Q4, d = e % Q4 * 4;
      const float2 s = ml[col];
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
      constexpr int U = 8;  // parts in flight
      for (int c = first; c <= last; c += U) {
        float4 y[U];
        float f[U];
#pragma unroll
        for (int k = 0; k < U; ++k) {
          const int64_t from = at(min(c + k, last), col);
          y[k] = __ldcg(reinterpret_cast<const float4*>(p.part_o + from * DIM + d));
          f[k] = __ldcg(p.part_ml + from).x;
        }
#pragma unroll
        for (int k = 0; k < U; ++k)
          if (c + k <= last) {
            const float g = ex2(f[k] - s.x);
            x.x = fmaf(y[k].x, g, x.x), x.y = fmaf(y[k].y, g, x.y), x.z = fmaf(y[k].z, g, x.z), x.w = fmaf(y[k].w, g, x.w);
          }
      }
      write_out(w, c0 + col, d, x, s.y);
    }
    __syncthreads();  // (ml is the next unit's)
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
  int first_nb = 0;  // of the thread's first row
  for (int r = threadIdx.x; r < p.a.rows; r += kThreads) {
    Walk w;
    const int64_t given = rows.look(r, w);
    mine += rows.places(w.nb);
    if (r < kThreads) first_nb = w.nb;
    if (cta == 0 && (given < 0 || given > rows.cap - (p.a.tokens - 1))) raise_status(p.a.status, kStatusIndex);
    if (w.nb == 0 && r % p.grid == cta) {  // no keys: zeros
      const int64_t n = (int64_t)p.a.tokens * p.a.heads * DIM / 8;
      uint4* dst = reinterpret_cast<uint4*>(reinterpret_cast<__nv_bfloat16*>(p.a.out) + (int64_t)r * p.a.tokens * p.a.heads * DIM);
      for (int64_t i = 0; i < n; ++i) dst[i] = make_uint4(0u, 0u, 0u, 0u);
    }
  }
  const int64_t total = block_sum(mine, s_sum) * hcs;
  const int64_t per = max(quotient(total + p.grid - 1, p.grid), (int64_t)(kStart + kWarps));
  const int64_t b0 = min(total, per * cta), b1 = min(total, b0 + per);
  if (b0 >= b1) return;
  // The row that b0 lies in: sums of kThreads rows at a time, then one after another within.
  {
    int64_t before = 0;
    for (int r0 = 0;; r0 += kThreads) {
      Walk w;
      w.nb = first_nb;
      if (r0 > 0) {
        w.nb = 0;
        if (r0 + (int)threadIdx.x < p.a.rows) rows.look(r0 + threadIdx.x, w);
      }
      const int64_t n = (int64_t)rows.places(w.nb) * hcs;
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
  const int unit = (int)quotient(b0 - s_u0, use.nb + kStart);  // of the row
  use.head = unit / p.chunks;
  use.chunk = unit - use.head * p.chunks;
  use.u0 = s_u0 + (int64_t)unit * (use.nb + kStart) + kStart;

  // This warp's blocks of a unit: every kWarps-th from the CTA's first of it on.
  auto from = [&](const Walk& w) { return (int)max((int64_t)0, b0 - w.u0) + k.warp; };
  auto to = [&](const Walk& w) { return (int)min((int64_t)w.nb, b1 - w.u0); };
  Walk get = use;
  int next = from(get), upto = to(get);  // the next block to copy, of `get`'s unit; its end in this share
  int put = 0;                           // its stage
  typename Kernel<DIM, NT>::Source source;
  k.open(source, get, next);
  auto fetch = [&]() {
    if (next >= upto && get.u0 + get.nb < b1) {
      do {
        rows.next(get);
        next = k.warp;
        upto = to(get);
      } while (next >= upto && get.u0 + get.nb < b1);
      k.open(source, get, next);
    }
    if (next < upto) {
      k.fetch(source, get, next, next + kWarps, put);
      next += kWarps;
    }
    copy_commit();
    put = put + 1 == C::kStages ? 0 : put + 1;
  };
  uint4 words[Kernel<DIM, NT>::kPer][Kernel<DIM, NT>::kWords];
  k.read_queries(use, words);
#pragma unroll 1
  for (int i = 0; i < C::kStages - 1; ++i) fetch();

  int take = 0;
  while (use.u0 < b1) {
    k.store_queries(use, words);
    __syncthreads();
    k.start_unit();
    const int end = to(use);
#pragma unroll 1
    for (int n = from(use); n < end; n += kWarps) {
      fetch();  // into the stage that the block before has left
      copy_wait<C::kStages - 1>();
      __syncwarp();
      const int j0 = n * C::kKeys;
      if (j0 + C::kKeys <= use.len && k.in_units(take)) k.template block<false>(take, j0);
      else k.template block<true>(take, j0);
      __syncwarp();
      take = take + 1 == C::kStages ? 0 : take + 1;
    }
    const int first = (int)quotient(use.u0, per), last = (int)quotient(use.u0 + use.nb - 1, per);
    const bool cut = first != last;
    Walk then = use;
    then.u0 = b1;  // (none)
    if (use.u0 + use.nb < b1) {
      then.u0 = use.u0;
      rows.next(then);
      if (then.u0 < b1) k.read_queries(then, words);  // while this unit ends
    }
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
    use = then;
  }
  copy_wait<0>();
}

// Tiles of 8 columns of a unit, which share its reads of the keys and their operands. Two and more at head_dim 128, three and more at 64 and
// two at 256 do not fit the registers and spill (40 to 900 bytes a thread): 16 rows of 5 drafts, 200 to 2000 keys, 32 heads on 8 of
// 128, three tiles a unit, 52 us.
int most_tiles(int dim) { return dim <= 128 ? 4 : dim == 256 ? 2 : 1; }

// One tile per unit where a block per warp covers all tiles' keys all the same (the keys are then read by several units, out of L2):
// a unit's start and end take as long as its tiles are many (5 x 32 queries over 700 keys, 8 kv heads: 16.8 us a call in a
// graph; with three tiles a unit 30.0).
int tiles_of(const PagedAttnArgs& a) {
  const int cols = a.tokens * (a.heads / a.c.kv_heads), dim = a.c.dim;
  const int tiles = (cols + 7) / 8, most = most_tiles(dim);
  const int64_t blocks = ((int64_t)a.table_width * a.c.page + 31) / 32 * a.rows * a.c.kv_heads;
  if (blocks * tiles <= (int64_t)4 * kWarps * device_sm_count()) return 1;
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
  p.page_shift = -1;
  const int64_t scales = (int64_t)a.c.kv_heads * a.c.page * C::kScale;
  const int64_t codes = (int64_t)a.c.page * C::kRow;  // (one page alone has no stride that would bound it)
  if (a.c.page >= 16 && (a.c.page & (a.c.page - 1)) == 0 && a.c.s_pos == C::kRow && a.c.s_page < 0x7fffffff && codes < 0x7fffffff &&
      scales < 0x7fffffff)
    p.page_shift = __builtin_ctz(a.c.page);
  p.page_scales = (uint32_t)scales;
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
  const int nt = tiles_of(a);
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
