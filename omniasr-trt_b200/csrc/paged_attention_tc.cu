// Attention of each row's newest tokens over a paged KV cache on the 5th-generation tensor cores (tcgen05 + TMEM):
// bf16 queries, bf16 or e4m3 pages, head_dim 64, 128, 256 or 512, pages of 8 .. 64 positions (powers of two) or of a multiple
// of 128.
//
// A unit is (row, kv head, chunk of at most 16 query columns): the row's T * G query vectors on that kv head share every
// key. The keys of all units, in 128-key tiles, are cut evenly between the CTAs (one per SM), so that every SM streams
// the same bytes whatever the lengths; a unit cut between CTAs leaves one partial result (maximum, sum, unnormalised
// output) per CTA, and the CTA that finishes last joins them in the order of the keys. Per tile, keys and head dims lie in
// the MMA's M, the query columns in its N:
//   S^T [128 keys x N]  = K [128 x D] Q^T            accumulated over 128-dim chunks
//   P^T = 2^(S^T scale log2e - m)                      one thread per key, m raised only when passed by 2^8
//   O^T [D x N]        += V^T [D x 128 keys] P^T       accumulated in TMEM over the unit's tiles
// K and V chunks stream through one ring of shared-memory slots in the order the MMAs use them (K of tile t + 2 before V of
// tile t), filled by TMA page by page. Two groups of softmax warps take the tiles in turn, each with a maximum, sums and an
// O of its own (the epilogue adds the two up), so that neither waits for the other: with one group, a tile of e4m3 keys took
// 1.1 us to its softmax and 0.75 us to HBM.
//
// e4m3 pages are fed to the tensor core as they are (kind::f8f6f4), at half the bytes of bf16; the query and the
// probabilities become two e4m3 pieces each, in columns of their own: q = 2^e (q1 + q2 / 16), q1 = rn(q 2^-e), q2 =
// rn(16 (q 2^-e - q1)), 4 + 4 significant bits, which hold a bf16 q exactly (down to 2^-22 of the vector's largest) and
// a probability to 8 bits down to 2^-5 (the largest lies between 2^4 and 2^8); below that in steps of 2^-13. Rounded to the
// nearest, the weights of a long flat tail would all be lost, or all counted half or twice (32,767 keys 12.5 nats below one
// other are a tenth of the sum), so the second piece is rounded by a threshold that runs evenly over the keys (dither):
// each weight's error then has mean zero, and a sum of n of them a deviation of at most sqrt(n) 2^-14 against a sum of 2^4 or
// more. The threshold goes by the key's place alone, so equal calls give equal bits; it costs nothing beside the multiply-add.
// The columns are there anyway: N is at least 16. A key's scale 2^ek multiplies its
// scores; a value's scale 2^ev joins the probability as an exponent: w = 2^(x + ev - m), O = sum w v8, l = sum w 2^-ev,
// with m the running maximum of x + ev, so that w stays in e4m3's range whatever the scales are. m is kept 2^4 below the
// maximum, w up to 2^8: the pieces' smallest step is then 2^-17 of a typical largest weight.
//
// What bounds it: HBM. bytes = keys * kv_heads * D * 2 * element (+ 2 scale bytes a key). 48 rows of 4096 keys, 8 kv heads of
// 128, 32 query heads, pages of 64: bf16 127 us (6346 GB/s), e4m3 71.5 us (5690 GB/s); 48 rows of 61 to 4093 in pages of 16,
// bf16, 74 us (5540 GB/s: 9 us of entry, schedule and last join). With 16 query heads to a kv head e4m3 takes 4.2 TB/s (a
// thread's 16 columns of two pieces each spill registers, as those of bf16 at head_dim 256 and 512 do). More than 16 query
// columns on a kv head are several units, each of which reads the keys: 5 tokens of 4 heads 260 us against 131 of one token
// (pages of 16). One row of a few hundred keys is latency: 12 us, of which a unit's ends are about 4000 clocks.

#include <cudaTypedefs.h>
#include <math.h>

#include <cuda_fp8.h>

#include <algorithm>

#include "attention.cuh"
#include "paged.cuh"
#include "tc.cuh"

namespace omni {
namespace pagedtc {

constexpr int BN = 128;            // keys per tile (the MMA's M)
constexpr int kMaxCols = 16;       // query columns per unit
constexpr int kMaxRows = 512;      // rows of one launch
constexpr int kScaleStages = 16;   // tiles of scale bytes in shared memory
constexpr int kMaxSlots = 20;      // ring slots
constexpr int kJoin = 16;          // parts of a cut unit that one CTA joins at a time
constexpr uint32_t kLayoutSw64 = 4;  // 64-byte swizzle (the TMA's CU_TENSOR_MAP_SWIZZLE_64B)
constexpr int kCtlBytes = 6400;    // control block (below)
constexpr float kRaise = 8.f;      // log2: a weight may reach 2^8 before its column's maximum is raised
constexpr float kHead8 = 4.f;      // e4m3: the maximum kept this far (log2) below the largest exponent seen
constexpr float kNone = -1e30f;    // bf16: the maximum of a column whose scores so far are all -inf
constexpr float kBelow = 64.f;     // bf16: a unit starts from maximum 0 unless its scores lie 2^64 below

template <bool FP8, int DIM, int NQT>
struct Cfg {
  static constexpr int CD = DIM < 128 ? DIM : 128;         // head dims of a chunk
  static constexpr int DC = DIM / CD;                      // chunks
  static constexpr int ES = FP8 ? 1 : 2;
  static constexpr int ROWB = CD * ES < 128 ? CD * ES : 128;  // bytes of a box's row, the swizzle's width
  static constexpr int NB = CD * ES / ROWB;                // boxes per chunk
  static constexpr int BOX = BN * ROWB;                    // 128 keys of a box
  static constexpr int GRP = 8 * ROWB;                     // eight of its rows
  static constexpr uint32_t LAYOUT = ROWB == 128 ? kLayoutSw128 : kLayoutSw64;
  static constexpr int SLOT = NB * BOX;                    // one chunk of a K or V tile
  static constexpr int N = FP8 ? (2 * NQT < 16 ? 16 : 2 * NQT) : 16;  // MMA columns
  static constexpr int QBOX = N * ROWB;                    // N rows of the query
  static constexpr int QB = DC * NB * QBOX;                // one query buffer
  static constexpr int PB = BN * N * (FP8 ? 1 : 2);        // one P buffer
  static constexpr int QN = !FP8 && DIM == 128 ? 3 : QB <= 8192 ? 4 : 2;  // query buffers
  static constexpr int FIXED = QN * QB + 2 * PB + 2 * kMaxRows * 4 + 64 + (FP8 ? kScaleStages * 2 * BN : 0);
  static constexpr int FIT = (232448 - kCtlBytes - 1024 - FIXED) / SLOT;
  static constexpr int SLOTS = FIT > kMaxSlots ? kMaxSlots : FIT;
  static constexpr int Q_OFF = SLOTS * SLOT;
  static constexpr int P_OFF = Q_OFF + QN * QB;
  static constexpr int SC_OFF = P_OFF + 2 * PB;            // scale bytes [stage][K, V][128]
  static constexpr int PRE_OFF = SC_OFF + (FP8 ? kScaleStages * 2 * BN : 0);  // int [rows + 1]: tiles before a row
  static constexpr int LEN_OFF = PRE_OFF + (kMaxRows + 16) * 4;               // int [rows]
  static constexpr int BYTES = LEN_OFF + kMaxRows * 4 + 1024;                 // + alignment slack
  static constexpr uint32_t S_COLS = 2 * N;                  // S^T of either softmax group
  static constexpr int OB = S_COLS + 4 * DC * N <= 512 ? 2 : 1;  // O^T buffers (units in turn), per softmax group
  static constexpr uint32_t COLS = S_COLS + 2 * OB * DC * N;
  static constexpr uint32_t TMEM = COLS <= 64 ? 64 : COLS <= 128 ? 128 : COLS <= 256 ? 256 : 512;
  static_assert(SLOTS >= DC, "a tile's V chunks are all resident when its stale rows are cleared");
  static_assert(BYTES + kCtlBytes <= 232448, "shared memory per block");
};

constexpr int kThreads = 512;  // 16 warps: one more would leave 96 registers a thread instead of 128
constexpr int W_LOADK = 4, W_MMA = 5, W_PV = 6, W_LOADV = 7, W_EPI = 8, W_SOFT1 = 12;  // softmax: warps 0-3 and 12-15

struct Params {
  const __nv_bfloat16* q;
  PageCache c;
  const int32_t* table;
  int64_t table_stride;
  const int64_t* lengths;
  __nv_bfloat16* out;
  int rows, tokens, heads, group;  // group: query heads per kv head
  int cols, chunk_cols, chunks;    // query columns per (row, kv head), per unit, units per (row, kv head)
  int cap;                         // keys a row can have
  int page_shift;                  // log2(page) for pages below 128, else -1
  float qscale;
  unsigned* counters;              // [CTA]: parts (or runs of parts) published of the cut unit that begins there;
                                   // [grid + 2 CTA + place]: parts of the run that begins with that slot's
  float* part_o;                   // [2 * CTA + place][column][DIM]; place 0: a unit begun in an earlier CTA, 1: in this one
  float2* part_ml;                 // [2 * CTA + place][column]
  int* status;
};

OMNI_DEV void mma_f8_ss(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// kind::f8f6f4 instruction descriptor: e4m3 A and B (format 0), fp32 accumulator.
constexpr uint32_t idesc_e4m3(int m, int n, int a_mn_major, int b_mn_major) {
  return (1u << 4) | ((uint32_t)a_mn_major << 15) | ((uint32_t)b_mn_major << 16) | ((uint32_t)(n >> 3) << 17) |
         ((uint32_t)(m >> 4) << 24);
}

OMNI_DEV void tmem_st16(uint32_t taddr, const float* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16};" ::"r"(taddr),
      "r"(__float_as_uint(v[0])), "r"(__float_as_uint(v[1])), "r"(__float_as_uint(v[2])), "r"(__float_as_uint(v[3])),
      "r"(__float_as_uint(v[4])), "r"(__float_as_uint(v[5])), "r"(__float_as_uint(v[6])), "r"(__float_as_uint(v[7])),
      "r"(__float_as_uint(v[8])), "r"(__float_as_uint(v[9])), "r"(__float_as_uint(v[10])), "r"(__float_as_uint(v[11])),
      "r"(__float_as_uint(v[12])), "r"(__float_as_uint(v[13])), "r"(__float_as_uint(v[14])), "r"(__float_as_uint(v[15]))
      : "memory");
}

OMNI_DEV bool sync_or(int id, int count, bool pred) {
  uint32_t out;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "barrier.cta.red.or.pred q, %2, %3, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(out)
      : "r"((uint32_t)pred), "r"(id), "r"(count)
      : "memory");
  return out != 0;
}

// Four bytes from global to shared memory, asynchronously; copy_arrive: an arrival once this thread's copies are there.
OMNI_DEV void copy4(void* dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_addr(dst)), "l"(src) : "memory");
}
OMNI_DEV void copy_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_addr(bar)) : "memory");
}

OMNI_DEV unsigned add_acq_rel(unsigned* p) {
  unsigned old;
  asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;" : "=r"(old) : "l"(p) : "memory");
  return old;
}

// 16 columns of this thread's lane without waiting; complete after tmem_wait.
OMNI_DEV void tmem_ld16_async(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
OMNI_DEV void tmem_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// Column totals over a warp of NV values per lane; every lane gets every column's (maximum or sum).
template <int NV, bool MAX>
OMNI_DEV void warp_all(float (&v)[NV]) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const float y = __shfl_xor_sync(0xffffffffu, v[j], o);
      v[j] = MAX ? fmaxf(v[j], y) : v[j] + y;
    }
}

// A CTA's part of one unit: tiles [t0, t1) of the unit's nt.
struct Seg {
  int b, u;        // row; unit within the row (kv head * chunks + chunk)
  int h, col0, ncol;  // the unit's kv head, first query column and columns
  int need;        // keys of the row's last query
  int t0, t1, nt;
  int first;       // first tile of the unit in the global numbering
};

// The segments of a CTA, in order. One division, in init: the roles come here between their tiles.
struct Walk {
  const Params* p;
  const int* pre;   // tiles before each row
  const int* len;
  int pos, end, b, u, nt, t, need;
  OMNI_DEV void row() {  // the row's tiles
    need = min(p->cap, len[b] + p->tokens - 1);
    nt = (need + BN - 1) / BN;
  }
  OMNI_DEV void init(const Params& p_, const int* pre_, const int* len_, int c0, int c1) {
    p = &p_;
    pre = pre_;
    len = len_;
    pos = c0;
    end = c1;
    int lo = 0, hi = p->rows - 1;  // the first row that ends past c0
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (pre[mid + 1] > c0) hi = mid;
      else lo = mid + 1;
    }
    b = lo;
    row();
    const int r = c0 - pre[b];
    u = nt > 0 ? r / nt : 0;
    t = r - u * nt;
  }
  OMNI_DEV bool next(Seg& s) {
    if (pos >= end) return false;
    if (t >= nt) {
      t = 0;
      if (++u >= p->c.kv_heads * p->chunks) {
        u = 0;
        do ++b;
        while (pre[b + 1] <= pos);  // rows without keys have no tiles
        row();
      }
    }
    s.b = b;
    s.u = u;
    s.need = need;
    s.nt = nt;
    s.t0 = t;
    s.t1 = min(nt, t + (end - pos));
    s.first = pos - t;
    s.h = u;
    s.col0 = 0;
    if (p->chunks > 1) {
      s.h = u / p->chunks;
      s.col0 = (u - s.h * p->chunks) * p->chunk_cols;
    }
    s.ncol = min(p->chunk_cols, p->cols - s.col0);
    t = s.t1;
    pos += s.t1 - s.t0;
    return true;
  }
};

// Token and head-of-group of query column `col` (a division only where a unit holds more than one token).
OMNI_DEV void column(const Params& p, int col, int& tok, int& g) {
  tok = p.tokens > 1 ? col / p.group : 0;
  g = col - tok * p.group;
}

struct alignas(16) Ctl {
  uint64_t full[kMaxSlots], empty[kMaxSlots];
  uint64_t s_full[2], s_free[2], p_full[2], pv_done[2], q_full[4], q_empty[4], o_full[2], o_free[2], ml_full[2], ml_free[2];
  uint64_t sc_full[kScaleStages];
  uint64_t drain;
  float red[2][4][kMaxCols];      // [softmax group][warp]: column maxima
  float sum[2][2][4][kMaxCols];   // [segment parity][softmax group][warp]: a finished segment's column sums
  float top[2][2][kMaxCols];      // ... and maxima
  float cq[8][kMaxCols];          // [segment]: score factor per column (scale, log2e, the query's exponent)
  int wsum[kThreads / 32], wmax[kThreads / 32];
  uint32_t tmem_base;
  int abort_flag;
  int loads[kMaxSlots];                  // loads issued into each ring slot
  float2 stat[kJoin][kMaxCols];   // epilogue: maxima and sums of the parts it joins,
  float weight[kJoin][kMaxCols];  // their weights,
  float2 joined[kMaxCols];        // and the whole's
  int last;                       // epilogue: this CTA joins the unit
  int odd;                        // epilogue: some whole unit has a column that is not finite
  int odd_cuts;                   // cut units that this CTA joined and that have one (it has a part of two at most):
  unsigned odd_cut[2];            // row << 16 | unit within the row
};
static_assert(sizeof(Ctl) <= kCtlBytes, "control block");

// The query row of column `col` of row b, kv head h.
OMNI_DEV int64_t query_row(const Params& p, int b, int h, int col, int* t) {
  int g;
  column(p, col, *t, g);
  return ((int64_t)b * p.tokens + *t) * p.heads + h * p.group + g;
}

// BadValues of a row's kv head (a value's scale that is infinite among them), by one warp; a lane looks at a key.
template <bool FP8, int DIM>
__device__ __noinline__ BadValues bad_page_values(const PageCache& c, const int32_t* table, int h, int from, int end) {
  return find_bad(from, end, [&](int j) {
    const int pi = j / c.page, off = j - pi * c.page;
    int64_t id = table[pi];
    if (id < 0 || id >= c.pages) id = 0;
    const int64_t at = id * c.s_page + (int64_t)h * c.s_head + (int64_t)off * c.s_pos;
    const uint4* row = reinterpret_cast<const uint4*>(reinterpret_cast<const unsigned char*>(c.v) + at * (FP8 ? 1 : 2));
    uint32_t any = FP8 && c.v_scale[(id * c.kv_heads + h) * c.page + off] == 255 ? 1u : 0u;
#pragma unroll 8
    for (int i = 0; i < DIM * (FP8 ? 1 : 2) / 16; ++i) {
      const uint4 u = __ldg(row + i);
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {  // a code that is NaN; a half whose exponent bits are all ones
        const uint32_t z = ~w[k] & (FP8 ? 0x7f7f7f7fu : 0x7f807f80u);
        any |= (z - (FP8 ? 0x01010101u : 0x00010001u)) & ~z & (FP8 ? 0x80808080u : 0x80008000u);
      }
    }
    return any != 0u;
  });
}

// One column straight from the formula, by one warp, for the draft columns of must_redo. Rare.
template <bool FP8, int DIM>
__device__ __noinline__ void exact_column(const __nv_bfloat16* q, const PageCache& c, const int32_t* table, int h, int lim,
                                          float qscale, __nv_bfloat16* out) {
  constexpr int NV = DIM / 32;
  const int lane = threadIdx.x & 31;
  float qv[NV], o[NV], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    qv[i] = __bfloat162float(q[i * 32 + lane]);
    o[i] = 0.f;
  }
  auto value = [](const void* base, int64_t at) {
    if (FP8) {
      const __half_raw r = __nv_cvt_fp8_to_halfraw(reinterpret_cast<const uint8_t*>(base)[at], __NV_E4M3);
      return __half2float(*reinterpret_cast<const __half*>(&r));
    }
    return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(base)[at]);
  };
  for (int j = 0; j < lim; ++j) {
    const int pi = j / c.page, off = j - pi * c.page;
    int64_t id = table[pi];
    if (id < 0 || id >= c.pages) id = 0;
    const int64_t at = id * c.s_page + (int64_t)h * c.s_head + (int64_t)off * c.s_pos;
    float ks = 1.f, vs = 1.f;
    if (FP8) {
      const int64_t si = (id * c.kv_heads + h) * c.page + off;
      ks = __uint_as_float((uint32_t)c.k_scale[si] << 23);
      vs = __uint_as_float((uint32_t)c.v_scale[si] << 23);
    }
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) s = fmaf(qv[i], value(c.k, at + i * 32 + lane), s);
#pragma unroll
    for (int w = 16; w > 0; w >>= 1) s += __shfl_xor_sync(0xffffffffu, s, w);
    s *= qscale * ks;
    const float mn = s > m ? s : m;
    const float base = mn == -INFINITY ? 0.f : mn;
    const float f = ex2(m - base), pr = ex2(s - base);
    m = mn;
    l = fmaf(l, f, pr);
#pragma unroll
    for (int i = 0; i < NV; ++i) o[i] = fmaf(pr * vs, value(c.v, at + i * 32 + lane), o[i] * f);
    if (l != l) break;  // a NaN score: the whole row is NaN
  }
  const float inv = l != 0.f ? 1.f / l : (lim > 0 ? NAN : 0.f);
#pragma unroll
  for (int i = 0; i < NV; ++i) out[i * 32 + lane] = __float2bfloat16_rn(l != l ? l : o[i] * inv);
}

// Every fourth column of unit u of row b, from `first` on, by one warp: those that are not finite are redone where must_redo says
// so. (NaN in every dim without a bad value: the column's sum is NaN, as a NaN score has it.)
template <bool FP8, int DIM>
__device__ __noinline__ void redo_columns(const Params& p, const int* len, int b, int u, int first) {
  const int lane = threadIdx.x & 31;
  const int h = u / p.chunks, col0 = (u - h * p.chunks) * p.chunk_cols, ncol = min(p.chunk_cols, p.cols - col0);
  const int need = min(p.cap, len[b] + p.tokens - 1);
  const int32_t* table = p.table + (int64_t)b * p.table_stride;
  BadValues bad{};
  bool known = false;
  for (int j = first; j < ncol; j += 4) {
    int t;
    const int64_t row = query_row(p, b, h, col0 + j, &t);
    bool odd = false, nan = true;
#pragma unroll
    for (int i = 0; i < DIM / 32; ++i) {
      const float x = __bfloat162float(p.out[row * DIM + i * 32 + lane]);
      odd |= !(fabsf(x) <= 3.3e38f);
      nan &= x != x;
    }
    if (!__any_sync(0xffffffffu, odd)) continue;
    if (!known) bad = bad_page_values<FP8, DIM>(p.c, table, h, max(0, len[b]), need);
    known = true;
    const int lim = min(need, len[b] + t);
    if (must_redo(bad, lim) && (bad.last >= lim || !__all_sync(0xffffffffu, nan)))
      exact_column<FP8, DIM>(p.q + row * DIM, p.c, table, h, lim, p.qscale, p.out + row * DIM);
  }
}

template <bool FP8, int DIM, int NQT>
__global__ void __launch_bounds__(kThreads, 1)
    paged_tc_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, const __grid_constant__ Params p) {
  using C = Cfg<FP8, DIM, NQT>;
  constexpr int CD = C::CD, DC = C::DC, N = C::N, SLOTS = C::SLOTS, SLOT = C::SLOT, ROWB = C::ROWB, NB = C::NB;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ Ctl ctl;
  int* pre = reinterpret_cast<int*>(smem + C::PRE_OFF);
  int* len = reinterpret_cast<int*>(smem + C::LEN_OFF);
  volatile int& abort_flag = ctl.abort_flag;
  volatile int* loads = ctl.loads;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  if (tid == 0) {
    for (int s = 0; s < SLOTS; ++s) {
      mbar_init(&ctl.full[s], 1);
      mbar_init(&ctl.empty[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&ctl.s_full[s], 1);
      mbar_init(&ctl.s_free[s], 128);
      mbar_init(&ctl.p_full[s], 128);
      mbar_init(&ctl.pv_done[s], 1);
      mbar_init(&ctl.o_full[s], 1);
      mbar_init(&ctl.o_free[s], 128);
      mbar_init(&ctl.ml_full[s], 256);
      mbar_init(&ctl.ml_free[s], 128);
    }
    for (int s = 0; s < 4; ++s) {
      mbar_init(&ctl.q_full[s], 4);
      mbar_init(&ctl.q_empty[s], 1);
    }
    for (int s = 0; s < kScaleStages; ++s) mbar_init(&ctl.sc_full[s], 32);
    mbar_init(&ctl.drain, 2);
    mbar_fence_init();
    abort_flag = 0;
    for (int s = 0; s < kMaxSlots; ++s) loads[s] = 0;
    ctl.odd = ctl.odd_cuts = 0;
  }
  if (warp == W_EPI) tmem_alloc(&ctl.tmem_base, C::TMEM);
  if (warp == W_LOADK && lane == 0) {
    prefetch_tmap(&kmap);
    prefetch_tmap(&vmap);
  }
  grid_launch_dependents();
  grid_dependency_wait();  // everything below may come from the kernel before

  // Tiles before each row, and the rows' lengths, in shared memory (each thread sums consecutive rows, then a block scan).
  const int per_row = p.c.kv_heads * p.chunks;
  {
    const int each = (p.rows + kThreads - 1) / kThreads;
    int mine = 0, most_tiles = 0;
    for (int i = 0; i < each; ++i) {
      const int b = tid * each + i;
      if (b >= p.rows) break;
      const int64_t raw = p.lengths[b];
      if (blockIdx.x == 0 && (raw < 0 || raw > p.cap - (p.tokens - 1))) raise_status(p.status, kStatusIndex);
      // The keys of the row's last query; a length out of range is clamped (and was reported), so that len + tokens is an int.
      const int64_t high = min(p.cap, 0x7fffffff - p.tokens);
      len[b] = (int)max(-(int64_t)p.tokens, min(raw, high));
      const int nt = (max(0, min(p.cap, len[b] + p.tokens - 1)) + BN - 1) / BN;
      most_tiles = max(most_tiles, nt);
      mine += nt * per_row;
      pre[b + 1] = mine;
    }
    most_tiles = __reduce_max_sync(0xffffffffu, most_tiles);
    if (lane == 0) ctl.wmax[warp] = most_tiles;
    int incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += y;
    }
    if (lane == 31) ctl.wsum[warp] = incl;
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    int before = incl - mine;
    for (int w = 0; w < warp; ++w) before += ctl.wsum[w];
    for (int i = 0; i < each; ++i) {
      const int b = tid * each + i;
      if (b >= p.rows) break;
      pre[b + 1] += before;
    }
    if (tid == 0) pre[0] = 0;
    __syncthreads();
  }
  const int total = pre[p.rows];
  // Tiles per CTA: an even share. Where that cuts units into many parts of many columns, more: a part costs about as long to
  // join, per 32 columns x chunks, as a tile takes.
  int per = max(1, (total + (int)gridDim.x - 1) / (int)gridDim.x);
  const int units = p.rows * per_row;
  if (p.chunk_cols * DC >= 16 && per < 16) {
    const int each = total / units;  // tiles of a unit, on average
    per = max(per, min(each, (int)sqrtf((float)(each * p.chunk_cols * DC) * (1.f / 32.f))));
  }
  int c0 = min(total, (int)blockIdx.x * per), c1 = min(total, c0 + per);
  // Joining costs some four tiles' time whatever it joins: units that there are CTAs for, and that are hardly longer than
  // the share, stay whole, one to a CTA (one row of 5 x 32 queries over 700 keys: 13.0 against 12.3 us, cut and whole).
  int longest = 0;
#pragma unroll 1
  for (int w = 0; w < kThreads / 32; ++w) longest = max(longest, ctl.wmax[w]);
  if (units <= (int)gridDim.x && longest <= per + 4) {
    const int b = (int)blockIdx.x / per_row, u = (int)blockIdx.x - b * per_row;
    c0 = c1 = 0;
    if (b < p.rows) {
      const int nt = (pre[b + 1] - pre[b]) / per_row;
      c0 = pre[b] + u * nt;
      c1 = c0 + nt;
    }
  }
  const int tiles = c1 - c0;
  const uint32_t tbase = ctl.tmem_base;
  auto wait = [&](uint64_t* bar, uint32_t parity) -> bool {
    if (mbar_wait_or(bar, parity, &abort_flag)) return true;
    abort_flag = 1;
    return false;
  };
  // Until `uses` loads into the slot have been issued. Every role walks the ring on its own, and a slot may hold K and V in
  // turn, so a role may come to a slot two uses early; a barrier's parity tells one use from the next only. A load is issued
  // once the one before it has landed and been consumed: after this, the slot's barriers are at most one use behind.
  auto wait_issued = [&](int slot, int uses) -> bool {
    if (loads[slot] >= uses) return true;
    const uint64_t t_start = global_ns();
    while (loads[slot] < uses) {
      if (abort_flag || global_ns() - t_start > kWaitLimitNs) {
        abort_flag = 1;
        return false;
      }
    }
    return true;
  };
  auto ring_skip = [&](int& slot, int& use) {  // past a tile's chunks of the other operand
    slot += DC;
    if (slot >= SLOTS) {
      slot -= SLOTS;
      ++use;
    }
  };
  // Ring positions of tile i's first K and V chunk, in the MMAs' order: K0 K1 K2 V0 K3 V1 .. K(n-1) V(n-3) V(n-2) V(n-1).
  auto k_chunk = [&](int i) { return DC * (i < 2 ? i : 2 * i - 2); };
  auto v_chunk = [&](int i) { return DC * min(2 * i + 3, tiles + i); };

  if (warp == W_LOADV) {  // the rows without keys: zeros, by this warp of every CTA
    for (int b = blockIdx.x; b < p.rows; b += gridDim.x) {
      if (pre[b + 1] != pre[b]) continue;
      uint4* o = reinterpret_cast<uint4*>(p.out + (int64_t)b * p.tokens * p.heads * DIM);
      for (int i = lane; i < p.tokens * p.heads * (DIM / 8); i += 32) o[i] = make_uint4(0u, 0u, 0u, 0u);
    }
  }

  if (tiles <= 0) {
    // nothing but giving the TMEM back
  } else if (warp == W_LOADK || warp == W_LOADV) {
    // ------------------------------------------------------------------ K (and the scale bytes) or V, page by page
    // Lane i holds the tile's i-th page (the only one, for pages of 128 positions and more), loaded a tile ahead. Two warps,
    // as a box takes its warp about 50 ns to issue, which small pages would wait for.
    const bool is_k = warp == W_LOADK;
    const CUtensorMap* map = is_k ? &kmap : &vmap;
    const bool leader = elect_one();
    const bool small = p.page_shift >= 0;
    const int rows_box = small ? p.c.page : BN;
    const int boxes = small ? BN >> p.page_shift : 1;
    Walk w;
    w.init(p, pre, len, c0, c1);
    Seg s{};
    int t = 0, ntile = 0;  // the tile in hand
    struct Tile {
      int h, live, row, id;  // kv head, boxes with keys, first row within the page, this lane's page
    };
    auto fetch = [&](Tile& x) {  // the tile (s, t): its page numbers start to load
      const int left = s.need - t * BN;
      x.h = s.h;
      x.live = small ? min(boxes, (left + rows_box - 1) >> p.page_shift) : 1;
      x.row = small ? 0 : (t * BN) % p.c.page;
      const int pi = small ? ((t * BN) >> p.page_shift) + lane : (t * BN) / p.c.page;
      x.id = lane < x.live ? __ldg(p.table + (int64_t)s.b * p.table_stride + pi) : 0;
    };
    auto step = [&]() {  // to the next tile; false past the last
      if (++ntile >= tiles) return false;
      if (++t >= s.t1) {
        w.next(s);
        t = s.t0;
      }
      return true;
    };
    int slot = is_k ? 0 : v_chunk(0) % SLOTS, use = is_k ? 0 : v_chunk(0) / SLOTS;
    w.next(s);
    t = s.t0;
    Tile x, nxt;
    fetch(x);
    nxt = x;
    for (int i = 0; i < tiles; ++i) {
      if (x.id < 0 || x.id >= (int)p.c.pages) {
        raise_status(p.status, kStatusIndex);
        x.id = 0;
      }
      const int left = s.need - t * BN;  // keys of this tile (before the walk goes on)
      if (step()) fetch(nxt);
      bool ok = true;
      for (int c = 0; c < DC; ++c) {
        // The slot's load before this one may be the other warp's.
        ok = use < 1 || (wait_issued(slot, use) && wait(&ctl.empty[slot], (use - 1) & 1));
        if (!__all_sync(0xffffffffu, ok)) {
          ok = false;
          break;
        }
        if (leader) mbar_arrive_expect_tx(&ctl.full[slot], (uint32_t)(x.live * rows_box * ROWB * NB));
        for (int k = 0; k < x.live; ++k) {
          const int id = __shfl_sync(0xffffffffu, x.id, k);
          if (leader) {
            unsigned char* dst = smem + slot * SLOT + k * rows_box * ROWB;
#pragma unroll
            for (int h = 0; h < NB; ++h)
              tma_load_4d(dst + h * C::BOX, map, c * CD + h * (ROWB / C::ES), x.row, x.h, id, &ctl.full[slot]);
          }
        }
        if (leader) loads[slot] = use + 1;
        __syncwarp();
        if (FP8 && is_k && c == 0) {
          // Four keys' scale bytes per lane (within one page), copied without waiting for them. The stage is free: this K
          // chunk went into a slot whose last one, at most 20 chunks (ten tiles) back, has been used, and an S^T is issued
          // after the reads of the scales two tiles before it.
          const int st = i % kScaleStages;
          const int pi = small ? (4 * lane) >> p.page_shift : 0;
          const int64_t id = __shfl_sync(0xffffffffu, x.id, pi);
          if (4 * lane < left) {
            const int64_t o = (id * p.c.kv_heads + x.h) * p.c.page + (small ? (4 * lane) & (p.c.page - 1) : x.row + 4 * lane);
            unsigned char* dst = smem + C::SC_OFF + st * 2 * BN + 4 * lane;
            copy4(dst, p.c.k_scale + o);
            copy4(dst + BN, p.c.v_scale + o);
          }
          copy_arrive(&ctl.sc_full[st]);
        }
        if (++slot == SLOTS) {
          slot = 0;
          ++use;
        }
      }
      if (!ok) break;
      // The other operand's chunks between this tile's and the next one's.
      if (is_k ? i >= 2 && i + 1 < tiles : i + 3 < tiles) ring_skip(slot, use);
      x = nxt;
    }
    if (FP8) asm volatile("cp.async.wait_all;" ::: "memory");
    __syncwarp();
  } else if (warp == W_MMA) {
    // ------------------------------------------------------------------ S^T(i) = K(i) Q^T
    // The issuing warps run converged, one elected lane issuing, so that the descriptors are warp-uniform: with a lone
    // thread issuing both products, four MMAs and their two commits took 520 clocks and a tile 1800.
    constexpr uint32_t IS = FP8 ? idesc_e4m3(128, N, 0, 0) : idesc_bf16(128, N, 0, 0);
    const uint64_t kd0 = smem_desc(smem_addr(smem), 16, C::GRP, C::LAYOUT);
    const uint64_t qd0 = smem_desc(smem_addr(smem + C::Q_OFF), 16, C::GRP, C::LAYOUT);
    const bool leader = elect_one();
    Walk w;
    w.init(p, pre, len, c0, c1);
    Seg s{};
    int i = 0, slot = 0, use = 0;
    bool ok = true;
    for (int n = 0; ok && w.next(s); ++n) {
      ok = __all_sync(0xffffffffu, wait(&ctl.q_full[n % C::QN], (n / C::QN) & 1));
      const uint64_t qd = qd0 + (uint64_t)((n % C::QN) * (C::QB >> 4));
      const int end = i + s.t1 - s.t0;
      for (; ok && i < end; ++i) {
        const int b = i & 1;
        if (i >= 2) ok = wait(&ctl.s_free[b], ((i >> 1) - 1) & 1);
#pragma unroll
        for (int c = 0; c < DC; ++c) {
          // The lanes leave their waits together, with one answer: none is still at a barrier that these MMAs move on.
          ok = __all_sync(0xffffffffu, ok && wait_issued(slot, use + 1) && wait(&ctl.full[slot], use & 1));
          if (!ok) break;
          tc_fence_after();
          if (leader) {
            const uint64_t kd = kd0 + (uint64_t)(slot * (SLOT >> 4));
            const uint32_t d = tbase + b * N;
#pragma unroll
            for (int kk = 0; kk < CD * C::ES / 32; ++kk) {  // 32 bytes of each row per MMA
              const int box = kk * 32 / ROWB, off = kk * 32 % ROWB;
              const uint64_t ko = (uint64_t)((box * C::BOX + off) >> 4);
              const uint64_t qo = (uint64_t)(((c * NB + box) * C::QBOX + off) >> 4);
              if constexpr (FP8) mma_f8_ss(d, kd + ko, qd + qo, IS, (c > 0 || kk > 0) ? 1u : 0u);
              else mma_bf16_ss(d, kd + ko, qd + qo, IS, (c > 0 || kk > 0) ? 1u : 0u);
            }
            tc_commit(&ctl.empty[slot]);
          }
          if (++slot == SLOTS) {
            slot = 0;
            ++use;
          }
        }
        if (!ok) break;
        if (leader) {
          tc_commit(&ctl.s_full[b]);
          if (i == end - 1) tc_commit(&ctl.q_empty[n % C::QN]);
        }
        __syncwarp();
        if (i >= 2 && i < tiles - 1) ring_skip(slot, use);  // V(i - 2) lies before K(i + 1)
      }
    }
    __syncwarp();
  } else if (warp == W_PV) {
    // ------------------------------------------------------------------ O^T += V(i)^T P(i)^T
    constexpr uint32_t IO = FP8 ? idesc_e4m3(128, N, 1, 1) : idesc_bf16(128, N, 1, 1);
    // (head_dim 64: the MMA's upper 64 rows read the same dims again, and nothing reads them.)
    const uint64_t vd0 = smem_desc(smem_addr(smem), CD == 64 ? 0 : C::BOX, C::GRP, C::LAYOUT);
    const uint64_t pd0 = smem_desc(smem_addr(smem + C::P_OFF), 128, 2048, kLayoutNone);
    const bool leader = elect_one();
    Walk w;
    w.init(p, pre, len, c0, c1);
    Seg s{};
    int i = 0, slot = v_chunk(0) % SLOTS, use = v_chunk(0) / SLOTS;
    bool ok = true;
    for (int n = 0; ok && w.next(s); ++n) {
      const int ob = C::OB == 2 ? n & 1 : 0;
      if (n >= C::OB) ok = __all_sync(0xffffffffu, wait(&ctl.o_free[ob], (n / C::OB - 1) & 1));
      const int begin = i, end = i + s.t1 - s.t0;
      for (; ok && i < end; ++i) {
        const int b = i & 1;
        ok = wait(&ctl.p_full[b], (i >> 1) & 1);
        const uint64_t pd = pd0 + (uint64_t)(b * (C::PB >> 4));
        const uint32_t fresh = i - begin < 2 ? 0u : 1u;  // a softmax group's first tile of the segment overwrites
#pragma unroll
        for (int c = 0; c < DC; ++c) {
          ok = __all_sync(0xffffffffu, ok && wait_issued(slot, use + 1) && wait(&ctl.full[slot], use & 1));
          if (!ok) break;
          tc_fence_after();
          if (leader) {
            const uint64_t vd = vd0 + (uint64_t)(slot * (SLOT >> 4));
            const uint32_t d = tbase + C::S_COLS + ((ob * 2 + b) * DC + c) * N;
#pragma unroll
            for (int kk = 0; kk < (FP8 ? 4 : 8); ++kk) {
              if constexpr (FP8) mma_f8_ss(d, vd + kk * (4 * C::GRP >> 4), pd + kk * (512 >> 4), IO, kk > 0 ? 1u : fresh);
              else mma_bf16_ss(d, vd + kk * (2 * C::GRP >> 4), pd + kk * (256 >> 4), IO, kk > 0 ? 1u : fresh);
            }
            tc_commit(&ctl.empty[slot]);
          }
          if (++slot == SLOTS) {
            slot = 0;
            ++use;
          }
        }
        if (!ok) break;
        if (leader) {
          tc_commit(&ctl.pv_done[b]);
          if (i == end - 1) tc_commit(&ctl.o_full[ob]);
        }
        __syncwarp();
        if (i + 3 < tiles) ring_skip(slot, use);  // K(i + 3) lies before V(i + 1)
      }
    }
    __syncwarp();
  } else if (warp < 4 || warp >= W_SOFT1) {
    // ------------------------------------------------------------------ softmax: thread = key of the tile
    // Group b takes the tiles of parity b, with its own S^T and P^T buffers.
    const int b = warp >= W_SOFT1 ? 1 : 0, wq = warp & 3, key_in = tid & 127;
    const int bar = b == 0 ? 1 : 3;
    const uint32_t lane_off = (uint32_t)(32 * wq) << 16;
    Walk w;
    w.init(p, pre, len, c0, c1);
    Seg s{};
    int seg0 = 0;  // the segment's first tile in this CTA's numbering
    bool quit = false;
    for (int n = 0; !quit && w.next(s); ++n) {
      const int need = s.need, ncol = s.ncol;
      int tok0, g0;                            // the first column's token and head
      column(p, s.col0, tok0, g0);
      const int lim0 = len[s.b] + tok0;        // the keys it sees; later tokens see more
      const int ob = C::OB == 2 ? n & 1 : 0;
      float m[NQT], l[NQT];
#pragma unroll
      for (int j = 0; j < NQT; ++j) m[j] = l[j] = 0.f;
      bool first = true;
      for (int i = seg0 + ((seg0 ^ b) & 1); i < seg0 + s.t1 - s.t0; i += 2) {
        const int t = s.t0 + i - seg0;
        const int key = t * BN + key_in;
        wait(&ctl.s_full[b], (i >> 1) & 1);
        float ks = 1.f, ev = 0.f, iv = 1.f;
        if constexpr (FP8) {
          const int st = i % kScaleStages;
          wait(&ctl.sc_full[st], (i / kScaleStages) & 1);
          const unsigned char* sc = smem + C::SC_OFF + st * 2 * BN;
          ks = __uint_as_float((uint32_t)sc[key_in] << 23);
          const int eb = key < need ? sc[BN + key_in] : 127;  // (past the row's keys the stage holds anything)
          ev = (float)(eb - 127);
          iv = __uint_as_float((uint32_t)(254 - eb) << 23);
        }
        tc_fence_after();
        __syncwarp();
        float sv[N];
#pragma unroll
        for (int c = 0; c < N / 16; ++c) tmem_ld16(tbase + lane_off + b * N + c * 16, sv + c * 16);
        tc_fence_before();
        float x[NQT];
#pragma unroll
        for (int j = 0; j < NQT; ++j) {
          if constexpr (FP8) x[j] = fmaf(fmaf(sv[NQT + j], 0.0625f, sv[j]) * ks, ctl.cq[n & 7][j], ev);
          else x[j] = sv[j] * p.qscale;
        }
        mbar_arrive(&ctl.s_free[b]);  // (after the last read of the queries' factors and the scales, too)
        bool over = FP8 && first;
        if (!FP8 && first) {  // a unit starts from maximum 0 unless its scores lie far below; -inf is such a score
#pragma unroll
          for (int j = 0; j < NQT; ++j) over |= x[j] < -kBelow && j < ncol && key < need;
        }
        if (NQT > ncol || (t + 1) * BN > lim0) {  // spare columns, or keys that some column does not see
          int tt = 0, g = g0;
#pragma unroll
          for (int j = 0; j < NQT; ++j) {
            if (j >= ncol || key >= min(need, lim0 + tt)) x[j] = -INFINITY;
            if (++g == p.group) {
              g = 0;
              ++tt;
            }
          }
        }
#pragma unroll
        for (int j = 0; j < NQT; ++j) over |= x[j] > m[j] + kRaise;
        const bool saw = abort_flag != 0;
        if (sync_or(bar, 128, over || saw)) {
          float v[NQT];
#pragma unroll
          for (int j = 0; j < NQT; ++j) v[j] = x[j];
          warp_all<NQT, true>(v);
          if (lane == 0) {
#pragma unroll
            for (int j = 0; j < NQT; ++j) ctl.red[b][wq][j] = v[j];
          }
          if (sync_or(bar, 128, saw)) {
            quit = true;
            break;
          }
          float scl[NQT];
          bool any = false;
#pragma unroll
          for (int j = 0; j < NQT; ++j) {
            const float top = fmaxf(fmaxf(ctl.red[b][0][j], ctl.red[b][1][j]), fmaxf(ctl.red[b][2][j], ctl.red[b][3][j]));
            float mn = m[j];
            if (FP8) {
              if (top != -INFINITY) mn = first ? top - kHead8 : (top > m[j] + kRaise ? top - kHead8 : m[j]);
            } else {
              // (No score but -inf yet: below whatever comes, and -inf less it is -inf.)
              mn = fmaxf(first ? kNone : m[j], top);
            }
            scl[j] = first ? 1.f : ex2(m[j] - mn);
            any |= scl[j] != 1.f;
            m[j] = mn;
            l[j] *= scl[j];
          }
          if (any && !first) {  // the same in every thread: the maxima are
            wait(&ctl.pv_done[b], ((i >> 1) - 1) & 1);  // O holds every earlier tile of the segment and group
            tc_fence_after();
            __syncwarp();
#pragma unroll 1
            for (int c = 0; c < DC; ++c) {
              const uint32_t o = tbase + lane_off + C::S_COLS + ((ob * 2 + b) * DC + c) * N;
              float ov[N];
#pragma unroll
              for (int k = 0; k < N / 16; ++k) tmem_ld16(o + k * 16, ov + k * 16);
#pragma unroll
              for (int j = 0; j < NQT; ++j) {
                ov[j] *= scl[j];
                if (FP8) ov[NQT + j] *= scl[j];
              }
#pragma unroll
              for (int k = 0; k < N / 16; ++k) tmem_st16(o + k * 16, ov + k * 16);
            }
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
          }
          named_sync(bar, 128);  // the maxima are read before the next tile writes them
        }
        float pr[NQT];
#pragma unroll
        for (int j = 0; j < NQT; ++j) {
          pr[j] = ex2(x[j] - m[j]);
          l[j] = FP8 ? fmaf(pr[j], iv, l[j]) : l[j] + pr[j];
        }
        if (i >= 2) wait(&ctl.pv_done[b], ((i >> 1) - 1) & 1);  // P(i - 2) is used up
        unsigned char* pb = smem + C::P_OFF + b * C::PB;
        if constexpr (FP8) {
          // The dither of this key, within half of the second piece's smallest step (2^-9): the tile's 128 keys in bit-reversed
          // order, moved on by a golden section from tile to tile. (A weight of 0 stays 0: half a step is rounded to even.)
          const float dither = (float)(int)(__brev(key_in) + (uint32_t)t * 0x9e3779b9u) * 0x1p-41f;
          uint32_t hw[NQT >= 4 ? NQT / 4 : 1], lw[NQT >= 4 ? NQT / 4 : 1];
#pragma unroll
          for (int k = 0; k < (NQT >= 4 ? NQT / 4 : 1); ++k) hw[k] = lw[k] = 0u;
#pragma unroll
          for (int j = 0; j < NQT; j += 2) {
            const float p0 = pr[j], p1 = j + 1 < NQT ? pr[j + 1 < NQT ? j + 1 : j] : 0.f;
            const uint32_t a = __nv_cvt_float2_to_fp8x2(make_float2(p0, p1), __NV_SATFINITE, __NV_E4M3);
            const __half2_raw hr = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)a, __NV_E4M3);
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&hr));
            const uint32_t r = __nv_cvt_float2_to_fp8x2(
                make_float2(fmaf(p0 - f.x, 16.f, dither), fmaf(p1 - f.y, 16.f, dither)), __NV_SATFINITE, __NV_E4M3);
            hw[j >> 2] |= a << (8 * (j & 3));
            lw[j >> 2] |= r << (8 * (j & 3));
          }
          // Columns 0 .. NQT - 1 the first pieces, NQT .. 2 NQT - 1 the second, zeros after them.
          uint4 w0, w1 = make_uint4(0u, 0u, 0u, 0u);
          if constexpr (NQT == 16) {
            w0 = make_uint4(hw[0], hw[1], hw[2], hw[3]);
            w1 = make_uint4(lw[0], lw[1], lw[2], lw[3]);
          } else if constexpr (NQT == 8) {
            w0 = make_uint4(hw[0], hw[1], lw[0], lw[1]);
          } else if constexpr (NQT == 4) {
            w0 = make_uint4(hw[0], lw[0], 0u, 0u);
          } else if constexpr (NQT == 2) {
            w0 = make_uint4((hw[0] & 0xffffu) | (lw[0] << 16), 0u, 0u, 0u);
          } else {
            w0 = make_uint4((hw[0] & 0xffu) | ((lw[0] & 0xffu) << 8), 0u, 0u, 0u);
          }
          *reinterpret_cast<uint4*>(pb + key_in * 16) = w0;
          if constexpr (N == 32) *reinterpret_cast<uint4*>(pb + 2048 + key_in * 16) = w1;
        } else {
          uint32_t wv[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const float lo = 2 * k < NQT ? pr[2 * k < NQT ? 2 * k : 0] : 0.f;
            const float hi = 2 * k + 1 < NQT ? pr[2 * k + 1 < NQT ? 2 * k + 1 : 0] : 0.f;
            const __nv_bfloat162 v2 = __floats2bfloat162_rn(lo, hi);
            wv[k] = *reinterpret_cast<const uint32_t*>(&v2);
          }
          *reinterpret_cast<uint4*>(pb + key_in * 16) = make_uint4(wv[0], wv[1], wv[2], wv[3]);
          *reinterpret_cast<uint4*>(pb + 2048 + key_in * 16) = make_uint4(wv[4], wv[5], wv[6], wv[7]);
        }
        if (t * BN + BN > need) {
          // The row's last tile: V rows past its keys may hold anything, and 0 x NaN is NaN. Cleared once loaded (the
          // producer has issued the chunk, so the slot's phase is the chunk's).
          const int vc = v_chunk(i);
          for (int c = 0; c < DC; ++c) {
            if (!wait_issued((vc + c) % SLOTS, (vc + c) / SLOTS + 1)) break;
            wait(&ctl.full[(vc + c) % SLOTS], ((vc + c) / SLOTS) & 1);
            if (key >= need) {
              unsigned char* row = smem + ((vc + c) % SLOTS) * SLOT + key_in * ROWB;
#pragma unroll
              for (int k = 0; k < ROWB / 16; ++k) {
#pragma unroll
                for (int x2 = 0; x2 < NB; ++x2) *reinterpret_cast<uint4*>(row + x2 * C::BOX + k * 16) = make_uint4(0u, 0u, 0u, 0u);
              }
            }
          }
        }
        fence_async_smem();
        tc_fence_before();
        mbar_arrive(&ctl.p_full[b]);
        first = false;
      }
      if (quit) break;
      seg0 += s.t1 - s.t0;
      // The segment's sums and maxima (sums of zero where the group had no tile), once the epilogue has read those of two
      // segments before.
      if (n >= 2) wait(&ctl.ml_free[n & 1], ((n >> 1) - 1) & 1);
      warp_all<NQT, false>(l);
      if (lane == 0) {
#pragma unroll
        for (int j = 0; j < NQT; ++j) ctl.sum[n & 1][b][wq][j] = l[j];
      }
      if (key_in == 0) {
#pragma unroll
        for (int j = 0; j < NQT; ++j) ctl.top[n & 1][b][j] = m[j];
      }
      mbar_arrive(&ctl.ml_full[n & 1]);
    }
  } else {
    // ------------------------------------------------------------------ epilogue: thread = head dim of each chunk
    const int d = tid - W_EPI * 32;
    const uint32_t lane_off = (uint32_t)(32 * (warp & 3)) << 16;
    Walk w, ahead;
    w.init(p, pre, len, c0, c1);
    ahead = w;
    Seg s{}, sq{};
    // (After an abort the waits return at once and these warps go through their segments all the same, so that no barrier
    // of theirs is left to some of them.)
    // These warps also load the queries, QN segments ahead: warp w the columns w, w + 4, .. of a segment. They are written
    // out as soon as a segment's last S^T has released its buffer, not after its O: a V chunk may wait for the slot of a K
    // chunk two tiles on, whose S^T needs the queries. (The factors of 8 segments are kept, as the softmax may still read
    // those of segment n when segment n + QN's are written.)
    constexpr int QC = (NQT + 3) / 4;
    const int wq = warp - W_EPI;
    uint2 qr[QC][DC];  // four dims per lane of each chunk (head_dim 64: of the first 16 lanes)
    auto query_load = [&]() {
#pragma unroll
      for (int k = 0; k < QC; ++k) {
        const int j = wq + 4 * k;
        if (j < sq.ncol) {
          int tt;
          const uint2* src = reinterpret_cast<const uint2*>(p.q + query_row(p, sq.b, sq.h, sq.col0 + j, &tt) * DIM) + lane;
#pragma unroll
          for (int c = 0; c < DC; ++c) qr[k][c] = CD == 128 || lane < 16 ? __ldg(src + c * 32) : make_uint2(0u, 0u);
        }
      }
    };
    // The 16-byte words of row r are stored at index ^ swizzle(r) (the 128- or 64-byte swizzle of the tensor maps).
    auto swizzle = [](int r) { return ROWB == 128 ? r & 7 : (r >> 1) & 3; };
    auto query_store = [&](int n) {
      unsigned char* qb = smem + C::Q_OFF + (n % C::QN) * C::QB;
#pragma unroll
      for (int k = 0; k < QC; ++k) {
        const int j = wq + 4 * k;
        if (j >= sq.ncol) continue;
        if constexpr (FP8) {
          float x[DC][4];
          uint32_t amax = 0u;
#pragma unroll
          for (int c = 0; c < DC; ++c) {
            x[c][0] = __uint_as_float(qr[k][c].x << 16), x[c][1] = __uint_as_float(qr[k][c].x & 0xffff0000u);
            x[c][2] = __uint_as_float(qr[k][c].y << 16), x[c][3] = __uint_as_float(qr[k][c].y & 0xffff0000u);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint32_t bits = __float_as_uint(x[c][e]) & 0x7fffffffu;
              amax = max(amax, bits < 0x7f800000u ? bits : 0u);
            }
          }
          amax = __reduce_max_sync(0xffffffffu, amax);
          int e = (int)(amax >> 23) - 127 - 7;  // the largest in [2^7, 2^8)
          e = amax == 0u ? 0 : (e < -100 ? -100 : e);
          const float inv = __uint_as_float((uint32_t)(127 - e) << 23);
#pragma unroll
          for (int c = 0; c < DC; ++c) {
            uint32_t hi = 0u, lo = 0u;
#pragma unroll
            for (int i = 0; i < 4; i += 2) {
              // (An infinity becomes NaN: the conversion would clip it.)
              float y0 = x[c][i] * inv, y1 = x[c][i + 1] * inv;
              y0 = fmaf(y0, 0.f, y0);
              y1 = fmaf(y1, 0.f, y1);
              const uint32_t a = __nv_cvt_float2_to_fp8x2(make_float2(y0, y1), __NV_SATFINITE, __NV_E4M3);
              const __half2_raw hr = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)a, __NV_E4M3);
              const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&hr));
              const uint32_t r =
                  __nv_cvt_float2_to_fp8x2(make_float2((y0 - f.x) * 16.f, (y1 - f.y) * 16.f), __NV_SATFINITE, __NV_E4M3);
              hi |= a << (8 * i);
              lo |= r << (8 * i);
            }
            const int r2 = NQT + j;
            unsigned char* box = qb + c * C::QBOX;
            if (CD == 128 || lane < 16) {
              *reinterpret_cast<uint32_t*>(box + j * ROWB + (((lane >> 2) ^ swizzle(j)) << 4) + (lane & 3) * 4) = hi;
              *reinterpret_cast<uint32_t*>(box + r2 * ROWB + (((lane >> 2) ^ swizzle(r2)) << 4) + (lane & 3) * 4) = lo;
            }
          }
          if (lane == 0) ctl.cq[n & 7][j] = p.qscale * __uint_as_float((uint32_t)(e + 127) << 23);
        } else {
#pragma unroll
          for (int c = 0; c < DC; ++c) {  // lanes 0-15 the chunk's first 64 dims, 16-31 the others
            unsigned char* box = qb + (NB * c + (lane >> 4)) * C::QBOX;
            if (CD == 128 || lane < 16)
              *reinterpret_cast<uint2*>(box + j * ROWB + ((((lane & 15) >> 1) ^ swizzle(j)) << 4) + (lane & 1) * 8) = qr[k][c];
          }
        }
      }
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&ctl.q_full[n % C::QN]);
    };
    for (int n = 0; n < C::QN && ahead.next(sq); ++n) {
      query_load();
      query_store(n);
    }
    constexpr bool DRAFTS = NQT > 1;  // (one column is one token, which sees every key)
    constexpr bool EARLY = QC * DC <= 8;  // loaded a segment before they are written out (while the registers hold them)
    bool more = ahead.next(sq);  // segment n + QN
    if (EARLY && more) query_load();
    for (int n = 0; w.next(s); ++n) {
      const int ob = C::OB == 2 ? n & 1 : 0;
      if (more) {
        if (!EARLY) query_load();
        wait(&ctl.q_empty[n % C::QN], (n / C::QN) & 1);
        query_store(n + C::QN);
        more = ahead.next(sq);
        if (EARLY && more) query_load();
      }
      wait(&ctl.o_full[ob], (n / C::OB) & 1);
      wait(&ctl.ml_full[n & 1], (n >> 1) & 1);
      tc_fence_after();
      __syncwarp();
      const int h = s.h, col0 = s.col0, ncol = s.ncol;
      int tok0, g0;
      column(p, col0, tok0, g0);
      // The two softmax groups' parts as one: weights 2^(m_b - m); a group that saw no key takes no part.
      float l[NQT], m[NQT], wt[2][NQT];
#pragma unroll
      for (int j = 0; j < NQT; ++j) {
        float ls[2], ms[2];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
          const auto& sum = ctl.sum[n & 1][b];
          ls[b] = (sum[0][j] + sum[1][j]) + (sum[2][j] + sum[3][j]);
          ms[b] = ls[b] != 0.f ? ctl.top[n & 1][b][j] : -INFINITY;
        }
        m[j] = fmaxf(ms[0], ms[1]);
#pragma unroll
        for (int b = 0; b < 2; ++b) wt[b][j] = ls[b] != 0.f ? ex2(ms[b] - m[j]) : 0.f;
        l[j] = ls[0] * wt[0][j] + ls[1] * wt[1][j];
      }
      mbar_arrive(&ctl.ml_free[n & 1]);
      bool bad = false;  // some result is not finite
      auto store = [&](int c, const float (&o)[NQT], const float (&sum)[NQT]) {
        int tt = tok0, g = g0;
        const int64_t row0 = (int64_t)s.b * p.tokens * p.heads + h * p.group;
#pragma unroll
        for (int j = 0; j < NQT; ++j) {
          if (j < ncol) {
            const int64_t row = row0 + tt * p.heads + g;
            // Nothing summed: a query that sees no key gets zeros, one whose keys all score -inf has no softmax.
            const float r = sum[j] != 0.f ? o[j] * __fdividef(1.f, sum[j]) : (len[s.b] + tt > 0 ? NAN : 0.f);
            if (DRAFTS && !(fabsf(r) <= 3.3e38f) && (CD == 128 || d < CD)) bad = true;
            if (CD == 128 || d < CD) p.out[row * DIM + c * CD + d] = __float2bfloat16_rn(r);
          }
          if (++g == p.group) {
            g = 0;
            ++tt;
          }
        }
      };
      const bool here = s.t0 == 0;  // the unit begins in this CTA
      bool emit = here && s.t1 == s.nt;
      const int place = (2 * (int)blockIdx.x + (here ? 1 : 0)) * kMaxCols;
#pragma unroll 1
      for (int c = 0; c < DC; ++c) {
        uint32_t v[2][N];
        float o[NQT];
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int k = 0; k < N / 16; ++k)
            tmem_ld16_async(tbase + lane_off + C::S_COLS + ((ob * 2 + b) * DC + c) * N + k * 16, v[b] + k * 16);
        tmem_wait();
#pragma unroll
        for (int b = 0; b < 2; ++b) {
#pragma unroll
          for (int j = 0; j < NQT; ++j) {
            const float x0 = __uint_as_float(v[b][j]);
            const float x = FP8 ? fmaf(__uint_as_float(v[b][(FP8 ? NQT : 0) + j]), 0.0625f, x0) : x0;
            const float add = wt[b][j] != 0.f ? x * wt[b][j] : 0.f;  // (a group without a tile: its O is stale)
            o[j] = b == 0 ? add : o[j] + add;
          }
        }
        if (c == DC - 1) {
          tc_fence_before();
          mbar_arrive(&ctl.o_free[ob]);
        }
        if (emit) {
          store(c, o, l);
        } else {
#pragma unroll
          for (int j = 0; j < NQT; ++j)
            if (j < ncol && (CD == 128 || d < CD)) p.part_o[(int64_t)(place + j) * DIM + c * CD + d] = o[j];
        }
      }
      if (!emit) {
        // A cut unit: its parts are joined in the order of the keys, by the CTA that publishes last; where there are more
        // than kJoin of them, in two steps (each run of kJoin parts by the last of its CTAs, then the runs).
        if (d == 0) {
#pragma unroll
          for (int j = 0; j < NQT; ++j)
            if (j < ncol) p.part_ml[place + j] = make_float2(m[j], l[j]);
        }
        const int f0 = s.first / per, parts = (s.first + s.nt - 1) / per - f0 + 1, mine = (int)blockIdx.x - f0;
        // True in the CTA that comes last of `of`; the parts of the others are visible to it then.
        auto arrive = [&](unsigned* counter, int of) -> bool {
          named_sync(2, 128);  // this CTA's part is written
          if (d == 0) {
            // Releases what the barrier has ordered before, acquires what the others released: no fences of their own.
            const bool last = add_acq_rel(counter) == (unsigned)(of - 1);
            if (last) *counter = 0;  // zero again for the next call
            ctl.last = last;
          }
          named_sync(2, 128);
          return ctl.last != 0;
        };
        auto slot_of = [&](int part) { return (2 * (f0 + part) + (part == 0 ? 1 : 0)) * kMaxCols; };
        // Joins `count` (at most kJoin) parts from `begin`, every `by`-th; `to`: a part's slot, or -1: the output.
        auto join = [&](int begin, int by, int count, int to) {
          // The parts' statistics first, 128 threads over (part, column): weights 2^(m_k - m), a part that saw no key taking
          // no part, and the sums.
          static_assert(kMaxCols == 16 && kJoin <= 16, "thread = part x 16 + column");
          const int kj = d & 15;
          for (int k = d >> 4; k < count; k += 8)
            if (kj < ncol) ctl.stat[k][kj] = __ldcg(p.part_ml + slot_of(begin + k * by) + kj);
          named_sync(2, 128);
          for (int k = d >> 4; k < count; k += 8) {
            if (kj >= ncol) break;
            float top = -INFINITY;
            for (int q = 0; q < count; ++q) top = ctl.stat[q][kj].y != 0.f ? fmaxf(top, ctl.stat[q][kj].x) : top;
            const float2 e = ctl.stat[k][kj];
            ctl.weight[k][kj] = e.y != 0.f ? ex2(e.x - top) : 0.f;
            if (k == 0) {
              float sum = 0.f;
              for (int q = 0; q < count; ++q) {
                const float2 f = ctl.stat[q][kj];
                if (f.y != 0.f) sum = fmaf(ex2(f.x - top), f.y, sum);
              }
              ctl.joined[kj] = make_float2(top, sum);
              if (to >= 0) p.part_ml[to + kj] = ctl.joined[kj];
            }
          }
          named_sync(2, 128);
          // Then the outputs: groups of columns, 32 loads in flight per thread.
          constexpr int JG = NQT < 8 ? NQT : 8, U = 32 / JG < kJoin ? 32 / JG : kJoin;
          const bool mine_d = CD == 128 || d < CD;
#pragma unroll 1
          for (int c = 0; c < DC; ++c) {
            float o[NQT];
#pragma unroll
            for (int j0 = 0; j0 < NQT; j0 += JG) {
#pragma unroll
              for (int j = 0; j < JG; ++j) o[j0 + j] = 0.f;
              if (j0 >= ncol) continue;
#pragma unroll 1
              for (int k0 = 0; k0 < count; k0 += U) {
                float v[U][JG];
#pragma unroll
                for (int k = 0; k < U; ++k) {
                  const float* src = p.part_o + (int64_t)(slot_of(begin + (k0 + k) * by) + j0) * DIM + c * CD + d;
#pragma unroll
                  for (int j = 0; j < JG; ++j) v[k][j] = mine_d && k0 + k < count && j0 + j < ncol ? __ldcg(src + j * DIM) : 0.f;
                }
#pragma unroll
                for (int k = 0; k < U; ++k) {
                  if (k0 + k < count) {
#pragma unroll
                    for (int j = 0; j < JG; ++j) {
                      const float wk = ctl.weight[k0 + k][j0 + j];
                      o[j0 + j] = wk != 0.f && j0 + j < ncol ? fmaf(wk, v[k][j], o[j0 + j]) : o[j0 + j];
                    }
                  }
                }
              }
            }
            if (to < 0) {
#pragma unroll
              for (int j = 0; j < NQT; ++j) l[j] = ctl.joined[j].y;
              store(c, o, l);
            } else {
#pragma unroll
              for (int j = 0; j < NQT; ++j)
                if (j < ncol && mine_d) p.part_o[(int64_t)(to + j) * DIM + c * CD + d] = o[j];
            }
          }
        };
        if (parts <= kJoin) {
          emit = arrive(p.counters + f0, parts);
          if (emit) join(0, 1, parts, -1);
        } else {
          const int begin = mine - mine % kJoin, count = min(kJoin, parts - begin);
          const int runs = (parts + kJoin - 1) / kJoin;
          if (arrive(p.counters + gridDim.x + 2 * (f0 + begin) + (begin == 0 ? 1 : 0), count)) {
            join(begin, 1, count, slot_of(begin));
            emit = arrive(p.counters + f0, runs);
            if (emit) join(0, kJoin, runs, -1);
          }
        }
      }
      if (emit) {
        if (DRAFTS && p.tokens > 1) {  // a column may have met a key it does not see
          // Redone when the CTA's units are done: it may take longer than the other roles wait for this one.
          if (sync_or(2, 128, bad) && d == 0) {
            if (here && s.t1 == s.nt) ctl.odd = 1;
            else ctl.odd_cut[ctl.odd_cuts++] = (unsigned)s.b << 16 | (unsigned)s.u;
          }
        }
      }
    }
    if (DRAFTS && p.tokens > 1 && !sync_or(2, 128, abort_flag != 0)) {
      for (int i = 0; i < ctl.odd_cuts; ++i) redo_columns<FP8, DIM>(p, len, ctl.odd_cut[i] >> 16, ctl.odd_cut[i] & 0xffff, wq);
      if (ctl.odd) {
        w.init(p, pre, len, c0, c1);
        while (w.next(s))
          if (s.t0 == 0 && s.t1 == s.nt) redo_columns<FP8, DIM>(p, len, s.b, s.u, wq);
      }
    }
  }
  __syncthreads();
  if (abort_flag) {
    if (tid == 0) raise_status(p.status, kStatusTimeout);
    if ((warp == W_MMA || warp == W_PV) && elect_one()) {
      tc_commit(&ctl.drain);  // every MMA issued has completed once this arrives
      mbar_wait(&ctl.drain, 0);
    }
    if (tid == W_LOADK * 32)  // the latest load of every slot lands before the shared memory goes away
      for (int i = 0; i < SLOTS; ++i)
        if (loads[i] > 0) mbar_wait(&ctl.full[i], (loads[i] - 1) & 1);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == W_EPI) {
    tc_fence_after();
    tmem_dealloc(tbase, C::TMEM);
  }
}

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      return (PFN_cuTensorMapEncodeTiled_v12000) nullptr;
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr);
  }();
  return fn;
}

bool page_map(CUtensorMap* map, const void* base, const PageCache& c) {
  const auto fn = encode_fn();
  if (!fn) return false;
  const bool fp8 = c.type == kFp8;
  const uint64_t es = fp8 ? 1 : 2;
  // An extent of one has a stride that nothing reads.
  auto st = [&](int64_t extent, int64_t stride) { return (cuuint64_t)(extent > 1 ? stride * es : 16); };
  const cuuint64_t dims[4] = {(cuuint64_t)c.dim, (cuuint64_t)c.page, (cuuint64_t)c.kv_heads, (cuuint64_t)c.pages};
  const cuuint64_t strides[3] = {st(c.page, c.s_pos), st(c.kv_heads, c.s_head), st(c.pages, c.s_page)};
  const bool half = fp8 && c.dim == 64;  // 64-byte rows
  const cuuint32_t box[4] = {(cuuint32_t)(fp8 && !half ? 128 : 64), (cuuint32_t)(c.page < BN ? c.page : BN), 1, 1};
  const cuuint32_t estr[4] = {1, 1, 1, 1};
  if (!strides[0] || !strides[1] || !strides[2]) return false;
  return fn(map, fp8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(base), dims, strides,
            box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, half ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <bool FP8, int DIM, int NQT>
cudaError_t launch_t(const CUtensorMap& k, const CUtensorMap& v, const Params& p, int grid, cudaStream_t stream) {
  using C = Cfg<FP8, DIM, NQT>;
  static PerDevice configured;
  if (const cudaError_t e = allow_smem(paged_tc_kernel<FP8, DIM, NQT>, C::BYTES, configured)) return e;
  return launch_dependent(paged_tc_kernel<FP8, DIM, NQT>, dim3(grid), dim3(kThreads), (size_t)C::BYTES, stream, k, v, p);
}

template <bool FP8, int DIM>
cudaError_t launch_cols(const CUtensorMap& k, const CUtensorMap& v, const Params& p, int grid, cudaStream_t s) {
  if (p.chunk_cols <= 1) return launch_t<FP8, DIM, 1>(k, v, p, grid, s);
  if (p.chunk_cols <= 2) return launch_t<FP8, DIM, 2>(k, v, p, grid, s);
  if (p.chunk_cols <= 4) return launch_t<FP8, DIM, 4>(k, v, p, grid, s);
  if (p.chunk_cols <= 8) return launch_t<FP8, DIM, 8>(k, v, p, grid, s);
  return launch_t<FP8, DIM, 16>(k, v, p, grid, s);
}

template <bool FP8>
cudaError_t launch_dim(const CUtensorMap& k, const CUtensorMap& v, const Params& p, int grid, cudaStream_t s) {
  if (p.c.dim == 64) return launch_cols<FP8, 64>(k, v, p, grid, s);
  if (p.c.dim == 128) return launch_cols<FP8, 128>(k, v, p, grid, s);
  if (p.c.dim == 256) return launch_cols<FP8, 256>(k, v, p, grid, s);
  return launch_cols<FP8, 512>(k, v, p, grid, s);
}

}  // namespace pagedtc

bool paged_tc_supported(int dtype, int type, int dim, int page) {
  const bool pages = page >= 128 ? page % 128 == 0 : page >= 8 && (page & (page - 1)) == 0;
  return dtype == kBF16 && (type == kBF16 || type == kFp8) && dim >= 64 && pages;
}

size_t paged_tc_workspace(int dim) {
  return kCounterBytes + (size_t)2 * device_sm_count() * pagedtc::kMaxCols * (dim * sizeof(float) + sizeof(float2));
}

cudaError_t launch_paged_attention_tc(const PagedAttnArgs& a, cudaStream_t stream) {
  using namespace pagedtc;
  CUtensorMap km, vm;
  if (!page_map(&km, a.c.k, a.c) || !page_map(&vm, a.c.v, a.c)) return cudaErrorNotSupported;
  const int grid = device_sm_count();
  Params p{};
  p.c = a.c;
  p.table_stride = a.table_stride;
  p.tokens = a.tokens;
  p.heads = a.heads;
  p.group = a.heads / a.c.kv_heads;
  p.cols = a.tokens * p.group;
  p.chunks = (p.cols + kMaxCols - 1) / kMaxCols;
  p.chunk_cols = (p.cols + p.chunks - 1) / p.chunks;
  p.chunks = (p.cols + p.chunk_cols - 1) / p.chunk_cols;
  p.cap = a.table_width * a.c.page;
  p.page_shift = -1;
  if (a.c.page < BN) {
    p.page_shift = 3;
    while ((1 << p.page_shift) < a.c.page) ++p.page_shift;
  }
  p.qscale = a.scale * kLog2e;
  p.counters = reinterpret_cast<unsigned*>(a.workspace);
  char* ws = reinterpret_cast<char*>(a.workspace) + kCounterBytes;
  p.part_o = reinterpret_cast<float*>(ws);
  p.part_ml = reinterpret_cast<float2*>(ws + (size_t)2 * grid * kMaxCols * a.c.dim * sizeof(float));
  p.status = a.status;
  // Rows per launch: what the shared-memory tables hold, and no more tiles than an int counts.
  const int64_t row_tiles = ((int64_t)(p.cap + BN - 1) / BN) * p.c.kv_heads * p.chunks;
  const int most = (int)std::min<int64_t>(kMaxRows, 0x7fffff00ll / std::max<int64_t>(1, row_tiles));
  if (most < 1) return cudaErrorNotSupported;
  for (int r0 = 0; r0 < a.rows; r0 += most) {
    p.rows = std::min(most, a.rows - r0);
    p.q = reinterpret_cast<const __nv_bfloat16*>(a.q) + (int64_t)r0 * a.tokens * a.heads * a.c.dim;
    p.out = reinterpret_cast<__nv_bfloat16*>(a.out) + (int64_t)r0 * a.tokens * a.heads * a.c.dim;
    p.table = a.table + (int64_t)r0 * a.table_stride;
    p.lengths = a.lengths + r0;
    const cudaError_t e = a.c.type == kFp8 ? launch_dim<true>(km, vm, p, grid, stream) : launch_dim<false>(km, vm, p, grid, stream);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

}  // namespace omni
