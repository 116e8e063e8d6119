// Device helpers shared by the tensor-core prefill kernels (prefill.cu, head_dim 128; prefill_wide.cu, head_dim
// 512): the A-from-TMEM MMA, TMEM loads and stores of one lane's columns, the softmax's packed f32x2 arithmetic, an
// FMA-pipe exponential, bf16 packing and a barrier that ORs a predicate over its threads.
#pragma once

#include "common.cuh"
#include "tc.cuh"

namespace omni {
namespace pfx {

// D (TMEM) = A (TMEM) x B (smem) [+ D]; issued by one thread.
OMNI_DEV void mma_bf16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

OMNI_DEV void tmem_ld32(uint32_t taddr, float* v) {
  uint32_t r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}

// 32 columns of this thread's lane without waiting (complete after tmem_wait_ld()).
OMNI_DEV void tmem_ld32_async(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}

// 2^x on the FMA and integer pipes, for x <= 127 (the softmax's arguments are at most 8): x = j + f with j the
// nearest integer (the 1.5 * 2^23 addition leaves j in the low mantissa bits of t) and f in [-0.5, 0.5]; 2^f from a
// cubic fitted here for relative error on [-0.5, 0.5] under the condition that it is 1 at 0 (1.02e-4 at most, far below
// bf16's 2^-9); 2^j added to the exponent field. x is clamped to -127, where the fields then cancel to exactly 0 (a masked
// key's weight must be zero: 2^-126 times the type's largest value is about 4); between -127 and -126 the result is a
// denormal below 2^-126. A NaN gives 0: what is not finite is carried into the row's sum (row_finite). Used for part of the
// probabilities, so that the special-function unit, which forms the others with ex2, is not the only pipe the
// exponentials load.
OMNI_DEV float ex2_fma(float x) {
  x = fmaxf(x, -127.f);
  const float t = x + 12582912.f;
  const float f = x - (t - 12582912.f);
  const float q = fmaf(fmaf(fmaf(0.05500906f, f, 0.24221097f), f, 0.6932829f), f, 1.f);
  return __uint_as_float(__float_as_uint(q) + (__float_as_uint(t) << 23));
}

// Packed pairs of floats for the f32x2 forms of fma / add (one instruction for two elements on the FMA pipe).
OMNI_DEV uint64_t f2_pack(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
OMNI_DEV void f2_unpack(uint64_t v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
OMNI_DEV uint64_t f2_fma(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
OMNI_DEV uint64_t f2_add(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
// Maxima that are NaN where an argument is.
OMNI_DEV float max3(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
OMNI_DEV float max2(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
// False where a row's scores, whose maximum this is, hold a NaN or +inf: the row has no softmax (NaN).
OMNI_DEV bool row_finite(float max) { return max < INFINITY; }

// Two floats rounded to bf16 and packed (lo in the low half).
OMNI_DEV uint32_t pack_bf16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

OMNI_DEV void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

OMNI_DEV void tmem_st32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}

OMNI_DEV void tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

OMNI_DEV void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

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

// Unit u -> (b, h, qt). The (row, head) pairs are taken in groups of `group`, and a group's units heaviest query
// tile first: the CTAs running at one time then read the K/V of about one group, which stays in L2.
OMNI_DEV void unit_of(int batch, int heads, int qtiles, int group, int u, int& b, int& h, int& qt) {
  const int bh_count = batch * heads;
  const int per_group = group * qtiles;
  const int g0 = (u / per_group) * group;
  const int gsize = min(group, bh_count - g0);
  const int r = u - g0 * qtiles;
  qt = qtiles - 1 - r / gsize;
  const int bh = g0 + r % gsize;
  b = bh / heads;
  h = bh % heads;
}

// A precomputed assignment of units to CTAs (kernel parameters): CTA c runs unit[start[c]] .. unit[start[c+1] - 1]
// in that order. The host builds it by list scheduling in the order unit_of numbers the units (each unit goes to
// the CTA that is free first, by a cost of its key tiles plus a unit's fixed cost), which keeps the CTAs' end times
// within about 1% where a round-robin assignment spreads them by 7-8% (config 4); the units a CTA runs at one time
// still belong to about one group. Shapes with more units than it holds, or grids larger than it covers, run
// round-robin (u = c, c + grid, ...).
constexpr int kSchedUnits = 4096;
constexpr int kSchedCtas = 160;
struct Sched {
  int on;
  uint16_t start[kSchedCtas + 1];
  uint16_t unit[kSchedUnits];
};

// The CTA's n-th unit, or -1 past its last.
OMNI_DEV int cta_unit(const Sched& s, int units, int n) {
  if (!s.on) {
    const int u = (int)blockIdx.x + n * (int)gridDim.x;
    return u < units ? u : -1;
  }
  const int k = (int)s.start[blockIdx.x] + n;
  return k < (int)s.start[blockIdx.x + 1] ? (int)s.unit[k] : -1;
}

// ---- packed sequences with grouped heads -----------------------------------------------------------------------------
// A unit's query tile holds `pos` consecutive positions of one kv head's G = heads / kv_heads query heads: tile row r is
// position r / G, head kv * G + r % G, so that the G heads share every key tile and a short sequence fills more of the
// 128 rows. Units are claimed by the CTAs as they become free (an atomic counter; the first by block index): sequences in
// order, each in groups of 16 kv heads, a group's longest query tiles first, so that the CTAs at work share keys in L2; but
// the last sequences, until they hold two units per CTA, as one, the longest units of all of them first: a last sequence
// of its own ends with one long unit on some CTAs and nothing on the others (8 prompts of 1400-1500, 8 heads of 512: 280
// against 268 us; all sequences as one lose the keys in L2, 16 heads of 128: 92 against 105).
// Claiming keeps the CTAs' end times together whatever the lengths, which the device alone knows; the warp that loads K
// claims, and hands the units to the other roles through a ring in shared memory. Where the units would leave half of the CTAs idle (a short chunk over many keys),
// each is cut into up to grid / units parts along its keys; a part leaves its maxima, sums and unnormalised output in fp32,
// and packed_join_kernel adds the parts up.
struct PackedSrc {
  const int64_t* q_offsets;
  const int64_t* k_offsets;
  int64_t q_tokens, k_tokens;
  int seqs, heads, kv_heads, group;  // group: query heads per kv head
  int pos;                           // positions per query tile
  unsigned pos_magic;                // ceil(2^32 / pos)
  unsigned* counters;                // [0] units claimed, [1] CTAs done: zero on entry and left zero
  int* meta;                         // null: no unit is cut. [0] units, [1] parts per unit; then PartMeta per unit
  float* parts;                      // [unit * parts per unit + part][(D + 2) * 128]: O [D][128 rows], maxima, sums
  const __nv_bfloat16 *q, *k, *v;    // for rows that need the exact form
  int64_t q_st, q_sh, k_st, k_sh, v_st, v_sh;
};

struct Unit {
  int b, h, qt;   // row, head, query tile; packed: parts per unit, kv head, parts of this unit
  int kt;         // key tiles (0: no more units)
  int q0, npos;   // packed: first token of the tile, positions in it
  int k0, lim0;   // first key token; keys the tile's first position sees (the next ones see one more each)
  int part;       // packed: the slot for this part's result, or -1: the unit is whole
};

// What packed_join_kernel needs of a unit: the parts there are and the unit as PackedWalk gives it.
struct PartMeta {
  int n, h, q0, npos, k0, lim0, pad[2];
};
constexpr int kMostParts = 16;

constexpr int kUnitRing = 3;
constexpr int kUnitHeads = 16;  // kv heads per scheduling group (as prefill_group)

// The claiming warp's place in the sequences: 32 of them at a time, one per lane.
struct PackedWalk {
  int s0;             // first sequence of the block in registers
  long long before;   // units of the sequences before it
  long long incl;     // units of the block's sequences up to this lane's
  int tiles;          // this lane's sequence: query tiles, first query / key token, queries, keys
  int q0, k0, lq, lk;
  int cut;            // parts per unit
  int w0;             // first lane of the group that is taken as one (32: none; only in the last block)
  int level;          // the group's units are found from the longest down: the key tiles in hand,
  long long above;    // and the group's units longer than that
  long long group;    // units of the group

  OMNI_DEV void load(const PackedSrc& p, int lane, int* status) {
    const int s = s0 + lane;
    tiles = 0;
    if (s < p.seqs) {
      const int64_t qa = p.q_offsets[s], qb = p.q_offsets[s + 1], ka = p.k_offsets[s], kb = p.k_offsets[s + 1];
      if (qa < 0 || qb < qa || qb > p.q_tokens || ka < 0 || kb < ka || kb > p.k_tokens) {
        raise_status(status, kStatusIndex);
      } else {
        q0 = (int)qa, lq = (int)(qb - qa), k0 = (int)ka, lk = (int)(kb - ka);
        tiles = (lq + p.pos - 1) / p.pos;
      }
    }
    long long c = (long long)tiles * p.kv_heads;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, c, o);
      if (lane >= o) c += y;
    }
    incl = c;
    w0 = 32;
    if (s0 + 32 >= p.seqs) {
      // The last sequences until they hold two units per CTA.
      const long long all = __shfl_sync(0xffffffffu, incl, 31);
      const unsigned in = __ballot_sync(0xffffffffu, all - incl < 2ll * gridDim.x && lk < (1 << 24));
      w0 = 32 - __clz(~in);  // the lanes from the top
      group = all - (w0 > 0 ? __shfl_sync(0xffffffffu, incl, (w0 - 1) & 31) : 0);
      level = (int)__reduce_max_sync(0xffffffffu, lane >= w0 && tiles > 0 ? (unsigned)max(1, (lk + 127) / 128) : 0u);
      above = 0;
    }
  }
  // This lane's query tiles of `l` key tiles and more, if it is of the group.
  OMNI_DEV int at_least(const PackedSrc& p, int lane, int l) const {
    if (lane < w0 || tiles == 0) return 0;
    if (l <= 1) return tiles;
    const int keys = 128 * (l - 1) + 1;  // tile qt sees min(lk, lk - lq + (qt + 1) pos) keys
    if (lk < keys) return 0;
    const int x = keys - (lk - lq);
    const int q = x <= 0 ? 0 : (p.pos == 1 ? x : (int)__umulhi((unsigned)(x + p.pos - 1), p.pos_magic)) - 1;
    return tiles - max(0, q);
  }
  OMNI_DEV void init(const PackedSrc& p, int lane, int* status) {
    before = 0;
    q0 = k0 = lq = lk = 0;
    cut = 1;
    if (p.meta) {  // few enough units that they may be cut: how many, and how long
      long long units = 0;
      int most = 0;
      for (s0 = 0; s0 < p.seqs; s0 += 32) {
        load(p, lane, nullptr);
        units += __shfl_sync(0xffffffffu, incl, 31);
        most = max(most, (int)__reduce_max_sync(0xffffffffu, tiles > 0 ? (unsigned)((lk + 127) / 128) : 0u));
      }
      const long long room = units > 0 ? (long long)gridDim.x / units : 1;
      cut = (int)max(1ll, min(min(room, (long long)kMostParts), (long long)(most / 2)));  // parts of two tiles at least
      if (blockIdx.x == 0 && lane == 0) {
        p.meta[0] = (int)units;
        p.meta[1] = cut;
      }
    }
    s0 = 0;
    load(p, lane, status);
  }
  // Part number `c` (ascending from call to call) of the units' parts; empty ones have kt = -1.
  OMNI_DEV Unit find_part(const PackedSrc& p, long long c, int lane, int* status) {
    if (cut == 1) return find(p, c, lane, status);
    const long long whole = c / cut;
    Unit r = find(p, whole, lane, status);
    if (r.kt == 0) return r;
    const int j = (int)(c - whole * cut), each = (r.kt + cut - 1) / cut;
    const int t0 = j * each, t1 = min(r.kt, t0 + each);
    if (t0 >= t1) {
      r.kt = -1;
      return r;
    }
    r.part = (int)c;
    r.b = cut;
    r.qt = (r.kt + each - 1) / each;
    r.k0 += t0 * 128;
    r.lim0 -= t0 * 128;
    r.kt = t1 - t0;
    return r;
  }
  // Unit number `u` (ascending from call to call); kt = 0 past the last. All lanes call it and get the same answer.
  OMNI_DEV Unit find(const PackedSrc& p, long long u, int lane, int* status) {
    Unit r;
    r.kt = 0;
    r.part = -1;
    for (;;) {
      if (w0 < 32) {
        const long long in_order = w0 > 0 ? __shfl_sync(0xffffffffu, incl, (w0 - 1) & 31) : 0;
        if (u >= before + in_order) return find_in_group(p, u - before - in_order, lane);
      }
      const unsigned hit = __ballot_sync(0xffffffffu, u < before + incl);
      if (!hit) {
        if (s0 + 32 >= p.seqs) return r;
        before += __shfl_sync(0xffffffffu, incl, 31);
        s0 += 32;
        load(p, lane, status);
        continue;
      }
      const int w = __ffs(hit) - 1;
      const int nt = __shfl_sync(0xffffffffu, tiles, w);
      int rem = (int)(u - before - (__shfl_sync(0xffffffffu, incl, w) - (long long)nt * p.kv_heads));
      const int sq = __shfl_sync(0xffffffffu, q0, w), sk = __shfl_sync(0xffffffffu, k0, w);
      const int nq = __shfl_sync(0xffffffffu, lq, w), nk = __shfl_sync(0xffffffffu, lk, w);
      const int hg = rem / (kUnitHeads * nt);
      rem -= hg * kUnitHeads * nt;
      const int gs = min(kUnitHeads, p.kv_heads - hg * kUnitHeads);
      fill(p, r, nt - 1 - rem / gs, hg * kUnitHeads + rem % gs, sq, sk, nq, nk);
      return r;
    }
  }
  OMNI_DEV void fill(const PackedSrc& p, Unit& r, int qt, int h, int sq, int sk, int nq, int nk) {
    r.h = h;
    r.b = 0;
    r.qt = qt;
    r.q0 = sq + qt * p.pos;
    r.npos = min(p.pos, nq - qt * p.pos);
    r.k0 = sk;
    r.lim0 = qt * p.pos + 1 + nk - nq;
    const int seen = r.lim0 + r.npos - 1;
    r.kt = seen > 128 ? (seen + 127) / 128 : 1;  // a tile that sees nothing still runs one (masked) key tile
  }
  // Unit number `u` of the group (ascending from call to call): levels from the longest down, within a level the lanes'
  // sequences in order, within a sequence tile by tile, the heads innermost.
  OMNI_DEV Unit find_in_group(const PackedSrc& p, long long u, int lane) {
    Unit r;
    r.kt = 0;
    r.part = -1;
    if (u >= group) return r;
    int longer, mine;  // this lane's tiles above the level, and of it and above
    for (;; --level) {
      longer = at_least(p, lane, level + 1);
      mine = at_least(p, lane, level);
      const long long n = (long long)__reduce_add_sync(0xffffffffu, (unsigned)(mine - longer)) * p.kv_heads;
      if (u < above + n) break;
      above += n;
    }
    int upto = mine - longer;  // tiles of the level up to this lane's
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += y;
    }
    const int rem = (int)(u - above);
    const int tile = rem / p.kv_heads;
    const int w = __ffs(__ballot_sync(0xffffffffu, tile < upto)) - 1;
    const int in_lane = tile - __shfl_sync(0xffffffffu, upto - (mine - longer), w);
    const int qt = __shfl_sync(0xffffffffu, tiles - longer, w) - 1 - in_lane;
    fill(p, r, qt, rem - tile * p.kv_heads, __shfl_sync(0xffffffffu, q0, w), __shfl_sync(0xffffffffu, k0, w),
         __shfl_sync(0xffffffffu, lq, w), __shfl_sync(0xffffffffu, lk, w));
    return r;
  }
};

// BadValues of ND head dims from d0 on, by one warp; a lane looks at a key.
template <int ND>
__device__ __noinline__ BadValues bad_values(const __nv_bfloat16* v, int64_t v_st, int from, int end, int d0) {
  auto bad = [&](int j) {
    const uint4* row = reinterpret_cast<const uint4*>(v + j * v_st + d0);
    uint32_t any = 0u;
#pragma unroll 8
    for (int i = 0; i < ND / 8; ++i) {
      const uint4 u = __ldg(row + i);
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int c = 0; c < 4; ++c) {  // a half whose exponent bits are all ones
        const uint32_t z = ~w[c] & 0x7f807f80u;
        any |= (z - 0x00010001u) & ~z & 0x80008000u;
      }
    }
    return any != 0u;
  };
  return find_bad(from, end, bad);
}
// Attention of one query row over its first `lim` keys, by one warp, straight from the formula: ND head dims from d0 on,
// into out[d0 ..], for the rows of must_redo. Keys past `lim` are not read. Rare, so it only has to be right.
template <int D, int ND>
__device__ __noinline__ void exact_row(const __nv_bfloat16* q, const __nv_bfloat16* k, int64_t k_st, const __nv_bfloat16* v,
                                       int64_t v_st, int lim, float qscale, __nv_bfloat16* out, int d0) {
  constexpr int N = D / 32, NO = ND / 32;
  const int lane = threadIdx.x & 31;
  v += d0;
  out += d0;
  float qv[N], o[NO], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) qv[i] = __bfloat162float(q[i * 32 + lane]);
#pragma unroll
  for (int i = 0; i < NO; ++i) o[i] = 0.f;
  for (int j0 = 0; j0 < lim; j0 += 4) {  // four keys' loads in flight
    __nv_bfloat16 kv[4][N], vv[4][NO];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int64_t j = min(j0 + c, lim - 1);
#pragma unroll
      for (int i = 0; i < N; ++i) kv[c][i] = k[j * k_st + i * 32 + lane];
#pragma unroll
      for (int i = 0; i < NO; ++i) vv[c][i] = v[j * v_st + i * 32 + lane];
    }
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      if (j0 + c >= lim) break;
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < N; ++i) s = fmaf(qv[i], __bfloat162float(kv[c][i]), s);
#pragma unroll
      for (int w = 16; w > 0; w >>= 1) s += __shfl_xor_sync(0xffffffffu, s, w);
      s *= qscale;
      const float mn = s > m ? s : m;
      const float base = mn == -INFINITY ? 0.f : mn;
      const float f = ex2(m - base), pr = ex2(s - base);
      m = mn;
      l = fmaf(l, f, pr);
#pragma unroll
      for (int i = 0; i < NO; ++i) o[i] = fmaf(pr, __bfloat162float(vv[c][i]), o[i] * f);
    }
    if (l != l) break;  // a NaN score: the whole row is NaN
  }
  const float inv = l != 0.f ? 1.f / l : (lim > 0 ? NAN : 0.f);  // every key it sees scores -inf: no softmax
#pragma unroll
  for (int i = 0; i < NO; ++i) out[i * 32 + lane] = __float2bfloat16_rn(l != l ? l : o[i] * inv);
}

// Rows `rows` (a bit each, from tile row row0 on) of a unit that are not finite: redone where must_redo says so. One warp.
template <int D, int ND>
__device__ __noinline__ void redo_rows(const PackedSrc& src, unsigned rows, int row0, int q0, int k0, int lim0, int h, int kt,
                                       float qscale, __nv_bfloat16* out, int d0) {
  const __nv_bfloat16* k = src.k + k0 * src.k_st + h * src.k_sh;
  const __nv_bfloat16* v = src.v + k0 * src.v_st + h * src.v_sh;
  const int end = (int)min((int64_t)kt * 128, src.k_tokens - k0);
  const BadValues bad = bad_values<ND>(v, src.v_st, max(lim0, 0), end, d0);
  for (; rows; rows &= rows - 1) {
    const int row = row0 + __ffs(rows) - 1, pos = row / src.group, head = h * src.group + row - pos * src.group;
    if (!must_redo(bad, lim0 + pos)) continue;
    const int64_t tok = q0 + pos;
    exact_row<D, ND>(src.q + tok * src.q_st + head * src.q_sh, k, src.k_st, v, src.v_st, lim0 + pos, qscale,
                     out + (tok * src.heads + head) * D, d0);
  }
}

// Such rows of a CTA's units, up to 32 units per warp (a lane holds one): they may take longer than the other roles wait for the
// epilogue, so they are redone when the CTA's units are done.
struct RedoList {
  unsigned rows = 0;
  int q0, k0, lim0, h, kt;
  int count = 0;
  OMNI_DEV bool add(const Unit& u, unsigned rows_, int lane) {  // true: the list is full
    if (lane == count) rows = rows_, q0 = u.q0, k0 = u.k0, lim0 = u.lim0, h = u.h, kt = u.kt;
    return ++count == 32;
  }
  template <int D>
  OMNI_DEV void run(const PackedSrc& src, int row0, float qscale, __nv_bfloat16* out) {
    __syncwarp();  // the rows' first results are written before they are written again
    for (int i = 0; i < count; ++i)
      redo_rows<D, D>(src, __shfl_sync(0xffffffffu, rows, i), row0, __shfl_sync(0xffffffffu, q0, i),
                      __shfl_sync(0xffffffffu, k0, i), __shfl_sync(0xffffffffu, lim0, i), __shfl_sync(0xffffffffu, h, i),
                      __shfl_sync(0xffffffffu, kt, i), qscale, out, 0);
    count = 0;
  }
};

}  // namespace pfx

// (row, head) pairs per scheduling group of the prefill kernels (prefill.cu).
int prefill_group(int bh_count);

// The list schedule of a prefill's units over `grid` CTAs (cached per shape; prefill.cu), or nullptr where the
// shape is past what a schedule holds: then the kernels run round-robin (prefill_round_robin()).
const pfx::Sched* prefill_schedule(int batch, int heads, int qtiles, int group, int grid);
const pfx::Sched& prefill_round_robin();

// The packed kernels' tensor maps (boxes of 128 keys, v_rows of V; false where a stride has none), unit source and grid
// (prefill.cu).
struct PackedArgs;
bool packed_maps(const PackedArgs& a, int positions, int v_rows, CUtensorMap* q, CUtensorMap* k, CUtensorMap* v);
pfx::PackedSrc packed_source(const PackedArgs& a, int positions);
int packed_grid(const PackedArgs& a, int positions);
int packed_cut_units();
cudaError_t launch_packed_join(const PackedArgs& a, const pfx::PackedSrc& src, cudaStream_t stream);

}  // namespace omni
