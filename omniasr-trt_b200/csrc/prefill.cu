// Causal prefill attention on the 5th-generation tensor cores (tcgen05 + TMEM), bf16: dense rows of head_dim 128, and packed
// sequences with grouped heads of head_dim 64 and 128 (PackedSrc, prefill_common.cuh; packed.cu has the formula).
//
// out[b, w, h] = softmax(q[b, h, w] . k[b, h, :w+1]^T * scale) . v[b, h, :w+1]   for w < W
// (F.scaled_dot_product_attention(q, k, v, is_causal=True) of the reference's prefill, decode.py:171; the
// reference-semantics form is modeling.py:398-399). Right-padded rows need nothing special: a valid query never
// sees a later (pad) key.
//
// Work unit: (row b, head h, 128-query tile qt) over key tiles 0..qt; units are taken by a persistent grid of one
// CTA per SM in groups of (b, h) pairs, heaviest first within a group (unit_of). Roles (512 threads):
//   warp 12 TMA: the K tiles (3-slot ring, two 64-column boxes each, 128-byte swizzle); warp 14 TMA: the V tiles;
//           the query tiles (2 slots) are loaded two units ahead by the first epilogue thread
//   warp 13 MMA: S = Q K^T into TMEM (M=128 queries, N=128 keys), triple-buffered, so that S(t + 3) needs only
//           O += P(t) V to have completed and the scores are ready before the softmax asks for them;
//   warp 15 MMA: O += P V with P read from TMEM (the tcgen05 "A in TMEM" form). Two issuing warps, because one
//           thread issues a tcgen05.mma in about 55 clocks at best (measured), while a 128x128x16 MMA takes the
//           tensor core about 64: a single issuer with its waits left the tensor core idle half the time. Each runs
//           converged with one elected lane issuing, its descriptors warp-uniform (12 packed prompts of 60 to 2047
//           tokens 172 -> 166 us, dense 752 -> 770 TFLOP/s over a lone thread).
//   warps 0-3 / 4-7  softmax warpgroups x = 0 / 1: thread t of warpgroup x owns query row t and the keys 64x .. 64x+63
//           of every tile, so twice the softmax warps per SM each form half a tile's exponentials. The two keep one
//           running max per row: each tile one barrier over both warpgroups asks whether any row's scores pass its
//           max by 2^8 (log2 units); only then are the tile maxima exchanged, the max raised and O rescaled in TMEM
//           (each warpgroup its 64 head dims). P (bf16 pairs) is written over the warpgroup's half of S in TMEM.
//           The scale-and-subtract and the row sums use the packed f32x2 FMA / add (two elements per instruction),
//           and one probability pair in four is exponentiated on the FMA pipe (ex2_fma) instead of the
//           special-function unit, which the exponentials otherwise saturate.
//   warps 8-11 epilogue: O / (l_0 + l_1) of each unit as bf16 rows, while the softmax warpgroups go on with the next.
// What bounds it: the softmax's chain. At head_dim 128 a tile is 1024 clocks of the tensor core and took 1930: 165 until the
// wait sees S, 120 to read it, 300 for maxima and the barrier, 1000 for the exponentials (768 of them the special-function
// unit's), the rest stores and hand-over. More of them on the FMA pipe (one pair in two: 172 -> 180 us) lose. Long calls
// are held by the power limit besides.
// TMEM: S0 [0,128) S1 [128,256) S2 [256,384) O [384,512); P of S buffer j, half x at 128j + 64x .. +32.

#include <cudaTypedefs.h>
#include <math.h>

#include <array>
#include <map>
#include <memory>
#include <mutex>
#include <queue>
#include <type_traits>
#include <vector>

#include "attention.cuh"
#include "prefill.cuh"
#include "paged.cuh"
#include "prefill_common.cuh"
#include "tc.cuh"
#include "trace.cuh"

namespace omni {
namespace prefill {

using namespace pfx;

constexpr int BM = 128;  // queries per tile
constexpr int BN = 128;  // keys per tile
constexpr int BOX = BN * 64 * 2;
// What depends on the head dim: 128, or 64 (packed sequences; half the bytes per tile, so twice the tiles in flight).
template <int D>
struct Cfg {
  static constexpr int TILE = BN * D * 2;
  static constexpr int QS = 2, KS = D == 64 ? 5 : 3, VS = D == 64 ? 6 : 2;  // query tiles (two units), K and V rings
  static constexpr int Q_OFF = 0;
  static constexpr int K_OFF = Q_OFF + QS * TILE;
  static constexpr int V_OFF = K_OFF + KS * TILE;
  static constexpr int SMEM_BYTES = V_OFF + VS * TILE;
};
constexpr int NSB = 3;  // S buffers in TMEM: S(t + 3) needs only O += P(t) V to have completed
constexpr int NWG = 2;        // softmax warpgroups; warpgroup x owns keys KW x .. KW x + KW - 1 of every tile
constexpr int KW = BN / NWG;  // keys per softmax warpgroup (a multiple of the 16-key MMA step)
constexpr int W_EPI = 4 * NWG, W_LOADK = W_EPI + 4, W_MMA = W_LOADK + 1, W_LOADV = W_LOADK + 2, W_MMA_PV = W_LOADK + 3;
constexpr int THREADS = 32 * (W_MMA_PV + 1);  // softmax, Q loader + epilogue, K loads, S MMAs, V loads, PV MMAs
constexpr int SM_THREADS = 128 * NWG;
constexpr uint32_t TMEM_COLS = 512;
constexpr uint32_t COL_S = 0, COL_O = 384;  // S buffer j at 128 j
constexpr uint32_t IDESC_S = idesc_bf16(BM, BN, 0, 0);
constexpr float kRescale = 8.f;
#ifndef OMNI_PREFILL_POLY_EVERY
#define OMNI_PREFILL_POLY_EVERY 4
#endif
constexpr int kPolyEvery = OMNI_PREFILL_POLY_EVERY;  // probabilities of one pair in this many by ex2_fma

struct Params {
  int batch, heads, width, qtiles;
  int group;  // (row, head) pairs per scheduling group
  float qscale;  // scale * log2(e)
  const __nv_bfloat16* q;
  int64_t q_sb, q_sh, q_sw;  // q[b, h, w, :] strides (elements)
  __nv_bfloat16* out;
  int64_t out_sb, out_sw, out_sh;  // out[b, w, h, :] strides (elements)
  int* status;
};

OMNI_DEV void unit_of(const Params& p, int u, int& b, int& h, int& qt) {
  pfx::unit_of(p.batch, p.heads, p.qtiles, p.group, u, b, h, qt);
}

// The CTA's control block: barriers, the row maxima exchanged between the softmax warpgroups, the unit's row sums
// for the epilogue, flags. One static struct, padded to 1024 bytes, so that the dynamic tile ring after it starts
// 1024-aligned (the kernel checks, and reports status bit 4 otherwise).
template <int D>
struct alignas(1024) Ctl {
  static constexpr int QS = Cfg<D>::QS, KS = Cfg<D>::KS, VS = Cfg<D>::VS;
  uint64_t k_full[KS], k_empty[KS], v_full[VS], v_empty[VS], q_full[QS], q_empty[QS];
  uint64_t s_full[NSB], p_full[NWG][NSB], pv_done[NSB], o_ready, o_free, l_full, l_free, drain;
  float tmax[NWG][BM];  // [warpgroup][row]: a tile's scaled row maxima, on the rare tiles that raise a max
  float msum[BM];       // [row]: the maximum of a unit's part
  float lsum[NWG][BM];  // [warpgroup][row]: the unit's row sums for the epilogue
  uint32_t tmem_base;
  int abort_flag, issued_k, issued_v, issued_q;  // loads the producers issued
  uint64_t u_full[kUnitRing], u_empty[kUnitRing];  // packed: the units claimed, for all roles
  Unit unit[kUnitRing];
};
static_assert(sizeof(Ctl<128>) + Cfg<128>::SMEM_BYTES <= 232448 && sizeof(Ctl<64>) + Cfg<64>::SMEM_BYTES <= 232448,
              "shared memory per block");
static_assert(NSB * 128 + 128 <= TMEM_COLS, "S buffers and O in TMEM");

// Src: Sched (dense rows) or PackedSrc (packed sequences with grouped heads).
template <typename Src, int D>
__global__ void __launch_bounds__(THREADS, 1)
    prefill_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                   const __grid_constant__ CUtensorMap vmap, const Params p, const __grid_constant__ Src src) {
  constexpr bool PACKED = std::is_same_v<Src, PackedSrc>;
  using C = Cfg<D>;
  constexpr int TILE = C::TILE, QS = C::QS, KS = C::KS, VS = C::VS, Q_OFF = C::Q_OFF, K_OFF = C::K_OFF, V_OFF = C::V_OFF;
  constexpr int DW = D / NWG;  // head dims of O each softmax warpgroup rescales
  constexpr uint32_t IDESC_O = idesc_bf16(BM, D, 0, 1);
  extern __shared__ __align__(1024) unsigned char smem[];
  __shared__ Ctl<D> ctl;
  uint64_t *k_full = ctl.k_full, *k_empty = ctl.k_empty, *v_full = ctl.v_full, *v_empty = ctl.v_empty;
  uint64_t *q_full = ctl.q_full, *q_empty = ctl.q_empty, *s_full = ctl.s_full, *pv_done = ctl.pv_done;
  uint64_t(*p_full)[NSB] = ctl.p_full;
  uint64_t &o_ready = ctl.o_ready, &o_free = ctl.o_free, &l_full = ctl.l_full, &l_free = ctl.l_free;
  uint64_t& drain = ctl.drain;
  volatile int& abort_flag = ctl.abort_flag;
  volatile int &issued_k = ctl.issued_k, &issued_v = ctl.issued_v, &issued_q = ctl.issued_q;

  const int tid = threadIdx.x;
  const int warp = tid >> 5;
  const int lane = tid & 31;
  const int units = p.batch * p.heads * p.qtiles;
  if (!PACKED && (int)blockIdx.x >= units) return;
  if (smem_addr(smem) & 1023u) {  // the swizzled tiles need a 1024-aligned ring
    if (tid == 0) raise_status(p.status, kStatusLayout);
    return;
  }

  if (tid == 0) {
    for (int s = 0; s < KS; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&k_empty[s], 1);
    }
    for (int s = 0; s < VS; ++s) {
      mbar_init(&v_full[s], 1);
      mbar_init(&v_empty[s], 1);
    }
    for (int j = 0; j < QS; ++j) {
      mbar_init(&q_full[j], 1);
      mbar_init(&q_empty[j], 1);
    }
    for (int j = 0; j < NSB; ++j) {
      mbar_init(&s_full[j], 1);
      mbar_init(&pv_done[j], 1);
      for (int x = 0; x < NWG; ++x) mbar_init(&p_full[x][j], 128);
    }
    mbar_init(&o_ready, 1);
    mbar_init(&o_free, 128);
    mbar_init(&l_full, SM_THREADS);
    mbar_init(&l_free, 128);
    mbar_init(&drain, 2);
    if (PACKED) {
      for (int j = 0; j < kUnitRing; ++j) {
        mbar_init(&ctl.u_full[j], 1);
        mbar_init(&ctl.u_empty[j], 3 + 4 * NWG + 4);  // V loads, S and P V issuers; softmax and epilogue warps
      }
    }
    mbar_fence_init();
    abort_flag = 0;
    issued_k = issued_v = issued_q = 0;
  }
  if (warp == W_EPI) tmem_alloc(&ctl.tmem_base, TMEM_COLS);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  grid_dependency_wait();  // q, k, v may come from the kernel before (launched as a programmatic dependent)
  if (tid == 0) OMNI_TRACE_AT(1599);
  OMNI_TRACE_CTA(0);
  const uint32_t tbase = ctl.tmem_base;
  // Every wait gives up at once when another role has given up (abort_flag), else after the bounded time.
  auto wait = [&](uint64_t* bar, uint32_t parity) -> bool {
    if (mbar_wait_or(bar, parity, &abort_flag)) return true;
    abort_flag = 1;
    return false;
  };
  // The CTA's n-th unit; false past its last (or, packed, after an abort). put: this role (or warp) is done with it.
  auto get = [&](int n, Unit& u) -> bool {
    if constexpr (PACKED) {
      if (!wait(&ctl.u_full[n % kUnitRing], (n / kUnitRing) & 1)) return false;
      u = ctl.unit[n % kUnitRing];
      return u.kt > 0;
    } else {
      const int i = cta_unit(src, units, n);
      if (i < 0) return false;
      unit_of(p, i, u.b, u.h, u.qt);
      u.kt = u.qt + 1;
      return true;
    }
  };
  // The same for a warp that runs converged: its lanes leave their waits together, with one answer, so that none is still at
  // a barrier that the MMAs issued next move on.
  auto wwait = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, wait(bar, parity)) != 0; };
  auto wget = [&](int n, Unit& u) { return __all_sync(0xffffffffu, get(n, u)) != 0; };
  auto put = [&](int n) {
    if constexpr (PACKED) mbar_arrive(&ctl.u_empty[n % kUnitRing]);
  };

  if (PACKED && warp == W_LOADK) {
    // ------------------------------------------------------------------ packed: claims, query and K loads
    if constexpr (PACKED) {
      if (lane == 0) {
        prefetch_tmap(&qmap);
        prefetch_tmap(&kmap);
      }
      PackedWalk walk;
      walk.init(src, lane, blockIdx.x == 0 ? p.status : nullptr);
      int tile = 0;
      long long next = blockIdx.x;
      for (int n = 0;; ++n) {
        const Unit u = walk.find_part(src, next, lane, blockIdx.x == 0 ? p.status : nullptr);
        if (u.kt < 0) {  // a part without keys
          unsigned c = 0;
          if (lane == 0) c = atomicAdd(src.counters, 1u);
          next = (long long)gridDim.x + __shfl_sync(0xffffffffu, c, 0);
          --n;
          continue;
        }
        bool ok = true;
        unsigned claim = 0;
        if (lane == 0) {
          const int us = n % kUnitRing;
          ok = n < kUnitRing || wait(&ctl.u_empty[us], (n / kUnitRing - 1) & 1);
          if (ok) {
            ctl.unit[us] = u;
            mbar_arrive(&ctl.u_full[us]);
          }
          if (ok && u.kt > 0) {
            const int qslot = n % QS;
            ok = n < QS || wait(&q_empty[qslot], (n / QS - 1) & 1);
            if (ok) {
              mbar_arrive_expect_tx(&q_full[qslot], (uint32_t)(src.group * src.pos * D * 2));
#pragma unroll
              for (int x = 0; x < D / 64; ++x)
                tma_load_4d(smem + Q_OFF + qslot * TILE + x * BOX, &qmap, 64 * x, 0, u.h, u.q0, &q_full[qslot]);
              issued_q = n + 1;
            }
            for (int kt = 0; kt < u.kt && ok; ++kt, ++tile) {
              // The next unit is claimed near the end of this one, so that no CTA holds units it starts late.
              if (kt == max(0, u.kt - 3)) claim = atomicAdd(src.counters, 1u);
              const int slot = tile % KS, use = tile / KS;
              if (use >= 1 && !wait(&k_empty[slot], (use - 1) & 1)) {
                ok = false;
                break;
              }
              mbar_arrive_expect_tx(&k_full[slot], TILE);
#pragma unroll
              for (int x = 0; x < D / 64; ++x)
                tma_load_4d(smem + K_OFF + slot * TILE + x * BOX, &kmap, 64 * x, u.k0 + kt * BN, u.h, 0, &k_full[slot]);
              issued_k = tile + 1;
            }
          }
        }
        ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
        if (!ok || u.kt == 0 || __any_sync(0xffffffffu, abort_flag != 0)) break;
        tile = __shfl_sync(0xffffffffu, tile, 0);
        next = (long long)gridDim.x + __shfl_sync(0xffffffffu, claim, 0);
      }
      if (lane == 0) {
        // The last CTA to stop claiming leaves the counters zero.
        if (atomicAdd(src.counters + 1, 1u) == gridDim.x - 1) {
          src.counters[0] = 0;
          src.counters[1] = 0;
        }
      }
    }
    __syncwarp();
  } else if (warp == W_LOADK || warp == W_LOADV) {
    // ------------------------------------------------------------------ producers
    if (lane == 0) {
      const bool is_k = warp == W_LOADK;
      const CUtensorMap* map = is_k ? &kmap : &vmap;
      prefetch_tmap(map);
      const int ns = is_k ? KS : VS;
      unsigned char* ring = smem + (is_k ? K_OFF : V_OFF);
      uint64_t* full = is_k ? k_full : v_full;
      uint64_t* empty = is_k ? k_empty : v_empty;
      int tile = 0;
      Unit u;
      for (int n = 0; get(n, u) && !abort_flag; ++n) {
        const int row0 = PACKED ? u.k0 : 0, b = PACKED ? 0 : u.b;
        for (int kt = 0; kt < u.kt && !abort_flag; ++kt, ++tile) {
          const int slot = tile % ns, use = tile / ns;
          if (use >= 1 && !wait(&empty[slot], (use - 1) & 1)) break;
          mbar_arrive_expect_tx(&full[slot], TILE);
#pragma unroll
          for (int x = 0; x < D / 64; ++x)
            tma_load_4d(ring + slot * TILE + x * BOX, map, 64 * x, row0 + kt * BN, u.h, b, &full[slot]);
          if (is_k) issued_k = tile + 1;
          else issued_v = tile + 1;
          OMNI_TRACE_AT(tile * 8 + (is_k ? 0 : 1));
        }
        put(n);
      }
    }
    __syncwarp();
  } else if (warp == W_MMA) {
    // ------------------------------------------------------------------ S issuer: S[t % NSB] = Q K(t)^T
    // S[t % NSB] is free once O += P(t - NSB) V has completed (P(t - NSB) lies over it); the unit's Q slot is
    // released after its last S (q_empty). Both issuing warps run converged, one elected lane issuing, so that the
    // descriptors are warp-uniform.
    {
      const bool leader = elect_one();
      // Slot s's descriptor is slot 0's with the start address (in 16-byte units, 14 bits) moved on by s tiles.
      const uint64_t kdesc0 = smem_desc(smem_addr(smem + K_OFF), 16, 1024, kLayoutSw128);
      const uint64_t qdesc0 = smem_desc(smem_addr(smem + Q_OFF), 16, 1024, kLayoutSw128);
      int tile = 0, nunit = 0, sb = 0;
      bool ok = true;
      Unit u;
      for (; wget(nunit, u) && ok; ++nunit) {
        const int qslot = nunit % QS;
        if (!wwait(&q_full[qslot], (nunit / QS) & 1)) break;
        const uint64_t qd = qdesc0 + (uint64_t)(qslot * (TILE >> 4));
        for (int kt = 0; kt < u.kt; ++kt, ++tile, sb = sb == NSB - 1 ? 0 : sb + 1) {
          const int slot = tile % KS;
          if (tile >= NSB && !wwait(&pv_done[sb], ((tile - NSB) / NSB) & 1)) {
            ok = false;
            break;
          }
          if (!wwait(&k_full[slot], (tile / KS) & 1)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t dcol = tbase + COL_S + sb * 128;
          const uint64_t kd = kdesc0 + (uint64_t)(slot * (TILE >> 4));
          if (leader) {
#pragma unroll
            for (int kk = 0; kk < D / 16; ++kk) {
              const uint64_t off = (uint64_t)((((kk >> 2) * BOX + (kk & 3) * 32) >> 4));
              mma_bf16_ss(dcol, qd + off, kd + off, IDESC_S, kk > 0 ? 1u : 0u);
            }
            tc_commit(&s_full[sb]);
            tc_commit(&k_empty[slot]);
            if (kt == u.kt - 1) tc_commit(&q_empty[qslot]);  // the unit's last read of its query tile
            OMNI_TRACE_AT(tile * 8 + 2);
          }
        }
        if (leader) put(nunit);
      }
    }
  } else if (warp == W_MMA_PV) {
    // ------------------------------------------------------------------ PV issuer: O += P(t) V(t)
    // The two key halves in turn, as their softmax warpgroups finish; a unit's first tile overwrites O once the
    // epilogue has read the previous unit's (o_free).
    {
      const bool leader = elect_one();
      const uint64_t vdesc0 = smem_desc(smem_addr(smem + V_OFF), BOX, 1024, kLayoutSw128);
      int tile = 0, nunit = 0;
      bool ok = true;
      Unit u;
      for (; wget(nunit, u) && ok; ++nunit) {
        for (int kt = 0; kt < u.kt; ++kt, ++tile) {
          const int pb = tile % NSB, pu = tile / NSB;
          const int slot = tile % VS;
          if (kt == 0 && nunit >= 1 && !wwait(&o_free, (nunit - 1) & 1)) {
            ok = false;
            break;
          }
          if (!wwait(&v_full[slot], (tile / VS) & 1)) {
            ok = false;
            break;
          }
          const uint64_t vd = vdesc0 + (uint64_t)(slot * (TILE >> 4));
          const uint32_t pcol = tbase + COL_S + pb * 128;
#pragma unroll
          for (int x = 0; x < NWG; ++x) {
            if (!wwait(&p_full[x][pb], pu & 1)) {
              ok = false;
              break;
            }
            tc_fence_after();
            if (leader) {
#pragma unroll
              for (int kk = 0; kk < KW / 16; ++kk)
                mma_bf16_ts(tbase + COL_O, pcol + x * KW + kk * 8, vd + (uint64_t)((KW / 16 * x + kk) * 128), IDESC_O,
                            (kt == 0 && x == 0 && kk == 0) ? 0u : 1u);
            }
          }
          if (!ok) break;
          if (leader) {
            tc_commit(&pv_done[pb]);
            tc_commit(&v_empty[slot]);
            OMNI_TRACE_AT(tile * 8 + 3);
          }
        }
        if (leader) {
          if (ok) tc_commit(&o_ready);
          put(nunit);
        }
      }
    }
    __syncwarp();
  } else if (warp < W_EPI) {
    // ------------------------------------------------------------------ softmax, keys KW x .. of every tile
    // The warpgroups leave their loops only on a decision taken at a barrier over all their threads, so that no
    // thread waits at a barrier the others have left: a wait that gives up sets abort_flag and the thread goes on
    // to the tile's barrier, where every thread sees it.
    const int x = warp >> 2;
    const int row = tid & 127;  // query row within the tile = TMEM lane
    const uint32_t lane_off = (uint32_t)(32 * (warp & 3)) << 16;
    const uint32_t col_o = tbase + lane_off + COL_O + x * DW;  // this warpgroup's head dims of O (rescale)
    int row_pos = 0;  // packed: the row's position within the tile
    if constexpr (PACKED) row_pos = row / src.group;
    int tile = 0, nunit = 0;
    bool quit = false;
    for (; !quit; ++nunit) {
      Unit u;
      const bool more = get(nunit, u);
      if constexpr (PACKED) {  // the claim's wait may have given up in some threads: decided by all of them
        if (sync_or(1, SM_THREADS, abort_flag != 0)) break;
      }
      if (!more) break;
      __syncwarp();
      if (PACKED && lane == 0) put(nunit);
      float m = -INFINITY, l = 0.f;
      for (int kt = 0; kt < u.kt; ++kt, ++tile) {
        const int sb = tile % NSB;
        if (row == 0 && x == 0 && tile < 300) OMNI_TRACE_AT(2400 + 1200 + tile);
        wait(&s_full[sb], (tile / NSB) & 1);
        if (row == 0 && x < 2) OMNI_TRACE_AT(tile * 8 + 4 + 2 * x);
        tc_fence_after();
        __syncwarp();
        const uint32_t scol = tbase + lane_off + COL_S + sb * 128 + x * KW;
        uint32_t raw[KW];
#pragma unroll
        for (int c = 0; c < KW / 32; ++c) tmem_ld32_async(scol + 32 * c, raw + 32 * c);
        tmem_wait_ld();
        if (row == 0 && x == 0 && tile < 400) OMNI_TRACE_AT(2400 + tile * 4);
        float v[KW];
#pragma unroll
        for (int i = 0; i < KW; ++i) v[i] = __uint_as_float(raw[i]);
        if constexpr (PACKED) {
          if ((kt + 1) * BN > u.lim0) {  // some row does not see all of the tile
            const int lim = u.lim0 + row_pos - kt * BN - x * KW;  // keys of the warpgroup's half that the row sees
#pragma unroll
            for (int i = 0; i < KW; ++i)
              if (i >= lim) v[i] = -INFINITY;
          }
        } else if (kt == u.kt - 1) {  // the diagonal tile: keys past the query
#pragma unroll
          for (int i = 0; i < KW; ++i)
            if (x * KW + i > row) v[i] = -INFINITY;
        }
        static_assert(KW % 16 == 0, "row max in 8 partials of two values per step");
        float part[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) part[j] = v[j];
#pragma unroll
        for (int i = 8; i < KW; i += 16)
#pragma unroll
          for (int j = 0; j < 8; ++j) part[j] = max3(part[j], v[i + j], v[i + 8 + j]);
        const float tmax = max3(max3(part[0], part[1], part[2]), max3(part[3], part[4], part[5]),
                                max2(part[6], part[7])) * p.qscale;
        // One barrier per tile over the warpgroups: does any row need a higher max (or has a NaN), or has any thread seen an abort?
        const bool saw_abort = abort_flag != 0;
        float mnew = m;
        bool slow = false;
        const bool any_raise = sync_or(1, SM_THREADS, !(tmax <= m + kRescale) || saw_abort);
        if (row == 0 && x == 0 && tile < 400) OMNI_TRACE_AT(2401 + tile * 4);
        if (any_raise) {
          if (sync_or(1, SM_THREADS, saw_abort)) {
            quit = true;
            break;
          }
          ctl.tmax[x][row] = tmax;
          if (!row_finite(tmax)) l = NAN;
          named_sync(2, SM_THREADS);
          float t2 = ctl.tmax[0][row];  // the same in every warpgroup
#pragma unroll
          for (int y = 1; y < NWG; ++y) t2 = fmaxf(t2, ctl.tmax[y][row]);
          if (t2 > m + kRescale) mnew = t2;
          slow = true;
        }
        // Probabilities (bf16 pairs) over this warpgroup's keys, and the row sum; formed before any rescale of O, so
        // that the scores are dead by then (register pressure).
        // Packed rows may have seen no key yet (or never see one): their probabilities are 2^(-inf - 0) = 0.
        const float mref = PACKED && mnew == -INFINITY ? 0.f : mnew;
        uint32_t w[KW / 2];
        uint64_t ls2[4];  // row-sum partials, two per packed register
#pragma unroll
        for (int j = 0; j < 4; ++j) ls2[j] = 0ull;
        const uint64_t sc2 = f2_pack(p.qscale, p.qscale), nm2 = f2_pack(-mref, -mref);
#pragma unroll
        for (int i = 0; i < KW / 2; ++i) {
          // x = s * scale - max for a pair in one packed FMA; one pair in kPolyEvery exponentiated on the FMA pipe,
          // the rest on the special-function unit.
          float x0, x1;
          f2_unpack(f2_fma(f2_pack(v[2 * i], v[2 * i + 1]), sc2, nm2), x0, x1);
          const bool poly = i % kPolyEvery == kPolyEvery - 1;
          const float p0 = poly ? ex2_fma(x0) : ex2(x0);
          const float p1 = poly ? ex2_fma(x1) : ex2(x1);
          ls2[i & 3] = f2_add(ls2[i & 3], f2_pack(p0, p1));
          w[i] = pack_bf16x2(p0, p1);
        }
        float ls[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) f2_unpack(ls2[j], ls[2 * j], ls[2 * j + 1]);
        if (slow) {
          const bool rescale = mnew != m && kt > 0;
          if (__any_sync(0xffffffffu, rescale)) {
            wait(&pv_done[(tile - 1) % NSB], ((tile - 1) / NSB) & 1);  // O holds every earlier tile
            tc_fence_after();
            __syncwarp();
            const float sc = rescale ? ex2(m - mnew) : 1.f;
#pragma unroll
            for (int c = 0; c < DW / 32; ++c) {
              float o[32];
              uint32_t ow[32];
              tmem_ld32(col_o + c * 32, o);
#pragma unroll
              for (int i = 0; i < 32; ++i) ow[i] = __float_as_uint(o[i] * sc);
              tmem_st32(col_o + c * 32, ow);
            }
            tmem_wait_st();
            l *= sc;
          }
          m = mnew;
        }
        l += ((ls[0] + ls[1]) + (ls[2] + ls[3])) + ((ls[4] + ls[5]) + (ls[6] + ls[7]));
        if (row == 0 && x == 0 && tile < 400) OMNI_TRACE_AT(2402 + tile * 4);
        // P over this warpgroup's scores, which are in registers already.
        if constexpr (KW / 2 == 32) tmem_st32(scol, w);
        else tmem_st16(scol, w);
        tmem_wait_st();
        if (row == 0 && x == 0 && tile < 400) OMNI_TRACE_AT(2403 + tile * 4);
        tc_fence_before();
        mbar_arrive(&p_full[x][sb]);
        if (row == 0 && x < 2) OMNI_TRACE_AT(tile * 8 + 5 + 2 * x);
      }
      if (quit) break;
      // The unit's row sums of these keys for the epilogue, once it has read the previous unit's (a unit of one or
      // two tiles can be finished before that, and l_full must not complete two phases ahead of its waiter).
      if (nunit >= 1) wait(&l_free, (nunit - 1) & 1);
      ctl.lsum[x][row] = l;
      if (PACKED && x == 0) ctl.msum[row] = m;
      mbar_arrive(&l_full);
    }
  } else if (warp < W_EPI + 4) {
    // ------------------------------------------------------------------ epilogue (thread = query row)
    const int row = tid & 127;
    const uint32_t lane_off = (uint32_t)(32 * (warp & 3)) << 16;
    // One thread also loads the query tiles, two units ahead: unit n + 2's goes into unit n's slot once unit n's last
    // S has completed (q_empty, before its O is ready), so a unit's first S never waits for its queries.
    const bool q_loader = tid == W_EPI * 32;
    auto load_q = [&](int n, int i) {
      int b, h, qt;
      unit_of(p, i, b, h, qt);
      const int qslot = n % QS;
      mbar_arrive_expect_tx(&q_full[qslot], TILE);
#pragma unroll
      for (int x = 0; x < D / 64; ++x)
        tma_load_4d(smem + Q_OFF + qslot * TILE + x * BOX, &qmap, 64 * x, qt * BM, h, b, &q_full[qslot]);
      issued_q = n + 1;
    };
    if constexpr (!PACKED) {
      if (q_loader) {
        prefetch_tmap(&qmap);
        for (int n = 0, i; n < QS && (i = cta_unit(src, units, n)) >= 0; ++n) load_q(n, i);
      }
    }
    int nunit = 0;
    RedoList list;  // packed
    Unit u;
    // The warp's loads from TMEM and its votes want all lanes, so none leaves alone when a wait has run out. Packed: the lanes
    // take one answer, as the issuers. Dense: they go through the CTA's units all the same, whose waits return at once then
    // (a vote per wait cost 3% of a call here).
    for (; PACKED ? wget(nunit, u) : get(nunit, u); ++nunit) {
      if constexpr (!PACKED) {
        const int ahead = q_loader ? cta_unit(src, units, nunit + QS) : -1;
        if (ahead >= 0 && wait(&q_empty[nunit % QS], (nunit / QS) & 1)) load_q(nunit + QS, ahead);
      } else {
        __syncwarp();
        if (lane == 0) put(nunit);
      }
      if constexpr (PACKED) {
        if (!wwait(&o_ready, nunit & 1) || !wwait(&l_full, nunit & 1)) break;
      } else {
        wait(&o_ready, nunit & 1);
        wait(&l_full, nunit & 1);
      }
      if (row == 0) OMNI_TRACE_AT(1600 + nunit * 2);
      tc_fence_after();
      __syncwarp();
      float l = 0.f;
#pragma unroll
      for (int y = 0; y < NWG; ++y) l += ctl.lsum[y][row];
      const float m = PACKED ? ctl.msum[row] : 0.f;
      mbar_arrive(&l_free);
      float inv = l > 0.f ? 1.f / l : l;  // (l is 0, or NaN)
      const int q = u.qt * BM + row;
      __nv_bfloat16* dst;
      bool live;
      int pos = 0, head = 0;
      if constexpr (PACKED) {
        pos = row / src.group;
        head = u.h * src.group + row - pos * src.group;
        live = pos < u.npos;
        // A row that sees no key: zeros.
        if (u.lim0 + pos <= 0) inv = 0.f;
        else if (m == -INFINITY) inv = NAN;  // every key it sees scores -inf: no softmax
        dst = p.out + ((int64_t)(u.q0 + pos) * src.heads + head) * D;
      } else {
        dst = p.out + (int64_t)u.b * p.out_sb + (int64_t)q * p.out_sw + (int64_t)u.h * p.out_sh;
        live = q < p.width;
      }
      float odd = 0.f;  // packed: turns NaN if a result of the row is not finite
      if constexpr (PACKED) {
        if (u.part >= 0) {  // a part of a unit: fp32, a column of rows at a time
          if (u.part % u.b == 0 && row == 0)
            reinterpret_cast<PartMeta*>(src.meta + 8)[u.part / u.b] = {u.qt, u.h, u.q0, u.npos, u.k0, u.lim0, {0, 0}};
          float* part = src.parts + (int64_t)u.part * ((D + 2) * BM) + row;
          // (A row whose sum is NaN takes part whatever its maximum is, and makes the whole NaN.)
          part[D * BM] = u.lim0 + pos <= 0 ? -INFINITY : l == l ? m : INFINITY;
          part[(D + 1) * BM] = u.lim0 + pos > 0 ? l : 0.f;
#pragma unroll 1
          for (int c = 0; c < D / 32; ++c, part += 32 * BM) {
            float o[32];
            tmem_ld32(tbase + lane_off + COL_O + c * 32, o);
            if (c == D / 32 - 1) {
              tc_fence_before();
              mbar_arrive(&o_free);
            }
#pragma unroll
            for (int i = 0; i < 32; ++i) part[i * BM] = o[i];
          }
          continue;
        }
      }
      // O in two halves of 64 columns (two loads in flight per wait), released to the next unit's first P V once the
      // second half is in registers, before it is scaled and stored (measured: 183.0 us per config-4 call against
      // 186.5 us with four 32-column reads and the release after the last store).
#pragma unroll 1
      for (int c = 0; c < D / 64; ++c) {
        uint32_t r0[64];
        tmem_ld32_async(tbase + lane_off + COL_O + c * 64, r0);
        tmem_ld32_async(tbase + lane_off + COL_O + c * 64 + 32, r0 + 32);
        tmem_wait_ld();
        if (c == D / 64 - 1) {
          tc_fence_before();
          mbar_arrive(&o_free);
        }
        if (live) {
          if constexpr (PACKED) {
#pragma unroll
            for (int i = 0; i < 64; ++i) odd = fmaf(__uint_as_float(r0[i]), 0.f, odd);
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            uint32_t w4[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int k = 8 * i + 2 * j;
              w4[j] = pack_bf16x2(__uint_as_float(r0[k]) * inv, __uint_as_float(r0[k + 1]) * inv);
            }
            *reinterpret_cast<uint4*>(dst + c * 64 + i * 8) = make_uint4(w4[0], w4[1], w4[2], w4[3]);
          }
        }
      }
      if constexpr (PACKED) {
        const bool redo = live && odd != 0.f && l == l;  // (a row whose sum is NaN is NaN)
        const unsigned rows = __ballot_sync(0xffffffffu, redo);
        if (rows && list.add(u, rows, lane)) list.run<D>(src, row - lane, p.qscale, p.out);
      }
      if (row == 0) OMNI_TRACE_AT(1601 + nunit * 2);
    }
    if constexpr (PACKED) {
      if (!__any_sync(0xffffffffu, abort_flag != 0)) list.run<D>(src, row - lane, p.qscale, p.out);
    }
  }
  __syncthreads();
  if (abort_flag) {
    if (tid == 0) raise_status(p.status, kStatusTimeout);
    if ((warp == W_MMA || warp == W_MMA_PV) && elect_one()) {
      // Every MMA an issuer thread issued has completed once its commit arrives (two issuers: two arrivals).
      tc_commit(&drain);
      mbar_wait(&drain, 0);
    }
    if (tid == W_LOADK * 32) {
      // Let the latest load of every slot land (a slot is refilled only after its previous load was consumed).
      for (int i = issued_k > KS ? issued_k - KS : 0; i < issued_k; ++i) mbar_wait(&k_full[i % KS], (i / KS) & 1);
      for (int i = issued_v > VS ? issued_v - VS : 0; i < issued_v; ++i) mbar_wait(&v_full[i % VS], (i / VS) & 1);
      for (int i = issued_q > QS ? issued_q - QS : 0; i < issued_q; ++i) mbar_wait(&q_full[i % QS], (i / QS) & 1);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == W_EPI) {
    tc_fence_after();
    tmem_dealloc(tbase, TMEM_COLS);
  }
  OMNI_TRACE_CTA(1);
}

bool encode_map(CUtensorMap* map, const void* base, const cuuint64_t* dims, const cuuint64_t* strides,
                const cuuint32_t* box) {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      return (PFN_cuTensorMapEncodeTiled_v12000) nullptr;
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr);
  }();
  if (!fn) return false;
  cuuint32_t estr[4] = {1, 1, 1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(base), dims, strides, box, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

bool make_map(CUtensorMap* map, const void* base, int64_t b, int64_t h, int64_t w, int64_t sb, int64_t sh,
              int64_t sw) {
  cuuint64_t dims[4] = {128, (cuuint64_t)w, (cuuint64_t)h, (cuuint64_t)b};
  cuuint64_t strides[3] = {(cuuint64_t)sw * 2, (cuuint64_t)sh * 2, (cuuint64_t)sb * 2};
  cuuint32_t box[4] = {64, 128, 1, 1};
  return encode_map(map, base, dims, strides, box);
}

}  // namespace prefill

// (row, head) pairs per scheduling group: about 16, so that one group's units cover the grid once or twice and its
// K/V (under 13 MB at width 1500) stay in L2 while the grid works through them. OMNIASR_PREFILL_GROUP overrides.
int prefill_group(int bh_count) {
  static const int env = [] {
    const char* e = getenv("OMNIASR_PREFILL_GROUP");
    return e ? atoi(e) : 0;
  }();
  int g = env > 0 ? env : 16;
  return g < bh_count ? g : bh_count;
}

// Fixed cost of a unit in key tiles (measured: a unit's first tile takes about 1.6 tiles' time).
constexpr float kPrefillUnitCost = 0.6f;

// The list schedule of `units` units (unit_of's numbering) over `grid` CTAs, cached per shape.
const pfx::Sched* prefill_schedule(int batch, int heads, int qtiles, int group, int grid) {
  static const bool off = [] {  // OMNIASR_PREFILL_SCHED=0: round-robin (for comparisons)
    const char* e = getenv("OMNIASR_PREFILL_SCHED");
    return e && atoi(e) == 0;
  }();
  const int units = batch * heads * qtiles;
  if (off || units > pfx::kSchedUnits || grid > pfx::kSchedCtas) return nullptr;
  static std::mutex mu;
  static std::map<std::array<int, 5>, std::unique_ptr<pfx::Sched>> cache;
  const std::array<int, 5> key{batch, heads, qtiles, group, grid};
  std::lock_guard<std::mutex> lock(mu);
  auto it = cache.find(key);
  if (it != cache.end()) return it->second.get();
  auto s = std::make_unique<pfx::Sched>();
  std::vector<std::vector<uint16_t>> lists(grid);
  using Slot = std::pair<float, int>;  // (time the CTA is free, CTA)
  std::priority_queue<Slot, std::vector<Slot>, std::greater<Slot>> free_at;
  for (int c = 0; c < grid; ++c) free_at.push({0.f, c});
  const int bh_count = batch * heads;
  for (int u = 0; u < units; ++u) {
    const int per_group = group * qtiles;  // unit_of's numbering, on the host
    const int g0 = (u / per_group) * group;
    const int gsize = std::min(group, bh_count - g0);
    const int qt = qtiles - 1 - (u - g0 * qtiles) / gsize;
    const Slot c = free_at.top();
    free_at.pop();
    lists[c.second].push_back((uint16_t)u);
    free_at.push({c.first + (float)(qt + 1) + kPrefillUnitCost, c.second});
  }
  s->on = 1;
  int k = 0;
  for (int c = 0; c < grid; ++c) {
    s->start[c] = (uint16_t)k;
    for (uint16_t u : lists[c]) s->unit[k++] = u;
  }
  s->start[grid] = (uint16_t)k;
  return cache.emplace(key, std::move(s)).first->second.get();
}

const pfx::Sched& prefill_round_robin() {
  static const pfx::Sched r = [] {
    pfx::Sched x{};
    x.on = 0;
    return x;
  }();
  return r;
}

cudaError_t launch_prefill(const PrefillArgs& a, cudaStream_t stream) {
  using namespace prefill;
  constexpr int SMEM_BYTES = Cfg<128>::SMEM_BYTES;
  CUtensorMap qm, km, vm;
  if (!make_map(&qm, a.q, a.batch, a.heads, a.width, a.q_sb, a.q_sh, a.q_sw) ||
      !make_map(&km, a.k, a.batch, a.heads, a.width, a.k_sb, a.k_sh, a.k_sw) ||
      !make_map(&vm, a.v, a.batch, a.heads, a.width, a.v_sb, a.v_sh, a.v_sw))
    return cudaErrorInvalidValue;
  static PerDevice configured;
  if (const cudaError_t e = allow_smem(prefill_kernel<Sched, 128>, SMEM_BYTES, configured)) return e;
  Params p;
  p.batch = a.batch;
  p.heads = a.heads;
  p.width = a.width;
  p.qtiles = (a.width + BM - 1) / BM;
  p.qscale = a.scale * kLog2e;
  p.group = omni::prefill_group(a.batch * a.heads);
  p.q = reinterpret_cast<const __nv_bfloat16*>(a.q);
  p.q_sb = a.q_sb;
  p.q_sh = a.q_sh;
  p.q_sw = a.q_sw;
  p.out = reinterpret_cast<__nv_bfloat16*>(a.out);
  p.out_sb = a.o_sb;
  p.out_sw = a.o_sw;
  p.out_sh = a.o_sh;
  p.status = a.status;
  const int units = a.batch * a.heads * p.qtiles;
  int grid = device_sm_count();
  if (grid > units) grid = units;
  if (grid <= 0) return cudaSuccess;
  const Sched* sched = prefill_schedule(p.batch, p.heads, p.qtiles, p.group, grid);
  return launch_dependent(prefill_kernel<Sched, 128>, dim3(grid), dim3(THREADS), (size_t)SMEM_BYTES, stream, qm, km, vm, p,
                          sched ? *sched : prefill_round_robin());
}

// Adds up the parts of a cut unit (block x: unit, y: 32 of its head dims; thread: tile row): o = sum 2^(m_s - m) O_s / sum
// 2^(m_s - m) l_s, in the order of the keys. Rows whose result is not finite are redone from the formula, in the block's dims
// (the other blocks write theirs).
template <int D>
__global__ void __launch_bounds__(128) packed_join_kernel(const __grid_constant__ pfx::PackedSrc src, float qscale,
                                                          __nv_bfloat16* out) {
  using namespace pfx;
  grid_launch_dependents();
  grid_dependency_wait();
  const int units = src.meta[0], cut = src.meta[1];
  if (cut <= 1 || (int)blockIdx.x >= units) return;
  const PartMeta u = reinterpret_cast<const PartMeta*>(src.meta + 8)[blockIdx.x];
  const int row = threadIdx.x, d0 = blockIdx.y * 32;
  const int pos = row / src.group, head = u.h * src.group + row - pos * src.group;
  const bool live = pos < u.npos;
  const float* part = src.parts + (int64_t)blockIdx.x * cut * ((D + 2) * 128) + row;
  float w[kMostParts], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int s = 0; s < kMostParts; ++s) {
    w[s] = s < u.n ? part[(int64_t)s * ((D + 2) * 128) + D * 128] : -INFINITY;
    m = fmaxf(m, w[s]);
  }
#pragma unroll
  for (int s = 0; s < kMostParts; ++s) {
    w[s] = w[s] > -INFINITY ? ex2(w[s] - m) : 0.f;
    if (w[s] != 0.f) l = fmaf(w[s], part[(int64_t)s * ((D + 2) * 128) + (D + 1) * 128], l);
  }
  float o[32];
#pragma unroll
  for (int i = 0; i < 32; ++i) o[i] = 0.f;
#pragma unroll 1
  for (int s = 0; s < u.n; ++s) {
    float ws = 0.f;
#pragma unroll
    for (int k = 0; k < kMostParts; ++k) ws = k == s ? w[k] : ws;
    float v[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = part[(int64_t)s * ((D + 2) * 128) + (d0 + i) * 128];
#pragma unroll
    for (int i = 0; i < 32; ++i) o[i] = ws != 0.f ? fmaf(ws, v[i], o[i]) : o[i];
  }
  const float inv = l != 0.f ? 1.f / l : (u.lim0 + pos > 0 ? NAN : 0.f);  // (keys that all score -inf: no softmax)
  const int64_t at = ((int64_t)(u.q0 + pos) * src.heads + head) * D;
  float odd = 0.f;
  if (live) {
    uint4* dst = reinterpret_cast<uint4*>(out + at + d0);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t p4[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float a = o[8 * i + 2 * j] * inv, b = o[8 * i + 2 * j + 1] * inv;
        odd = fmaf(a, 0.f, fmaf(b, 0.f, odd));
        p4[j] = pack_bf16x2(a, b);
      }
      dst[i] = make_uint4(p4[0], p4[1], p4[2], p4[3]);
    }
  }
  const bool redo = live && odd != 0.f && l == l;
  __syncwarp();  // the rows' first results are written before they are written again
  const unsigned rows = __ballot_sync(0xffffffffu, redo);
  if (rows)
    redo_rows<D, 32>(src, rows, row & ~31, u.q0, u.k0, u.lim0, u.h, max(1, (u.lim0 + u.npos - 1 + 127) / 128), qscale, out, d0);
}

cudaError_t launch_packed_join(const PackedArgs& a, const pfx::PackedSrc& src, cudaStream_t stream) {
  if (!src.meta) return cudaSuccess;
  const dim3 grid((unsigned)packed_cut_units(), (unsigned)(a.dim / 32));
  const float qscale = a.scale * kLog2e;
  __nv_bfloat16* out = reinterpret_cast<__nv_bfloat16*>(a.out);
  switch (a.dim) {
    case 64: return launch_dependent(packed_join_kernel<64>, grid, dim3(128), 0, stream, src, qscale, out);
    case 128: return launch_dependent(packed_join_kernel<128>, grid, dim3(128), 0, stream, src, qscale, out);
    case 256: return launch_dependent(packed_join_kernel<256>, grid, dim3(128), 0, stream, src, qscale, out);
    default: return launch_dependent(packed_join_kernel<512>, grid, dim3(128), 0, stream, src, qscale, out);
  }
}

// Units are cut while there are at most this many.
int packed_cut_units() { return device_sm_count() / 2; }

// Whether a call may have that few units: it has one per tile of its queries at least.
static bool may_cut(int64_t q_tokens, int heads, int kv_heads) {
  const int positions = 128 / (heads / kv_heads);
  return (q_tokens + positions - 1) / positions * kv_heads <= packed_cut_units();
}

size_t packed_workspace(int dtype, int64_t q_tokens, int heads, int kv_heads, int dim) {
  if (const size_t parts = packed_parts_bytes(dtype, q_tokens, heads, kv_heads, dim)) return kCounterBytes + parts;
  if (dtype != kBF16 || dim < 64 || heads / kv_heads > 128 || !may_cut(q_tokens, heads, kv_heads)) return 256;
  return kCounterBytes + 32 + sizeof(pfx::PartMeta) * packed_cut_units() + 256 +
         sizeof(float) * 128 * (size_t)(dim + 2) * device_sm_count();
}

bool packed_maps(const PackedArgs& a, int positions, int v_rows, CUtensorMap* q, CUtensorMap* k, CUtensorMap* v) {
  using prefill::encode_map;
  const int group = a.heads / a.kv_heads;
  // An extent of one has a stride that nothing reads; PyTorch leaves any number there.
  auto st = [](int64_t extent, int64_t stride) { return (cuuint64_t)(extent > 1 ? stride * 2 : 16); };
  const cuuint64_t qd[4] = {(cuuint64_t)a.dim, (cuuint64_t)group, (cuuint64_t)a.kv_heads, (cuuint64_t)a.q_tokens};
  const cuuint64_t qs[3] = {st(group, a.q_sh), st(a.kv_heads, group * a.q_sh), st(a.q_tokens, a.q_st)};
  const cuuint32_t qb[4] = {64, (cuuint32_t)group, 1, (cuuint32_t)positions};
  const cuuint64_t kd[4] = {(cuuint64_t)a.dim, (cuuint64_t)a.k_tokens, (cuuint64_t)a.kv_heads, 1};
  const cuuint64_t ks[3] = {st(a.k_tokens, a.k_st), st(a.kv_heads, a.k_sh), 16};
  const cuuint64_t vs[3] = {st(a.k_tokens, a.v_st), st(a.kv_heads, a.v_sh), 16};
  const cuuint32_t kb[4] = {64, 128, 1, 1}, vb[4] = {64, (cuuint32_t)v_rows, 1, 1};
  for (int i = 0; i < 3; ++i)
    if (!qs[i] || !ks[i] || !vs[i]) return false;
  return encode_map(q, a.q, qd, qs, qb) && encode_map(k, a.k, kd, ks, kb) && encode_map(v, a.v, kd, vs, vb);
}

pfx::PackedSrc packed_source(const PackedArgs& a, int positions) {
  pfx::PackedSrc s;
  s.q_offsets = a.q_offsets;
  s.k_offsets = a.k_offsets;
  s.q_tokens = a.q_tokens;
  s.k_tokens = a.k_tokens;
  s.seqs = a.seqs;
  s.heads = a.heads;
  s.kv_heads = a.kv_heads;
  s.group = a.heads / a.kv_heads;
  s.pos = positions;
  s.pos_magic = 0xffffffffu / (unsigned)positions + 1;
  s.counters = a.counters;
  s.meta = nullptr;
  s.parts = nullptr;
  if (may_cut(a.q_tokens, a.heads, a.kv_heads)) {
    char* ws = reinterpret_cast<char*>(a.counters) + kCounterBytes;
    s.meta = reinterpret_cast<int*>(ws);
    s.parts = reinterpret_cast<float*>(ws + (32 + sizeof(pfx::PartMeta) * packed_cut_units() + 255) / 256 * 256);
  }
  s.q = reinterpret_cast<const __nv_bfloat16*>(a.q);
  s.k = reinterpret_cast<const __nv_bfloat16*>(a.k);
  s.v = reinterpret_cast<const __nv_bfloat16*>(a.v);
  s.q_st = a.q_st, s.q_sh = a.q_sh, s.k_st = a.k_st, s.k_sh = a.k_sh, s.v_st = a.v_st, s.v_sh = a.v_sh;
  return s;
}

int packed_grid(const PackedArgs& a, int positions) {
  // Units that are cut may give every CTA a part; others are at most this many.
  const int64_t units = may_cut(a.q_tokens, a.heads, a.kv_heads) ? device_sm_count()
                                                                 : (a.q_tokens / positions + a.seqs) * a.kv_heads;
  return (int)std::min<int64_t>(device_sm_count(), units);
}

template <int D>
cudaError_t launch_packed_d(const PackedArgs& a, cudaStream_t stream) {
  using namespace prefill;
  constexpr int SMEM_BYTES = Cfg<D>::SMEM_BYTES;
  const int positions = BM / (a.heads / a.kv_heads);
  CUtensorMap qm, km, vm;
  if (!packed_maps(a, positions, BN, &qm, &km, &vm)) return cudaErrorNotSupported;
  static PerDevice configured;
  if (const cudaError_t e = allow_smem(prefill_kernel<PackedSrc, D>, SMEM_BYTES, configured)) return e;
  Params p{};
  p.qscale = a.scale * kLog2e;
  p.out = reinterpret_cast<__nv_bfloat16*>(a.out);
  p.status = a.status;
  const pfx::PackedSrc src = packed_source(a, positions);
  const cudaError_t e = launch_dependent(prefill_kernel<PackedSrc, D>, dim3(packed_grid(a, positions)), dim3(THREADS),
                                         (size_t)SMEM_BYTES, stream, qm, km, vm, p, src);
  return e != cudaSuccess ? e : launch_packed_join(a, src, stream);
}

cudaError_t launch_packed_tc(const PackedArgs& a, cudaStream_t stream) {
  return a.dim == 64 ? launch_packed_d<64>(a, stream) : launch_packed_d<128>(a, stream);
}

}  // namespace omni
