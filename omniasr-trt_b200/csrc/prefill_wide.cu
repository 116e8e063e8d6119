// Causal prefill attention on the 5th-generation tensor cores (tcgen05 + TMEM), bf16: dense rows of head_dim 512 -- the shipped
// omniASR-LLM decoder's 8 heads x 512 (omniasr_trt/modeling.py:30-35) -- and packed sequences with grouped heads of head_dim
// 256 (one pass) and 512 (two; PackedSrc, prefill_common.cuh; packed.cu has the formula).
//
// out[b, w, h] = softmax(q[b, h, w] . k[b, h, :w+1]^T * scale) . v[b, h, :w+1]   for w < W
// (F.scaled_dot_product_attention(q, k, v, is_causal=True) of the reference's prefill, decode.py:171).
//
// The head_dim-128 kernel (prefill.cu) keeps a 128 x 128 fp32 accumulator per query tile in TMEM; at head_dim 512
// the accumulator alone (128 x 512 fp32) fills all of TMEM, and one query tile is 128 KB of shared memory. So a unit
// (row b, head h, 128-query tile qt) runs as two passes over its key tiles, pass p accumulating head dims
// 256p .. 256p + 255 of O: both passes form the same scores S = Q K^T over all 512 dims (four 128-dim chunks
// accumulated in TMEM) and the same probabilities; the second pass recomputes them (one and a half times the
// minimum MMA work) instead of storing them. The work is MMA-bound at this head_dim: a tile pass is 32 SS MMAs
// (128 x 128 x 16) for S and 32 TS MMAs (128 x 64 x 16) for P V, against one softmax of a 128 x 128 tile.
//
// Shared memory (224 KB): the unit's query tile as four 128-dim chunks (loaded once for both passes; chunk c is
// refilled with the next unit's as soon as the last S MMA that reads it has completed), a 2-slot ring of 128-dim K
// chunks, a 2-slot ring of 64-dim V sub-chunks (128 keys each; 128-byte swizzle throughout).
// TMEM (512 columns): S double-buffered at [0, 128) and [128, 256), O of the pass's 256 dims at [256, 512); P (bf16
// pairs) over S, read by the A-from-TMEM MMA.
// Packed sequences use the same ring bytes in finer pieces: K in 64-dim boxes, so that more loads are in flight while one is
// used, and V in slots of 32 keys x 256 dims, so that P V is 8 MMAs of N = 256 instead of 32 of N = 64. Issuing from converged
// warps (prefill.cu): 8 prompts of 1500, 16 heads of 256 on 4, 177 -> 157 us (939 TFLOP/s), of 512 454 -> 421 (702).
// Roles (512 threads), as in prefill.cu: warp 12 K chunk loads, warp 14 V sub-chunk loads, warp 13 S MMAs, warp 15
// P V MMAs, warps 0-3 / 4-7 softmax warpgroups (thread = query row, warpgroup x the keys 64x .. 64x + 63 of every
// tile, one running max per row shared through a barrier per tile), warps 8-11 the epilogue (and the query loads,
// by its first thread).

#include <cudaTypedefs.h>
#include <math.h>

#include <type_traits>

#include "attention.cuh"
#include "prefill.cuh"
#include "paged.cuh"
#include "prefill_common.cuh"

namespace omni {
namespace prefillw {

using namespace pfx;

constexpr int DH = 256;            // head dims of O per pass
constexpr int NSUB = DH / 64;      // 64-dim V sub-chunks per pass
constexpr int BM = 128;            // queries per tile
constexpr int BN = 128;            // keys per tile
constexpr int CHUNK = BN * 128 * 2;  // 128 rows x 128 dims
constexpr int BOX = BN * 64 * 2;     // 128 rows x 64 dims: one TMA box
// What depends on the head dim: 512, or 256 (packed sequences; O of all 256 dims is one pass, and the query tile leaves room
// for deeper rings).
template <int D>
struct Cfg {
  static constexpr int DC = D / 128;   // 128-dim chunks of Q and K
  static constexpr int PASSES = D / DH;
  static constexpr int KS = D == 256 ? 3 : 2, VS = D == 256 ? 4 : 2;
  static constexpr int Q_OFF = 0;
  static constexpr int K_OFF = Q_OFF + DC * CHUNK;
  static constexpr int V_OFF = K_OFF + KS * CHUNK;
  static constexpr int SMEM_BYTES = V_OFF + VS * BOX;
};
constexpr int NSB = 2;
constexpr int NWG = 2;
constexpr int KW = BN / NWG;  // keys per softmax warpgroup
constexpr int DW = DH / NWG;  // head dims of O each softmax warpgroup rescales
constexpr int W_EPI = 4 * NWG, W_LOADK = W_EPI + 4, W_MMA = W_LOADK + 1, W_LOADV = W_LOADK + 2, W_MMA_PV = W_LOADK + 3;
constexpr int THREADS = 32 * (W_MMA_PV + 1);
constexpr int SM_THREADS = 128 * NWG;
constexpr uint32_t TMEM_COLS = 512;
constexpr uint32_t COL_S = 0, COL_O = NSB * 128;
constexpr uint32_t IDESC_S = idesc_bf16(BM, BN, 0, 0);
constexpr uint32_t IDESC_O = idesc_bf16(BM, 64, 0, 1);
constexpr uint32_t IDESC_O256 = idesc_bf16(BM, DH, 0, 1);
constexpr int VK = 32;  // packed: keys of a V slot (all 256 dims of the pass)
constexpr float kRescale = 8.f;
constexpr int kPolyEvery = 4;  // probabilities of one pair in this many by ex2_fma

struct Params {
  int batch, heads, width, qtiles;
  int group;
  float qscale;  // scale * log2(e)
  __nv_bfloat16* out;
  int64_t out_sb, out_sw, out_sh;
  int* status;
};

template <int D>
struct alignas(1024) Ctl {
  static constexpr int DC = Cfg<D>::DC, KS = Cfg<D>::KS, VS = Cfg<D>::VS;
  uint64_t k_full[2 * KS], k_empty[2 * KS], v_full[VS], v_empty[VS], q_full[DC], q_empty[DC];
  uint64_t s_full[NSB], pv_done[NSB], p_full[NWG][NSB];
  uint64_t o_ready, o_free, l_full, l_free, drain;
  float tmax[NWG][BM];
  float msum[BM];  // [row]: the maximum of a unit's part
  float lsum[NWG][BM];
  uint32_t tmem_base;
  int abort_flag, issued_k, issued_v, issued_q;
  uint64_t u_full[kUnitRing], u_empty[kUnitRing];  // packed: the units claimed, for all roles
  Unit unit[kUnitRing];
};
static_assert(sizeof(Ctl<512>) + Cfg<512>::SMEM_BYTES <= 232448 && sizeof(Ctl<256>) + Cfg<256>::SMEM_BYTES <= 232448,
              "shared memory per block");
static_assert(NSB * 128 + DH <= TMEM_COLS, "S buffers and O in TMEM");

// Src: Sched (dense rows) or PackedSrc (packed sequences with grouped heads).
template <typename Src, int D>
__global__ void __launch_bounds__(THREADS, 1)
    prefill_wide_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                        const __grid_constant__ CUtensorMap vmap, const Params p, const __grid_constant__ Src src) {
  constexpr bool PACKED = std::is_same_v<Src, PackedSrc>;
  using C = Cfg<D>;
  constexpr int DC = C::DC, PASSES = C::PASSES, KS = C::KS, VS = C::VS, Q_OFF = C::Q_OFF, K_OFF = C::K_OFF, V_OFF = C::V_OFF;
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
  if (smem_addr(smem) & 1023u) {
    if (tid == 0) raise_status(p.status, kStatusLayout);
    return;
  }
  if (tid == 0) {
    for (int s = 0; s < 2 * KS; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&k_empty[s], 1);
    }
    for (int s = 0; s < VS; ++s) {
      mbar_init(&v_full[s], 1);
      mbar_init(&v_empty[s], 1);
    }
    for (int c = 0; c < DC; ++c) {
      mbar_init(&q_full[c], 1);
      mbar_init(&q_empty[c], 1);
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
  const uint32_t tbase = ctl.tmem_base;
  auto wait = [&](uint64_t* bar, uint32_t parity) -> bool {
    if (mbar_wait_or(bar, parity, &abort_flag)) return true;
    abort_flag = 1;
    return false;
  };
  auto decode = [&](int u, int& b, int& h, int& qt) { unit_of(p.batch, p.heads, p.qtiles, p.group, u, b, h, qt); };

  // The CTA's n-th unit; false past its last (or, packed, after an abort). put: this role (or warp) is done with it.
  auto get = [&](int n, Unit& u) -> bool {
    if constexpr (PACKED) {
      if (!wait(&ctl.u_full[n % kUnitRing], (n / kUnitRing) & 1)) return false;
      u = ctl.unit[n % kUnitRing];
      return u.kt > 0;
    } else {
      const int i = cta_unit(src, units, n);
      if (i < 0) return false;
      decode(i, u.b, u.h, u.qt);
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
      int kc = 0;
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
          for (int pass = 0; pass < PASSES && ok; ++pass)
            for (int kt = 0; kt < u.kt && ok; ++kt) {
              // The next unit is claimed with the last tile, so that no CTA holds units it starts late.
              if (pass == PASSES - 1 && kt == u.kt - 1) claim = atomicAdd(src.counters, 1u);
              for (int c = 0; c < DC && ok; ++c, ++kc) {
                if (pass == 0 && kt == 0) {
                  ok = n < 1 || wait(&q_empty[c], (n - 1) & 1);
                  if (!ok) break;
                  mbar_arrive_expect_tx(&q_full[c], (uint32_t)(src.group * src.pos) * 256u);
                  unsigned char* dst = smem + Q_OFF + c * CHUNK;
                  tma_load_4d(dst, &qmap, c * 128, 0, u.h, u.q0, &q_full[c]);
                  tma_load_4d(dst + BOX, &qmap, c * 128 + 64, 0, u.h, u.q0, &q_full[c]);
                  issued_q = n * DC + c + 1;
                }
                for (int x = 0; x < 2 && ok; ++x) {
                  const int kb = 2 * kc + x, slot = kb % (2 * KS), use = kb / (2 * KS);
                  ok = use < 1 || wait(&k_empty[slot], (use - 1) & 1);
                  if (!ok) break;
                  mbar_arrive_expect_tx(&k_full[slot], BOX);
                  tma_load_4d(smem + K_OFF + slot * BOX, &kmap, c * 128 + 64 * x, u.k0 + kt * BN, u.h, 0, &k_full[slot]);
                  issued_k = kb + 1;
                }
              }
            }
        }
        ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
        if (!ok || u.kt == 0 || __any_sync(0xffffffffu, abort_flag != 0)) break;
        kc = __shfl_sync(0xffffffffu, kc, 0);
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
  } else if (warp == W_LOADK) {
    // ------------------------------------------------------------------ K: chunk c of key tile kt, both passes
    if (lane == 0) {
      prefetch_tmap(&kmap);
      int kc = 0;
      Unit u;
      for (int n = 0; get(n, u) && !abort_flag; ++n) {
        for (int pass = 0; pass < PASSES && !abort_flag; ++pass)
          for (int kt = 0; kt < u.kt && !abort_flag; ++kt)
            for (int c = 0; c < DC && !abort_flag; ++c, ++kc) {
              const int slot = kc % KS, use = kc / KS;
              if (use >= 1 && !wait(&k_empty[slot], (use - 1) & 1)) break;
              mbar_arrive_expect_tx(&k_full[slot], CHUNK);
              unsigned char* dst = smem + K_OFF + slot * CHUNK;
              tma_load_4d(dst, &kmap, c * 128, kt * BN, u.h, u.b, &k_full[slot]);
              tma_load_4d(dst + BOX, &kmap, c * 128 + 64, kt * BN, u.h, u.b, &k_full[slot]);
              issued_k = kc + 1;
            }
      }
    }
    __syncwarp();
  } else if (warp == W_LOADV) {
    // ------------------------------------------------------------------ V: the pass's 64-dim sub-chunks of tile kt
    if (lane == 0) {
      prefetch_tmap(&vmap);
      int vc = 0;
      Unit u;
      for (int n = 0; get(n, u) && !abort_flag; ++n) {
        for (int pass = 0; pass < PASSES && !abort_flag; ++pass)
          for (int kt = 0; kt < u.kt && !abort_flag; ++kt)
            for (int sc = 0; sc < NSUB && !abort_flag; ++sc, ++vc) {
              const int slot = vc % VS, use = vc / VS;
              if (use >= 1 && !wait(&v_empty[slot], (use - 1) & 1)) break;
              mbar_arrive_expect_tx(&v_full[slot], BOX);
              unsigned char* dst = smem + V_OFF + slot * BOX;
              if constexpr (PACKED) {  // keys VK sc .. of all the pass's dims, in 64-dim boxes
#pragma unroll
                for (int x = 0; x < DH / 64; ++x)
                  tma_load_4d(dst + x * (VK * 128), &vmap, pass * DH + x * 64, u.k0 + kt * BN + VK * sc, u.h, 0, &v_full[slot]);
              } else {
                tma_load_4d(dst, &vmap, pass * DH + sc * 64, kt * BN, u.h, u.b, &v_full[slot]);
              }
              issued_v = vc + 1;
            }
        put(n);
      }
    }
    __syncwarp();
  } else if (warp == W_MMA) {
    // ------------------------------------------------------------------ S[t % NSB] = sum over chunks Q_c K_c(t)^T
    {
      const bool leader = elect_one();  // the issuing warps run converged (prefill.cu)
      const uint64_t kdesc0 = smem_desc(smem_addr(smem + K_OFF), 16, 1024, kLayoutSw128);
      const uint64_t qdesc0 = smem_desc(smem_addr(smem + Q_OFF), 16, 1024, kLayoutSw128);
      int tile = 0, kc = 0;
      bool ok = true;
      Unit u;
      for (int n = 0; wget(n, u) && ok; ++n) {
        for (int pass = 0; pass < PASSES && ok; ++pass) {
          for (int kt = 0; kt < u.kt && ok; ++kt, ++tile) {
            const int sb = tile % NSB;
            if (tile >= NSB && !wwait(&pv_done[sb], ((tile - NSB) / NSB) & 1)) {
              ok = false;
              break;
            }
            const uint32_t dcol = tbase + COL_S + sb * 128;
            for (int c = 0; c < DC; ++c, ++kc) {
              if (pass == 0 && kt == 0 && !wwait(&q_full[c], n & 1)) {
                ok = false;
                break;
              }
              if constexpr (PACKED) {
                for (int x = 0; x < 2; ++x) {
                  const int kb = 2 * kc + x, slot = kb % (2 * KS);
                  if (!wwait(&k_full[slot], (kb / (2 * KS)) & 1)) {
                    ok = false;
                    break;
                  }
                  tc_fence_after();
                  const uint64_t qd = qdesc0 + (uint64_t)((2 * c + x) * (BOX >> 4));
                  const uint64_t kd = kdesc0 + (uint64_t)(slot * (BOX >> 4));
                  if (leader) {
#pragma unroll
                    for (int kk = 0; kk < 4; ++kk)
                      mma_bf16_ss(dcol, qd + kk * 2, kd + kk * 2, IDESC_S, (c > 0 || x > 0 || kk > 0) ? 1u : 0u);
                    tc_commit(&k_empty[slot]);
                  }
                }
                if (!ok) break;
              } else {
                const int slot = kc % KS;
                if (!wwait(&k_full[slot], (kc / KS) & 1)) {
                  ok = false;
                  break;
                }
                tc_fence_after();
                const uint64_t qd = qdesc0 + (uint64_t)(c * (CHUNK >> 4));
                const uint64_t kd = kdesc0 + (uint64_t)(slot * (CHUNK >> 4));
                if (leader) {
#pragma unroll
                  for (int kk = 0; kk < 8; ++kk) {
                    const uint64_t off = (uint64_t)((((kk >> 2) * BOX + (kk & 3) * 32) >> 4));
                    mma_bf16_ss(dcol, qd + off, kd + off, IDESC_S, (c > 0 || kk > 0) ? 1u : 0u);
                  }
                  tc_commit(&k_empty[slot]);
                }
              }
              if (leader && pass == PASSES - 1 && kt == u.kt - 1) tc_commit(&q_empty[c]);  // the unit's last read of query chunk c
            }
            if (!ok) break;
            if (leader) tc_commit(&s_full[sb]);
            __syncwarp();
          }
        }
        if (leader) put(n);
      }
      if (!ok) abort_flag = 1;
    }
  } else if (warp == W_MMA_PV) {
    // ------------------------------------------------------------------ O[:, 64 sc ..] += P(t) V(t)[:, sc]
    {
      const bool leader = elect_one();
      const uint64_t vdesc0 = smem_desc(smem_addr(smem + V_OFF), BOX, 1024, kLayoutSw128);
      const uint64_t vdesc32 = smem_desc(smem_addr(smem + V_OFF), VK * 128, 1024, kLayoutSw128);
      int tile = 0, vc = 0, item = 0;
      bool ok = true;
      Unit u;
      for (int n = 0; wget(n, u) && ok; ++n) {
        for (int pass = 0; pass < PASSES && ok; ++pass, ++item) {
          for (int kt = 0; kt < u.kt && ok; ++kt, ++tile) {
            const int pb = tile % NSB, pu = tile / NSB;
            if (kt == 0 && item >= 1 && !wwait(&o_free, (item - 1) & 1)) {
              ok = false;
              break;
            }
            const uint32_t pcol = tbase + COL_S + pb * 128;
            if constexpr (PACKED) {
              for (int sc = 0; sc < BN / VK; ++sc, ++vc) {
                const int slot = vc % VS, x = sc * VK / KW;
                if (sc * VK % KW == 0) ok = wwait(&p_full[x][pb], pu & 1);
                ok = ok && wwait(&v_full[slot], (vc / VS) & 1);
                if (!ok) break;
                tc_fence_after();
                const uint64_t vd = vdesc32 + (uint64_t)(slot * (BOX >> 4));
                if (leader) {
#pragma unroll
                  for (int kk = 0; kk < VK / 16; ++kk)
                    mma_bf16_ts(tbase + COL_O, pcol + x * KW + (sc * VK % KW / 16 + kk) * 8, vd + (uint64_t)(kk * 128), IDESC_O256,
                                (kt == 0 && sc == 0 && kk == 0) ? 0u : 1u);
                  tc_commit(&v_empty[slot]);
                }
              }
              if (!ok) break;
              if (leader) tc_commit(&pv_done[pb]);
              __syncwarp();
            } else {
              for (int x = 0; x < NWG && ok; ++x) ok = wwait(&p_full[x][pb], pu & 1);
              if (!ok) break;
              tc_fence_after();
              for (int sc = 0; sc < NSUB; ++sc, ++vc) {
                const int slot = vc % VS;
                if (!wwait(&v_full[slot], (vc / VS) & 1)) {
                  ok = false;
                  break;
                }
                tc_fence_after();
                const uint64_t vd = vdesc0 + (uint64_t)(slot * (BOX >> 4));
                if (leader) {
#pragma unroll
                  for (int x = 0; x < NWG; ++x)
#pragma unroll
                    for (int kk = 0; kk < KW / 16; ++kk)
                      mma_bf16_ts(tbase + COL_O + sc * 64, pcol + x * KW + kk * 8,
                                  vd + (uint64_t)((KW / 16 * x + kk) * 128), IDESC_O,
                                  (kt == 0 && x == 0 && kk == 0) ? 0u : 1u);
                  tc_commit(&v_empty[slot]);
                }
              }
              if (!ok) break;
              if (leader) tc_commit(&pv_done[pb]);
              __syncwarp();
            }
          }
          if (ok && leader) tc_commit(&o_ready);
        }
        if (leader) put(n);
      }
      if (!ok) abort_flag = 1;
    }
    __syncwarp();
  } else if (warp < W_EPI) {
    // ------------------------------------------------------------------ softmax, keys KW x .. of every tile
    const int x = warp >> 2;
    const int row = tid & 127;
    const uint32_t lane_off = (uint32_t)(32 * (warp & 3)) << 16;
    const uint32_t col_o = tbase + lane_off + COL_O + x * DW;  // this warpgroup's head dims of O (rescale)
    int tile = 0, item = 0;
    bool quit = false;
    int row_pos = 0;  // packed: the row's position within the tile
    if constexpr (PACKED) row_pos = row / src.group;
    for (int n = 0; !quit; ++n) {
      Unit u;
      const bool more = get(n, u);
      if constexpr (PACKED) {  // the claim's wait may have given up in some threads: decided by all of them
        if (sync_or(1, SM_THREADS, abort_flag != 0)) break;
      }
      if (!more) break;
      __syncwarp();
      if (PACKED && lane == 0) put(n);
      for (int pass = 0; pass < PASSES && !quit; ++pass, ++item) {
        float m = -INFINITY, l = 0.f;
        for (int kt = 0; kt < u.kt; ++kt, ++tile) {
          const int sb = tile % NSB;
          wait(&s_full[sb], (tile / NSB) & 1);
          tc_fence_after();
          __syncwarp();
          const uint32_t scol = tbase + lane_off + COL_S + sb * 128 + x * KW;
          uint32_t raw[KW];
#pragma unroll
          for (int c = 0; c < KW / 32; ++c) tmem_ld32_async(scol + 32 * c, raw + 32 * c);
          tmem_wait_ld();
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
          float part[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) part[j] = v[j];
#pragma unroll
          for (int i = 8; i < KW; i += 16)
#pragma unroll
            for (int j = 0; j < 8; ++j) part[j] = max3(part[j], v[i + j], v[i + 8 + j]);
          const float tmax = max3(max3(part[0], part[1], part[2]), max3(part[3], part[4], part[5]),
                                  max2(part[6], part[7])) * p.qscale;
          const bool saw_abort = abort_flag != 0;
          float mnew = m;
          bool slow = false;
          if (sync_or(1, SM_THREADS, !(tmax <= m + kRescale) || saw_abort)) {
            if (sync_or(1, SM_THREADS, saw_abort)) {
              quit = true;
              break;
            }
            ctl.tmax[x][row] = tmax;
            if (!row_finite(tmax)) l = NAN;
            named_sync(2, SM_THREADS);
            float t2 = ctl.tmax[0][row];
#pragma unroll
            for (int y = 1; y < NWG; ++y) t2 = fmaxf(t2, ctl.tmax[y][row]);
            if (t2 > m + kRescale) mnew = t2;
            slow = true;
          }
          const float mref = PACKED && mnew == -INFINITY ? 0.f : mnew;  // a packed row may have seen no key
          uint32_t w[KW / 2];
          uint64_t ls2[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) ls2[j] = 0ull;
          const uint64_t sc2 = f2_pack(p.qscale, p.qscale), nm2 = f2_pack(-mref, -mref);
#pragma unroll
          for (int i = 0; i < KW / 2; ++i) {
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
              wait(&pv_done[(tile - 1) % NSB], ((tile - 1) / NSB) & 1);  // O holds every earlier tile of the pass
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
          tmem_st32(scol, w);
          tmem_wait_st();
          tc_fence_before();
          mbar_arrive(&p_full[x][sb]);
        }
        if (quit) break;
        if (item >= 1) wait(&l_free, (item - 1) & 1);
        ctl.lsum[x][row] = l;
        if (PACKED && x == 0) ctl.msum[row] = m;
        mbar_arrive(&l_full);
      }
    }
  } else if (warp < W_EPI + 4) {
    // ------------------------------------------------------------------ epilogue (thread = query row)
    const int row = tid & 127;
    const uint32_t lane_off = (uint32_t)(32 * (warp & 3)) << 16;
    const bool q_loader = tid == W_EPI * 32;
    auto load_q = [&](int n, int i) {  // unit i (the CTA's n-th) into the query chunks, each once it is free
      int b, h, qt;
      decode(i, b, h, qt);
      for (int c = 0; c < DC; ++c) {
        if (n >= 1 && !wait(&q_empty[c], (n - 1) & 1)) return;
        mbar_arrive_expect_tx(&q_full[c], CHUNK);
        unsigned char* dst = smem + Q_OFF + c * CHUNK;
        tma_load_4d(dst, &qmap, c * 128, qt * BM, h, b, &q_full[c]);
        tma_load_4d(dst + BOX, &qmap, c * 128 + 64, qt * BM, h, b, &q_full[c]);
        issued_q = n * DC + c + 1;  // chunk loads issued
      }
    };
    if constexpr (!PACKED) {
      if (q_loader) {
        prefetch_tmap(&qmap);
        const int u0 = cta_unit(src, units, 0);
        if (u0 >= 0) load_q(0, u0);
      }
    }
    int item = 0;
    RedoList list;  // packed
    Unit u;
    bool ok = true;  // (no lane leaves alone: prefill.cu)
    for (int n = 0; PACKED ? ok && wget(n, u) : get(n, u); ++n) {
      int pos = 0, head = 0;
      float odd = 0.f, sum = 0.f;  // packed: turns NaN if a result of the row is not finite; the row's sum
      bool live;
      __nv_bfloat16* row_out;
      if constexpr (PACKED) {
        __syncwarp();
        if (lane == 0) put(n);
        pos = row / src.group;
        head = u.h * src.group + row - pos * src.group;
        live = pos < u.npos;
        row_out = p.out + ((int64_t)(u.q0 + pos) * src.heads + head) * D;
      } else {
        const int q = u.qt * BM + row;
        live = q < p.width;
        row_out = p.out + (int64_t)u.b * p.out_sb + (int64_t)q * p.out_sw + (int64_t)u.h * p.out_sh;
      }
      for (int pass = 0; pass < PASSES; ++pass, ++item) {
        if constexpr (!PACKED) {
          if (pass == PASSES - 1 && q_loader) {  // the next unit's queries, as the last S MMAs of this one free the chunks
            const int un = cta_unit(src, units, n + 1);
            if (un >= 0) load_q(n + 1, un);
          }
        }
        if constexpr (PACKED) {
          ok = wwait(&o_ready, item & 1) && wwait(&l_full, item & 1);
          if (!ok) break;
        } else {
          wait(&o_ready, item & 1);
          wait(&l_full, item & 1);
        }
        tc_fence_after();
        __syncwarp();
        float l = 0.f;
#pragma unroll
        for (int y = 0; y < NWG; ++y) l += ctl.lsum[y][row];
        const float m = PACKED ? ctl.msum[row] : 0.f;
        mbar_arrive(&l_free);
        // A packed row that sees no key: zeros.
        float inv = PACKED && u.lim0 + pos <= 0 ? 0.f : l > 0.f ? 1.f / l : l;  // (l is 0, or NaN)
        if (PACKED && m == -INFINITY && u.lim0 + pos > 0) inv = NAN;  // every key it sees scores -inf: no softmax
        __nv_bfloat16* dst = row_out + pass * DH;
        if constexpr (PACKED) {
          if (u.part >= 0) {  // a part: fp32, a column of rows at a time
            float* part = src.parts + (int64_t)u.part * ((D + 2) * BM) + row;
            // (A row whose sum is NaN takes part whatever its maximum is, and makes the whole NaN.)
            part[D * BM] = u.lim0 + pos <= 0 ? -INFINITY : l == l ? m : INFINITY;
            part[(D + 1) * BM] = u.lim0 + pos > 0 ? l : 0.f;
            part += pass * DH * BM;
#pragma unroll 1
            for (int c = 0; c < DH / 32; ++c, part += 32 * BM) {
              float o[32];
              tmem_ld32(tbase + lane_off + COL_O + c * 32, o);
              if (c == DH / 32 - 1) {
                tc_fence_before();
                mbar_arrive(&o_free);
              }
#pragma unroll
              for (int i = 0; i < 32; ++i) part[i * BM] = o[i];
            }
            continue;
          }
        }
#pragma unroll 1
        for (int c = 0; c < DH / 64; ++c) {
          uint32_t r0[64];
          tmem_ld32_async(tbase + lane_off + COL_O + c * 64, r0);
          tmem_ld32_async(tbase + lane_off + COL_O + c * 64 + 32, r0 + 32);
          tmem_wait_ld();
          if (c == DH / 64 - 1) {  // O is in registers: the next pass may overwrite it
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
        if constexpr (PACKED) sum = l;
      }
      if constexpr (PACKED) {
        if (u.part >= 0 && u.part % u.b == 0 && row == 0)  // a unit's first part
          reinterpret_cast<PartMeta*>(src.meta + 8)[u.part / u.b] = {u.qt, u.h, u.q0, u.npos, u.k0, u.lim0, {0, 0}};
        const bool redo = live && u.part < 0 && odd != 0.f && sum == sum && ok;  // (a row whose sum is NaN is NaN)
        const unsigned rows = __ballot_sync(0xffffffffu, redo);
        if (rows && list.add(u, rows, lane)) list.run<D>(src, row - lane, p.qscale, p.out);
      }
    }
    if constexpr (PACKED) {
      if (!__any_sync(0xffffffffu, abort_flag != 0)) list.run<D>(src, row - lane, p.qscale, p.out);
    }
  }
  __syncthreads();
  if (abort_flag) {
    if (tid == 0) raise_status(p.status, kStatusTimeout);
    if ((warp == W_MMA || warp == W_MMA_PV) && elect_one()) {
      tc_commit(&drain);
      mbar_wait(&drain, 0);
    }
    if (tid == W_LOADK * 32) {
      constexpr int KR = PACKED ? 2 * KS : KS;  // K ring slots
      for (int i = issued_k > KR ? issued_k - KR : 0; i < issued_k; ++i) mbar_wait(&k_full[i % KR], (i / KR) & 1);
      for (int i = issued_v > VS ? issued_v - VS : 0; i < issued_v; ++i) mbar_wait(&v_full[i % VS], (i / VS) & 1);
      // the latest load of every query chunk (load i fills chunk i % DC for the (i / DC)-th time)
      for (int i = issued_q > DC ? issued_q - DC : 0; i < issued_q; ++i) mbar_wait(&q_full[i % DC], (i / DC) & 1);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == W_EPI) {
    tc_fence_after();
    tmem_dealloc(tbase, TMEM_COLS);
  }
}

bool make_map(CUtensorMap* map, const void* base, int64_t b, int64_t h, int64_t w, int64_t sb, int64_t sh,
              int64_t sw) {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      return (PFN_cuTensorMapEncodeTiled_v12000) nullptr;
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr);
  }();
  if (!fn) return false;
  cuuint64_t dims[4] = {512, (cuuint64_t)w, (cuuint64_t)h, (cuuint64_t)b};
  cuuint64_t strides[3] = {(cuuint64_t)sw * 2, (cuuint64_t)sh * 2, (cuuint64_t)sb * 2};
  cuuint32_t box[4] = {64, 128, 1, 1};
  cuuint32_t estr[4] = {1, 1, 1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(base), dims, strides, box, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace prefillw

cudaError_t launch_prefill_wide(const PrefillArgs& a, cudaStream_t stream) {
  using namespace prefillw;
  constexpr int SMEM_BYTES = Cfg<512>::SMEM_BYTES;
  CUtensorMap qm, km, vm;
  if (!make_map(&qm, a.q, a.batch, a.heads, a.width, a.q_sb, a.q_sh, a.q_sw) ||
      !make_map(&km, a.k, a.batch, a.heads, a.width, a.k_sb, a.k_sh, a.k_sw) ||
      !make_map(&vm, a.v, a.batch, a.heads, a.width, a.v_sb, a.v_sh, a.v_sw))
    return cudaErrorInvalidValue;
  static PerDevice configured;
  if (const cudaError_t e = allow_smem(prefill_wide_kernel<Sched, 512>, SMEM_BYTES, configured)) return e;
  Params p;
  p.batch = a.batch;
  p.heads = a.heads;
  p.width = a.width;
  p.qtiles = (a.width + BM - 1) / BM;
  p.qscale = a.scale * kLog2e;
  p.group = omni::prefill_group(a.batch * a.heads);
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
  return launch_dependent(prefill_wide_kernel<Sched, 512>, dim3(grid), dim3(THREADS), (size_t)SMEM_BYTES, stream, qm, km, vm, p,
                          sched ? *sched : prefill_round_robin());
}

template <int D>
cudaError_t launch_packed_wide_d(const PackedArgs& a, cudaStream_t stream) {
  using namespace prefillw;
  constexpr int SMEM_BYTES = Cfg<D>::SMEM_BYTES;
  const int positions = BM / (a.heads / a.kv_heads);
  CUtensorMap qm, km, vm;
  if (!packed_maps(a, positions, VK, &qm, &km, &vm)) return cudaErrorNotSupported;
  static PerDevice configured;
  if (const cudaError_t e = allow_smem(prefill_wide_kernel<PackedSrc, D>, SMEM_BYTES, configured)) return e;
  Params p{};
  p.qscale = a.scale * kLog2e;
  p.out = reinterpret_cast<__nv_bfloat16*>(a.out);
  p.status = a.status;
  const pfx::PackedSrc src = packed_source(a, positions);
  const cudaError_t e = launch_dependent(prefill_wide_kernel<PackedSrc, D>, dim3(packed_grid(a, positions)), dim3(THREADS),
                                         (size_t)SMEM_BYTES, stream, qm, km, vm, p, src);
  return e != cudaSuccess ? e : launch_packed_join(a, src, stream);
}

cudaError_t launch_packed_tc_wide(const PackedArgs& a, cudaStream_t stream) {
  return a.dim == 256 ? launch_packed_wide_d<256>(a, stream) : launch_packed_wide_d<512>(a, stream);
}

}  // namespace omni
