// The paged cache's write: RoPE of q and k (after a norm per head, where asked), k and v into the pages as they hold them
// (the model's type, e4m3 codes, 4-bit codes). Included by paged_cache.cu (without the norm) and paged_norm.cu (with it).
//
// It moves each byte once and computes next to nothing: HBM for prompts, latency for single tokens.
#pragma once

#include <cuda_fp8.h>

#include "attention.cuh"
#include "common.cuh"
#include "int4.cuh"
#include "paged.cuh"
#include "rope_kv.cuh"

namespace omni {
namespace {

constexpr int kOwnType = -1;  // pages of the model's type

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

constexpr int kRopeThreads = 256;

// One CTA: the vectors [item0, item0 + per) of one token (heads of q, then k, then v). A vector is taken by L lanes,
// 16 bytes per lane and step, so a thread keeps the same dims for all its vectors and loads their cos / sin once.
// IL vectors per thread are in flight together.
// (Prompts of 32 + 2 x 8 heads of 128, 291 MB: 61 us with four vectors per thread of which the fourth had nothing to do,
// 53 us, 5470 GB/s, with three and registers for six CTAs per SM; a CTA that walks tokens with the next one's loads in
// flight needs twice the registers: 93 us.)
// KIND: what the pages hold. NORM: q and k are normed per head first, x * rsqrt(mean x^2 + eps) * w, all in fp32 with the one rounding
// after the rotation; the weights come out of L1 (held in registers they cost a CTA per SM: 71 us for the prompts below with the norm, 65 without), and
// the sum of squares is a shuffle reduction over the vector's lanes of values that are there already.
template <typename T, int D, int KIND, bool NORM, int IL>
__global__ void __launch_bounds__(kRopeThreads, D * sizeof(T) > 512 ? 2 : KIND == kInt4 ? 5 : IL == 4 ? 5 : 6) paged_rope_kernel(const PagedRopeArgs a, int per) {
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
        u[j][v] = it < i1 ? reinterpret_cast<const uint4*>(src + (int64_t)it * D)[v * L + lane]
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
      const float4 f = pos_ok ? reinterpret_cast<const float4*>(a.cs + p * D + (v * L + lane) * kVec)[i]
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
      float inv_rms = 1.f;
      if constexpr (NORM) {
        if (!__all_sync(0xffffffffu, it >= a.heads + kvh)) {  // (a warp of v vectors has nothing to norm)
          float sum = 0.f;
#pragma unroll
          for (int v = 0; v < NV; ++v) {
            float x[kVec];
            Elem<T>::unpack(u[j][v], x);
#pragma unroll
            for (int i = 0; i < kVec; ++i) sum = fmaf(x[i], x[i], sum);
          }
#pragma unroll
          for (int o = L / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
          inv_rms = rsqrtf(fmaf(sum, 1.f / D, a.eps));
        }
      }
      if (turn) {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
          float x[kVec];
          Elem<T>::unpack(u[j][v], x);
          if constexpr (NORM) {
            float w[kVec];
            Elem<T>::unpack(reinterpret_cast<const uint4*>(it < a.heads ? a.q_norm : a.k_norm)[v * L + lane], w);
#pragma unroll
            for (int i = 0; i < kVec; ++i) x[i] = x[i] * inv_rms * w[i];
          }
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
      if constexpr (KIND == kFp8) {
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
      } else if constexpr (KIND == kInt4) {
        if (__all_sync(0xffffffffu, it < a.heads)) continue;
        constexpr int GL = 32 / kVec;  // lanes per group
        uint8_t* row = reinterpret_cast<uint8_t*>(is_k ? a.c.k : a.c.v) + dst;
        uint16_t* scales = reinterpret_cast<uint16_t*>(is_k ? a.c.k_scale : a.c.v_scale) + ((pg * kvh + h) * a.c.page + off) * (D / 32);
#pragma unroll
        for (int v = 0; v < NV; ++v) {
          Elem<T>::unpack(r[v], y[v]);  // the vector as the model's type holds it
          float lo = y[v][0], hi = y[v][0];
          uint32_t amax = 0u;  // (past infinity's bits: a NaN)
#pragma unroll
          for (int i = 0; i < kVec; ++i) {
            lo = fminf(lo, y[v][i]);
            hi = fmaxf(hi, y[v][i]);
            amax = max(amax, __float_as_uint(y[v][i]) & 0x7fffffffu);
          }
#pragma unroll
          for (int o = GL / 2; o > 0; o >>= 1) {
            lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
            hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
            amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, o));
          }
          const bool finite = amax < 0x7f800000u;
          const uint32_t bits = finite ? (uint32_t)__bfloat16_as_ushort(__float2bfloat16_rn((hi > -lo ? hi : lo) * -0.125f)) : 0x7fffu;
          const float s = finite ? bf16_value(bits) : 0.f;
          const bool fast = sizeof(T) == 2 && (s == 0.f || fabsf(s) >= kInt4Fast);
          const float inv = fast && s != 0.f ? __fdividef(1.f, s) : 0.f;
          if (write) {
            const int w = v * L + lane;  // the vector's 16-byte word
#pragma unroll
            for (int q = 0; q < kVec / 4; ++q) {
              const int quad = w * (kVec / 4) + q;
              reinterpret_cast<uint16_t*>(row)[is_k ? quad_at<D, true>(quad) : quad_at<D, false>(quad)] =
                  (uint16_t)(fast ? int4_codes_bf16(y[v] + 4 * q, inv) : int4_codes(y[v] + 4 * q, s));
            }
            if (lane % GL == 0) scales[w / GL] = (uint16_t)bits;
          }
        }
      } else if (write) {
        T* row = reinterpret_cast<T*>(is_k ? a.c.k : a.c.v) + dst;
#pragma unroll
        for (int v = 0; v < NV; ++v) reinterpret_cast<uint4*>(row)[v * L + lane] = r[v];
      }
    }
  }
}

template <typename T, int D, int KIND, bool NORM>
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
    case 1: return launch_dependent(paged_rope_kernel<T, D, KIND, NORM, 1>, grid, dim3(kRopeThreads), 0, s, a, per);
    case 2: return launch_dependent(paged_rope_kernel<T, D, KIND, NORM, 2>, grid, dim3(kRopeThreads), 0, s, a, per);
    case 3: return launch_dependent(paged_rope_kernel<T, D, KIND, NORM, 3>, grid, dim3(kRopeThreads), 0, s, a, per);
    default: return launch_dependent(paged_rope_kernel<T, D, KIND, NORM, 4>, grid, dim3(kRopeThreads), 0, s, a, per);
  }
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

template <typename T, int KIND, bool NORM>
cudaError_t rope_dim(const PagedRopeArgs& a, cudaStream_t s) {
#define CALL(D) rope_launch<T, D, KIND == kInt4 && D < 32 ? -1 : KIND, NORM>(a, s)
  if (KIND == kInt4 && a.c.dim < 32) return cudaErrorInvalidValue;
  OMNI_DIM_SWITCH(a.c.dim, CALL)
#undef CALL
}

template <typename T, bool NORM>
cudaError_t rope_kind(const PagedRopeArgs& a, cudaStream_t s) {
  if (a.c.type == kFp8) return rope_dim<T, kFp8, NORM>(a, s);
  if (a.c.type == kInt4) return rope_dim<T, kInt4, NORM>(a, s);
  return rope_dim<T, kOwnType, NORM>(a, s);
}

}  // namespace
}  // namespace omni
