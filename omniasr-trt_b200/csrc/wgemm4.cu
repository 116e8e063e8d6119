// Decode GEMM over 4-bit weights with group scales: y[m, j] = sum_k x[m, k] W[j, k], W[j, k] = s[j, k / group] (c[j, k] - 8), for at
// most 64 token rows; bf16 x and y, fp32 sums, one rounding after the epilogue (store, residual, SwiGLU).
//
// Bound by the weights' bytes (0.53 per weight with groups of 128; the products of 8 tokens are a tenth of what the tensor cores do
// meanwhile), so the weights go from global memory straight into the registers that feed the tensor cores, once: a lane's 16
// bytes are 32 codes of one weight row, and two of them (the rows g and g + 8 of a 16-row tile) the A operands of eight
// mma.m16n8k16. Dequantised tiles in shared memory, as tcgen05 would want them, would write and read four times the weights'
// bytes there, more than its bandwidth next to HBM's rate. A pair of codes becomes two bf16 by one shift, one and-or (128 + c,
// exact) and one packed subtraction (c - 8, exact); a group's sum is scaled once, in fp32.
//
// Layout of the codes (laid out once, kernels.int4_weights): 8 weight rows x 128 columns are 512 contiguous bytes, a row's 64
// of them 16 for each of the four lanes that hold it; lane t's word w has columns 32 w + 8 t .. + 7, even ones in the low half
// (nibbles 0 to 3), odd ones in the high half, so that a shift by 4 i brings columns 2 i, 2 i + 1 to the two halves, which is the
// order of the tokens' memory.
//
// A CTA takes one 16-row tile (SwiGLU: 8 gate and their 8 inner rows), its eight warps the blocks of 128 columns in turn, four of a
// warp's blocks in flight; their sums meet in shared memory in warp order.

#include "common.cuh"
#include "int4.cuh"
#include "wgemm4.cuh"

namespace omni {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kAhead = 4;  // blocks of a warp in flight

OMNI_DEV void mma_bf16(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Codes 2 i and 2 i + 1 of a word as bf16 (c - 8).
OMNI_DEV uint32_t pair_of(uint32_t w, int i) {
  const uint32_t v = ((w >> (4 * i)) & 0x000f000fu) | 0x43004300u;  // 128 + c
  uint32_t r;
  asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(v), "r"(0x43084308u));
  return r;
}

template <int NT, int PER>  // tiles of 8 tokens; groups per block of 128 columns
__global__ void __launch_bounds__(kThreads) gemm4_kernel(const Gemm4Args a) {
  __shared__ float sums[kWarps][8 * NT][17];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  grid_launch_dependents();
  const bool swiglu = a.mode == kGemmSwiglu;
  const int j0 = blockIdx.x * (swiglu ? 8 : 16);
  // This lane's two weight rows.
  const int r0 = j0 + g, r1 = swiglu ? a.n + j0 + g : j0 + 8 + g;
  const bool on0 = swiglu ? j0 + g < a.n : r0 < a.wrows, on1 = swiglu ? j0 + g < a.n : r1 < a.wrows;
  const uint4* c0 = a.codes + ((int64_t)(r0 >> 3) * a.blocks * 8 + (r0 & 7)) * 4 + t;
  const uint4* c1 = a.codes + ((int64_t)(r1 >> 3) * a.blocks * 8 + (r1 & 7)) * 4 + t;
  const uint16_t* s0 = a.scales + (int64_t)(r0 >> 3) * a.groups * 8 + (r0 & 7);
  const uint16_t* s1 = a.scales + (int64_t)(r1 >> 3) * a.groups * 8 + (r1 & 7);
  float acc[NT][4];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[n][i] = 0.f;
  bool waited = false;
  for (int b0 = warp; b0 < a.blocks; b0 += kWarps * kAhead) {
    uint4 u0[kAhead], u1[kAhead];
    uint32_t f0[kAhead][PER], f1[kAhead][PER];
#pragma unroll
    for (int p = 0; p < kAhead; ++p) {
      const int b = b0 + p * kWarps;
      const bool in = b < a.blocks;
      u0[p] = in && on0 ? __ldcs(c0 + (int64_t)b * 32) : make_uint4(0u, 0u, 0u, 0u);
      u1[p] = in && on1 ? __ldcs(c1 + (int64_t)b * 32) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
      for (int q = 0; q < PER; ++q) {
        const int s = b * PER + q;
        f0[p][q] = in && on0 && s < a.groups ? __ldg(s0 + (int64_t)s * 8) : 0u;
        f1[p][q] = in && on1 && s < a.groups ? __ldg(s1 + (int64_t)s * 8) : 0u;
      }
    }
    if (!waited) {  // (the weights do not come from the kernel before)
      grid_dependency_wait();
      waited = true;
    }
#pragma unroll
    for (int p = 0; p < kAhead; ++p) {
      const int b = b0 + p * kWarps;
      if (b >= a.blocks) break;
      const uint32_t w0[4] = {u0[p].x, u0[p].y, u0[p].z, u0[p].w}, w1[4] = {u1[p].x, u1[p].y, u1[p].z, u1[p].w};
      float sum[NT][4];
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        if (w % (4 / PER) == 0) {
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) sum[n][i] = 0.f;
        }
        uint32_t p0[4], p1[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          p0[i] = pair_of(w0[w], i);
          p1[i] = pair_of(w1[w], i);
        }
        const int col = b * 128 + w * 32 + t * 8;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const int m = n * 8 + g;
          const uint4 x = m < a.rows && col < a.k ? __ldg(reinterpret_cast<const uint4*>(a.x + m * a.ldx + col)) : make_uint4(0u, 0u, 0u, 0u);
          mma_bf16(sum[n], p0[0], p1[0], p0[1], p1[1], x.x, x.y);
          mma_bf16(sum[n], p0[2], p1[2], p0[3], p1[3], x.z, x.w);
        }
        if ((w + 1) % (4 / PER) == 0) {
          const int q = w / (4 / PER);
          const float e0 = bf16_value(f0[p][q]), e1 = bf16_value(f1[p][q]);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            acc[n][0] = fmaf(e0, sum[n][0], acc[n][0]);
            acc[n][1] = fmaf(e0, sum[n][1], acc[n][1]);
            acc[n][2] = fmaf(e1, sum[n][2], acc[n][2]);
            acc[n][3] = fmaf(e1, sum[n][3], acc[n][3]);
          }
        }
      }
    }
  }
  if (!waited) grid_dependency_wait();
  // [warp][token][row]: rows g, g + 8 and tokens 2 t, 2 t + 1 of each tile.
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    sums[warp][n * 8 + 2 * t][g] = acc[n][0];
    sums[warp][n * 8 + 2 * t + 1][g] = acc[n][1];
    sums[warp][n * 8 + 2 * t][g + 8] = acc[n][2];
    sums[warp][n * 8 + 2 * t + 1][g + 8] = acc[n][3];
  }
  __syncthreads();
  const int outs = swiglu ? 8 : 16;
  for (int e = threadIdx.x; e < outs * a.rows; e += kThreads) {
    const int m = e / outs, j = e - m * outs;
    if (j0 + j >= a.n) continue;
    float y = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) y += sums[w][m][j];
    if (swiglu) {
      float inner = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) inner += sums[w][m][j + 8];
      y = inner * (y / (1.f + __expf(-y)));
    } else if (a.mode == kGemmResidual) {
      y += __bfloat162float(a.residual[m * a.ld_res + j0 + j]);
    }
    a.y[m * a.ld_y + j0 + j] = __float2bfloat16_rn(y);
  }
}

template <int NT>
cudaError_t launch(const Gemm4Args& a, cudaStream_t s) {
  const int per = a.mode == kGemmSwiglu ? 8 : 16;
  const dim3 grid((unsigned)((a.n + per - 1) / per));
  if (a.group == 128) return launch_dependent(gemm4_kernel<NT, 1>, grid, dim3(kThreads), 0, s, a);
  if (a.group == 64) return launch_dependent(gemm4_kernel<NT, 2>, grid, dim3(kThreads), 0, s, a);
  return launch_dependent(gemm4_kernel<NT, 4>, grid, dim3(kThreads), 0, s, a);
}

}  // namespace

cudaError_t launch_decode_gemm_int4(const Gemm4Args& a, cudaStream_t s) {
  if (a.rows <= 8) return launch<1>(a, s);
  if (a.rows <= 16) return launch<2>(a, s);
  if (a.rows <= 32) return launch<4>(a, s);
  return launch<8>(a, s);
}

}  // namespace omni
