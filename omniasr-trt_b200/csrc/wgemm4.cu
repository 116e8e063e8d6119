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
// A CTA takes one 16-row tile (SwiGLU: 8 gate and their 8 inner rows), its warps the blocks of 128 columns in turn, a few
// of a warp's blocks in flight; their sums meet in shared memory in warp order. Measured: 8 tokens, 2 x 11008 x 4096 SwiGLU, 13.4 us (7.1 at HBM's
// rate). From between 16 and 32 tokens on the tokens' reads out of L2 bound it: 22016 x 4096, 64 tokens 75 us (a bf16 library product 37).

#include <type_traits>

#include "attention.cuh"
#include "common.cuh"
#include "int4.cuh"
#include "wgemm4.cuh"

namespace omni {
namespace {

OMNI_DEV void mma_bf16(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Codes 2 i and 2 i + 1 of a word as bf16 (c - 8). `mask` is 0x000f000f out of the kernel's parameters: with two immediates the and-or
// would be two instructions.
OMNI_DEV uint32_t pair_of(uint32_t w, int i, uint32_t mask) {
  const uint32_t v = ((w >> (4 * i)) & mask) | 0x43004300u;  // 128 + c
  uint32_t r;
  asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(v), "r"(0x43084308u));
  return r;
}

// Tokens come from the kernel before: an ordinary load, which stays behind the wait for it.
OMNI_DEV uint4 token_words(const __nv_bfloat16* p) { return *reinterpret_cast<const uint4*>(p); }

// A block of 128 columns of two weight rows (words u0, u1; scales f0, f1 per group) times NT tiles of 8 tokens; x(n, w): a lane's 8
// columns 32 w + 8 t .. of token n * 8 + g.
template <int NT, int PER, typename X>
OMNI_DEV void block_product(const uint4& u0, const uint4& u1, const uint32_t (&f0)[PER], const uint32_t (&f1)[PER], uint32_t mask, X x,
                            float (&acc)[NT][4]) {
  const uint32_t w0[4] = {u0.x, u0.y, u0.z, u0.w}, w1[4] = {u1.x, u1.y, u1.z, u1.w};
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
      p0[i] = pair_of(w0[w], i, mask);
      p1[i] = pair_of(w1[w], i, mask);
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const uint4 v = x(n, w);
      mma_bf16(sum[n], p0[0], p1[0], p0[1], p1[1], v.x, v.y);
      mma_bf16(sum[n], p0[2], p1[2], p0[3], p1[3], v.z, v.w);
    }
    if ((w + 1) % (4 / PER) == 0) {
      const float e0 = bf16_value(f0[w / (4 / PER)]), e1 = bf16_value(f1[w / (4 / PER)]);
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

constexpr int kAhead = 4;  // blocks of a warp in flight

// NT tiles of 8 tokens, PER groups per block of 128 columns, W warps. (CTAs per SM for the registers: with fewer of them a CTA's
// loads wait for the ones before.)
template <int NT, int PER, int W>
__global__ void __launch_bounds__(32 * W, W == 4 ? 5 : NT <= 4 ? 2 : 1) gemm4_kernel(const Gemm4Args a) {
  __shared__ float sums[W][8 * NT][17];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  grid_launch_dependents();
  const bool swiglu = a.mode == kGemmSwiglu;
  const int outs = swiglu ? 8 : 16, j0 = blockIdx.x * outs;
  // This lane's two weight rows (past the last: the last, whose sums nobody takes).
  const int r0 = min(j0 + g, a.n - 1), r1 = swiglu ? a.n + r0 : min(j0 + 8 + g, a.n - 1);
  const uint4* c0 = a.codes + ((int64_t)(r0 >> 3) * a.blocks * 8 + (r0 & 7)) * 4 + t + warp * 32;
  const uint4* c1 = a.codes + ((int64_t)(r1 >> 3) * a.blocks * 8 + (r1 & 7)) * 4 + t + warp * 32;
  const uint16_t* s0 = a.scales + (int64_t)(r0 >> 3) * a.groups * 8 + (r0 & 7) + warp * PER * 8;
  const uint16_t* s1 = a.scales + (int64_t)(r1 >> 3) * a.groups * 8 + (r1 & 7) + warp * PER * 8;
  const __nv_bfloat16* x[NT];  // (of a token past the last: the last)
#pragma unroll
  for (int n = 0; n < NT; ++n) x[n] = a.x + min(n * 8 + g, a.rows - 1) * a.ldx + warp * 128 + t * 8;
  float acc[NT][4];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[n][i] = 0.f;
  bool waited = false;
  const int whole = a.k / 128;
  int b = warp;
  auto run = [&](auto count) {  // `count` of the warp's blocks, all whole, their weights in flight together
    constexpr int N = decltype(count)::value;
    uint4 u0[N], u1[N];
    uint32_t f0[N][PER], f1[N][PER];
#pragma unroll
    for (int p = 0; p < N; ++p) {
      u0[p] = __ldcs(c0 + p * W * 32);
      u1[p] = __ldcs(c1 + p * W * 32);
    }
#pragma unroll
    for (int p = 0; p < N; ++p)
#pragma unroll
      for (int q = 0; q < PER; ++q) {
        f0[p][q] = __ldg(s0 + (p * W * PER + q) * 8);
        f1[p][q] = __ldg(s1 + (p * W * PER + q) * 8);
      }
    if (!waited) {  // (the weights do not come from the kernel before)
      grid_dependency_wait();
      waited = true;
    }
#pragma unroll
    for (int p = 0; p < N; ++p)
      block_product<NT, PER>(u0[p], u1[p], f0[p], f1[p], a.mask,
                             [&](int n, int w) { return token_words(x[n] + p * W * 128 + w * 32); }, acc);
    c0 += N * W * 32;
    c1 += N * W * 32;
    s0 += N * W * PER * 8;
    s1 += N * W * PER * 8;
#pragma unroll
    for (int n = 0; n < NT; ++n) x[n] += N * W * 128;
    b += N * W;
  };
  while (b + (kAhead - 1) * W < whole) run(std::integral_constant<int, kAhead>());
  while (b < whole) run(std::integral_constant<int, 1>());
  if (b < a.blocks) {  // the last block, cut short (one warp's)
    const uint4 u0 = __ldcs(c0), u1 = __ldcs(c1);
    uint32_t f0[PER], f1[PER];
#pragma unroll
    for (int q = 0; q < PER; ++q) {
      const bool on = b * PER + q < a.groups;
      f0[q] = on ? __ldg(s0 + q * 8) : 0u;
      f1[q] = on ? __ldg(s1 + q * 8) : 0u;
    }
    if (!waited) grid_dependency_wait();
    waited = true;
    block_product<NT, PER>(u0, u1, f0, f1, a.mask,
                           [&](int n, int w) {
                             return b * 128 + w * 32 + t * 8 < a.k ? token_words(x[n] + w * 32) : make_uint4(0u, 0u, 0u, 0u);
                           },
                           acc);
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
  for (int e = threadIdx.x; e < outs * a.rows; e += 32 * W) {
    const int m = swiglu ? e >> 3 : e >> 4, j = e & (outs - 1), col = j0 + j;
    if (col >= a.n) continue;
    float y = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) y += sums[w][m][j];
    if (swiglu) {
      float inner = 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w) inner += sums[w][m][j + 8];
      y = inner * (y / (1.f + __expf(-y)));
    } else if (a.mode == kGemmResidual) {
      y += __bfloat162float(a.residual[m * a.ld_res + col]);
    }
    a.y[m * a.ld_y + col] = __float2bfloat16_rn(y);
  }
}

template <int NT, int W>
cudaError_t launch(const Gemm4Args& a, int tiles, cudaStream_t s) {
  const dim3 grid((unsigned)tiles), block(32 * W);
  if (a.group == 128) return launch_dependent(gemm4_kernel<NT, 1, W>, grid, block, 0, s, a);
  if (a.group == 64) return launch_dependent(gemm4_kernel<NT, 2, W>, grid, block, 0, s, a);
  return launch_dependent(gemm4_kernel<NT, 4, W>, grid, block, 0, s, a);
}

}  // namespace

cudaError_t launch_decode_gemm_int4(const Gemm4Args& args, cudaStream_t s) {
  Gemm4Args a = args;
  a.mask = 0x000f000fu;
  const int tiles = a.mode == kGemmSwiglu ? (a.n + 7) / 8 : (a.n + 15) / 16, sms = device_sm_count();
  if (a.rows <= 8) {
    // Five CTAs of 4 warps on an SM or two of 8: a wave of the former takes 2.2 times as long (k = 4096: 7 against 3.2 us).
    const int four = (tiles + 5 * sms - 1) / (5 * sms), eight = (tiles + 2 * sms - 1) / (2 * sms);
    return four * 11 < eight * 5 ? launch<1, 4>(a, tiles, s) : launch<1, 8>(a, tiles, s);
  }
  if (a.rows <= 16) return launch<2, 8>(a, tiles, s);
  if (a.rows <= 32) return launch<4, 8>(a, tiles, s);
  return launch<8, 8>(a, tiles, s);
}

}  // namespace omni
