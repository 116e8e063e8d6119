// Decode GEMM over 4-bit weights (wgemm4.cu).
#pragma once

#include <stdint.h>

#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "wgemm.cuh"

namespace omni {

struct Gemm4Args {
  const __nv_bfloat16* x;  // [rows, k], row stride ldx
  int64_t ldx;
  const uint4* codes;     // [ceil(weight rows / 8), blocks, 8, 4] 16-byte words
  const uint16_t* scales; // bf16 [ceil(weight rows / 8), groups, 8]
  int rows, n, k;         // token rows, outputs, reduction length
  int blocks, groups;     // ceil(k / 128), ceil(k / group)
  int group;              // 32, 64 or 128
  uint32_t mask;          // set by the launcher
  int mode;               // GemmMode: store, residual, SwiGLU
  const __nv_bfloat16* residual;
  int64_t ld_res;
  __nv_bfloat16* y;
  int64_t ld_y;
};
cudaError_t launch_decode_gemm_int4(const Gemm4Args& a, cudaStream_t stream);

}  // namespace omni
