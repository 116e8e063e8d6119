// paged_norm_rope_kv: paged_rope_kv with q and k normed per head before they are rotated,
//   x -> x * rsqrt(mean(x^2) + eps) * w   (w [D], one for q and one for k),
// in the same pass: the vectors are in registers between their load and their store, so the norm costs no traffic.

#include "paged_rope.cuh"

namespace omni {

cudaError_t launch_paged_norm_rope_kv(int dtype, const PagedRopeArgs& a, cudaStream_t stream) {
  if (a.n <= 0) return cudaSuccess;
  return dtype == kBF16 ? rope_kind<__nv_bfloat16, true>(a, stream) : rope_kind<float, true>(a, stream);
}

}  // namespace omni
