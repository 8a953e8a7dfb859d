// er_kv_attend_bf16.cu -- attention over bf16 paged key-value caches.
#include "er_kv_attend_mma.cuh"

namespace er {

KernelShape attend_shape_bf16(int d, int group, int q_dtype) {
  return q_dtype == ER_DTYPE_BF16 ? shape_dp<__nv_bfloat16, __nv_bfloat16>(d, group) : shape_dp<__nv_bfloat16, float>(d, group);
}

int attend_bf16(const AttendArgs& a, int q_dtype, cudaStream_t st) {
  return q_dtype == ER_DTYPE_BF16 ? attend_dp<__nv_bfloat16, __nv_bfloat16>(a, st) : attend_dp<__nv_bfloat16, float>(a, st);
}

}  // namespace er
