// er_kv_attend_f32.cu -- attention over fp32 paged key-value caches.
#include "er_kv_attend_mma.cuh"

namespace er {

KernelShape attend_shape_f32(int d, int group, int q_dtype) {
  return q_dtype == ER_DTYPE_BF16 ? shape_dp<float, __nv_bfloat16>(d, group) : shape_dp<float, float>(d, group);
}

int attend_f32(const AttendArgs& a, int q_dtype, cudaStream_t st) {
  return q_dtype == ER_DTYPE_BF16 ? attend_dp<float, __nv_bfloat16>(a, st) : attend_dp<float, float>(a, st);
}

}  // namespace er
