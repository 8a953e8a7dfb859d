// er_kv_tree_f32.cu -- tree attention over fp32 caches.
#include "er_kv_tree_mma.cuh"

namespace er {

namespace {
// Three parts of everything: fewer rows and tiles the wider the heads.
using S64 = TreeShape<3, 3, 3, 64, 128, 64, 2, 2>;
using S128 = TreeShape<3, 3, 3, 128, 64, 64, 1, 1>;
using S256 = TreeShape<3, 3, 3, 256, 32, 64, 1, 1>;

template <typename TQ>
int launch(const TreeArgs& a, const CUtensorMap* maps, cudaStream_t st) {
  const int d = a.kv.d;
  return d <= 64    ? tree_launch<S64, float, TQ>(a, maps, st)
         : d <= 128 ? tree_launch<S128, float, TQ>(a, maps, st)
                    : tree_launch<S256, float, TQ>(a, maps, st);
}
}  // namespace

TreeLaunch tree_shape_f32(int d) {
  return d <= 64 ? tree_shape<S64>() : d <= 128 ? tree_shape<S128>() : tree_shape<S256>();
}

int tree_f32(const TreeArgs& a, int q_dtype, const CUtensorMap* maps, cudaStream_t st) {
  return q_dtype == ER_DTYPE_BF16 ? launch<__nv_bfloat16>(a, maps, st) : launch<float>(a, maps, st);
}

}  // namespace er
