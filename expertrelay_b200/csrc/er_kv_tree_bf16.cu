// er_kv_tree_bf16.cu -- tree attention over bf16 caches.
#include "er_kv_tree_mma.cuh"

namespace er {

namespace {
using bf = __nv_bfloat16;
// By head_dim, as much as fits: 128 rows of queries, tiles of keys and of values under way. fp32 queries take three
// times the room.
using B64 = TreeShape<1, 1, 2, 64, 128, 64, 6, 6>;
using B128 = TreeShape<1, 1, 2, 128, 128, 64, 4, 4>;
using B256 = TreeShape<1, 1, 2, 256, 128, 64, 2, 2>;
using F64 = TreeShape<1, 3, 3, 64, 128, 64, 6, 6>;
using F128 = TreeShape<1, 3, 3, 128, 128, 64, 3, 2>;
using F256 = TreeShape<1, 3, 3, 256, 64, 64, 2, 2>;
}  // namespace

TreeLaunch tree_shape_bf16(int d, int q_dtype) {
  if (q_dtype == ER_DTYPE_BF16) return d <= 64 ? tree_shape<B64>() : d <= 128 ? tree_shape<B128>() : tree_shape<B256>();
  return d <= 64 ? tree_shape<F64>() : d <= 128 ? tree_shape<F128>() : tree_shape<F256>();
}

int tree_bf16(const TreeArgs& a, int q_dtype, const CUtensorMap* maps, cudaStream_t st) {
  const int d = a.kv.d;
  if (q_dtype == ER_DTYPE_BF16)
    return d <= 64    ? tree_launch<B64, bf, bf>(a, maps, st)
           : d <= 128 ? tree_launch<B128, bf, bf>(a, maps, st)
                      : tree_launch<B256, bf, bf>(a, maps, st);
  return d <= 64    ? tree_launch<F64, bf, float>(a, maps, st)
         : d <= 128 ? tree_launch<F128, bf, float>(a, maps, st)
                    : tree_launch<F256, bf, float>(a, maps, st);
}

}  // namespace er
