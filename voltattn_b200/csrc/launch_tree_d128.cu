// Launchers of the tree-attention kernel (decode_tree.cuh), head dimension 128.
#include "launch_tree.cuh"

namespace va {
namespace host {

int launch_tree_d128(int fmt, const TreeParams& p, int rows, cudaStream_t st) {
    return launch_tree_dim<128>(fmt, p, rows, st);
}

}  // namespace host
}  // namespace va
