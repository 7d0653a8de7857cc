// tree_attention of bf16 tensors: the kernel of tree_kernel.hpp for each shape.
#include "tree_kernel.hpp"

namespace slc_tree {
Plan plan_bf16(int rows, int head_dim) { return plan_impl<slc::bf16_t>(rows, head_dim); }
int launch_bf16(const TreeArgs& a, const Plan& plan, hipStream_t stream) {
  return launch_impl<slc::bf16_t>(a, plan, stream);
}
}  // namespace slc_tree
