// tree_attention of fp16 tensors: the kernel of tree_kernel.hpp for each shape.
#include "tree_kernel.hpp"

namespace slc_tree {
Plan plan_f16(int rows, int head_dim) { return plan_impl<slc::f16_t>(rows, head_dim); }
int launch_f16(const TreeArgs& a, const Plan& plan, hipStream_t stream) {
  return launch_impl<slc::f16_t>(a, plan, stream);
}
}  // namespace slc_tree
