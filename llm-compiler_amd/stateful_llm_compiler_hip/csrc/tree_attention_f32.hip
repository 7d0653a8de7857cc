// tree_attention of fp32 tensors: the kernel of tree_kernel.hpp for each shape.
#include "tree_kernel.hpp"

namespace slc_tree {
Plan plan_f32(int rows, int head_dim) { return plan_impl<float>(rows, head_dim); }
int launch_f32(const TreeArgs& a, const Plan& plan, hipStream_t stream) {
  return launch_impl<float>(a, plan, stream);
}
}  // namespace slc_tree
