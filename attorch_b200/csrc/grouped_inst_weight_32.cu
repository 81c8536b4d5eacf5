// Instantiates the grouped product (weight) for fp32 elements, multiplied as TF32.
#include "grouped_launch.cuh"

namespace ab200 {
int launch_grouped_weight_32(const GroupedProblem& p, int bn, bool pair, cudaStream_t stream) {
  if (pair) return launch_grouped_cfg<GroupedCfg<256, 4, true, true, 2>>(p, stream);
  if (bn == 128) return launch_grouped_cfg<GroupedCfg<128, 4, true, true>>(p, stream);
  return ERR_BAD_SHAPE;
}
}  // namespace ab200
