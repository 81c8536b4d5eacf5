// Instantiates the grouped product (input) for 2-byte elements.
#include "grouped_launch.cuh"

namespace ab200 {
int launch_grouped_input_16(const GroupedProblem& p, int bn, bool pair, cudaStream_t stream) {
  if (pair) return launch_grouped_cfg<GroupedCfg<256, 2, false, false, 2>>(p, stream);
  if (bn == 64) return launch_grouped_cfg<GroupedCfg<64, 2, false, false>>(p, stream);
  if (bn == 128) return launch_grouped_cfg<GroupedCfg<128, 2, false, false>>(p, stream);
  if (bn == 256) return launch_grouped_cfg<GroupedCfg<256, 2, false, false>>(p, stream);
  return ERR_BAD_SHAPE;
}
}  // namespace ab200
