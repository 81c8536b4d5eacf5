// Instantiates the grouped product for e4m3 elements with block scales.
#include "grouped_launch.cuh"

namespace ab200 {
int launch_grouped_8(const GroupedProblem& p, int bn, bool pair, cudaStream_t stream) {
  if (pair) return launch_grouped_cfg<GroupedCfg<256, 1, false, false, 2>>(p, stream);
  if (bn == 32) return launch_grouped_cfg<GroupedCfg<32, 1, false, false>>(p, stream);
  if (bn == 64) return launch_grouped_cfg<GroupedCfg<64, 1, false, false>>(p, stream);
  if (bn == 128) return launch_grouped_cfg<GroupedCfg<128, 1, false, false>>(p, stream);
  return ERR_BAD_SHAPE;
}
}  // namespace ab200
