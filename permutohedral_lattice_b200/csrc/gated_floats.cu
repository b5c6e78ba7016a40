// The gated feed-forward block of rows of floats.
#include "gated_launch.cuh"

namespace pl {

int gated_floats(GatedArgs p, GatedPass pass, bool pack, cudaStream_t st) { return gated_of<float>(p, pass, pack, st); }

}  // namespace pl
