// Gradients of channel products of float rows.
#include "mix_back_launch.cuh"

namespace pl {

int mix_backward_floats(const MixBackArgs& a, const pl_mix_gradients& d, cudaStream_t st) { return launch_back<float>(a, d, st); }

}  // namespace pl
