// Norms of rows of floats.
#include "norm_launch.cuh"

namespace pl {

int norm_of_floats(NormArgs& a, bool backward, int ctas, cudaStream_t st) { return norm_of<float>(a, backward, ctas, st); }

}  // namespace pl
