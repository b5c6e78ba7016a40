// Norms of rows of float16.
#include "norm_launch.cuh"

namespace pl {

int norm_of_halves(NormArgs& a, bool backward, int ctas, cudaStream_t st) { return norm_of<__half>(a, backward, ctas, st); }

}  // namespace pl
