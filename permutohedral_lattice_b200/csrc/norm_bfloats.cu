// Norms of rows of bfloat16.
#include "norm_launch.cuh"

namespace pl {

int norm_of_bfloats(NormArgs& a, bool backward, int ctas, cudaStream_t st) { return norm_of<__nv_bfloat16>(a, backward, ctas, st); }

}  // namespace pl
