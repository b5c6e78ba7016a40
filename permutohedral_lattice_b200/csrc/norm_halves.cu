// Norms of rows of 16-bit values.
#include "norm_launch.cuh"

namespace pl {

int norm_of_halves(NormArgs& a, int dtype, bool backward, int ctas, cudaStream_t st) {
    return dtype == PL_F16 ? norm_of<__half>(a, backward, ctas, st) : norm_of<__nv_bfloat16>(a, backward, ctas, st);
}

}  // namespace pl
