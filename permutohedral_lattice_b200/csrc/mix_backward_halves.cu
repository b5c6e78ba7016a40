// Gradients of channel products of rows of 16-bit values.
#include "mix_back_launch.cuh"

namespace pl {

int mix_backward_halves(const MixBackArgs& a, int dtype, const pl_mix_gradients& d, cudaStream_t st) {
    return dtype == PL_F16 ? launch_back<__half>(a, d, st) : launch_back<__nv_bfloat16>(a, d, st);
}

}  // namespace pl
