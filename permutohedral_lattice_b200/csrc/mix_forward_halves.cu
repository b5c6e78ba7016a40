// Channel products of rows of 16-bit values.
#include "mix_launch.cuh"

namespace pl {

template <typename T>
static int forward_halves(const MixArgs& a, cudaStream_t st) {
    if (tiny(a.k, a.k2, a.n)) return launch_tiny<T>(a, st);
    if (a.weight_dtype != PL_F32) return forward_of<T, T, MIX_PAIRS>(a, st);
    // As for floats.  Beyond the rounding of a result to float16 75 channels of mixed signs to 16 are 1.4e-7 of the terms' magnitudes off,
    // in parts 4e-8, which shows where they cancel; us of two million rows 101 and 98, 64 to 32 131 and 138, one million rows of 128 to 32
    // 135 and 147.
    if (a.k + a.k2 <= 48 && a.n <= 32) return forward_of<T, T, MIX_PLAIN>(a, st);
    return forward_of<T, T, MIX_PARTED>(a, st);
}

int mix_forward_halves(const MixArgs& a, int dtype, cudaStream_t st) {
    return dtype == PL_F16 ? forward_halves<__half>(a, st) : forward_halves<__nv_bfloat16>(a, st);
}

}  // namespace pl
