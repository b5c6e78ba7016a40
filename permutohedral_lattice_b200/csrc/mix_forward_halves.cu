// Channel products of rows of 16-bit values.
#include "mix_launch.cuh"

namespace pl {

template <typename T>
static int forward_halves(const MixArgs& a, cudaStream_t st) {
    if (tiny(a.k, a.k2, a.n)) return launch_tiny<T>(a, st);
    if (a.weight_dtype != PL_F32) return forward_of<T, T, MIX_PAIRS>(a, st);
    // Few products to a sum: what the tensor cores cut stays below 2^-21 of it (75 channels of one sign: 0.9e-6 off in all, so 0.2e-6).
    if (a.k + a.k2 <= 48 && a.n <= 32) return forward_of<T, T, MIX_PLAIN>(a, st);
    return forward_of<T, T, MIX_PARTED>(a, st);
}

int mix_forward_halves(const MixArgs& a, int dtype, cudaStream_t st) {
    return dtype == PL_F16 ? forward_halves<__half>(a, st) : forward_halves<__nv_bfloat16>(a, st);
}

}  // namespace pl
