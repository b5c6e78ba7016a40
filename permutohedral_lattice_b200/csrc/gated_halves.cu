// The gated feed-forward block of rows of 16-bit values.
#include "gated_launch.cuh"

namespace pl {

int gated_halves(GatedArgs p, int dtype, GatedPass pass, bool pack, cudaStream_t st) {
    return dtype == PL_F16 ? gated_of<__half>(p, pass, pack, st) : gated_of<__nv_bfloat16>(p, pass, pack, st);
}

}  // namespace pl
