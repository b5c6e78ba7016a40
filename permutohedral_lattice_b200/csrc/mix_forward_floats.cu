// Channel products of float rows.
#include "mix_launch.cuh"
#include "mix_tensor.cuh"

namespace pl {

template <typename TO>
static int launch_forward_wide(const MixArgs& a, cudaStream_t st) {
    const size_t smem = wide_smem(a.k, a.k2);
    PL_TRY((ensure_dynamic_smem<mix_forward_wide<TO>>(smem)));
    const long long tiles = (a.rows + 15) / 16;
    const unsigned ctas = (unsigned)std::min<long long>((tiles + WIDE_WARPS - 1) / WIDE_WARPS, num_sms());
    mix_forward_wide<TO><<<ctas, 32 * WIDE_WARPS, smem, st>>>(a);
    PL_COUNT_LAUNCHES(1);
    PL_CUDA(cudaGetLastError());
    return PL_OK;
}

template <typename TO, typename W>
static int launch_forward_tensor(const MixArgs& a, cudaStream_t st) {
    PL_TRY((ensure_dynamic_smem<mix_forward_tensor<TO, W>>(TC_SMEM)));
    mix_forward_tensor<TO, W><<<grid_for(a.rows, TC_ROWS, 1), TC_THREADS, TC_SMEM, st>>>(a);
    PL_COUNT_LAUNCHES(1);
    PL_CUDA(cudaGetLastError());
    return PL_OK;
}

template <typename TO>
static int forward_floats(const MixArgs& a, cudaStream_t st) {
    if constexpr (std::is_same<TO, float>::value) {
        if (tiny(a.k, a.k2, a.n) && !a.transposed) return launch_tiny<float>(a, st);   // (which takes weights as they are)
    }
    if (a.n > 64 && tensor_pays(a)) {
        if constexpr (!std::is_same<TO, float>::value) {
            if (a.weight_dtype != PL_F32) return launch_forward_tensor<TO, TO>(a, st);   // (the other weights are of the output's type)
        }
        return launch_forward_tensor<TO, float>(a, st);
    }
    if (a.n > 64) return launch_forward_wide<TO>(a, st);
    // Few products to a sum: what the tensor cores cut stays below 2^-21 of it.  Sums of one sign, off by parts of the norm: 16 x 512x512 rows of
    // 21 + 21 channels to 21 with a softmax 227 us and 4.7e-7, in parts 248 and 1.3e-7; 8 to 8 67 and 1.4e-7 either way; two million rows of
    // 75 channels to 16 138 and 7.3e-7, in parts 141 and 1.1e-7; 64 to 32 183 and 5.6e-7, in parts 189 and 1.2e-7.
    if (a.k + a.k2 <= 48 && a.n <= 32) return forward_of<float, TO, MIX_PLAIN>(a, st);
    return forward_of<float, TO, MIX_PARTED>(a, st);
}

int mix_forward_floats(const MixArgs& a, int out_dtype, cudaStream_t st) {
    return out_dtype == PL_F32   ? forward_floats<float>(a, st)
           : out_dtype == PL_F16 ? forward_floats<__half>(a, st)
                                 : forward_floats<__nv_bfloat16>(a, st);
}

}  // namespace pl
