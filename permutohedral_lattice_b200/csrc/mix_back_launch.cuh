// The launches of the kernels of the gradients, for the translation units that compile them.
#pragma once
#include "mix_launch.cuh"

namespace pl {

template <typename T>
static constexpr int dtype_of() { return std::is_same<T, float>::value ? PL_F32 : std::is_same<T, __half>::value ? PL_F16 : PL_BF16; }

static int add_shares(const MixBackArgs& a, const pl_mix_gradients& d, int ctas, cudaStream_t st) {
    const unsigned grid = (unsigned)(((a.k + a.k2 + 1) * a.n + 31) / 32);
#define PL_ADD(W) \
    mix_add_shares<W><<<grid, 256, 0, st>>>(a.shares, ctas, a.k, a.k2, a.n, static_cast<W*>(d.weight), static_cast<W*>(d.weight2), static_cast<W*>(d.bias))
    if (a.weight_dtype == PL_F32) PL_ADD(float);
    else if (a.weight_dtype == PL_F16) PL_ADD(__half);
    else PL_ADD(__nv_bfloat16);
#undef PL_ADD
    PL_COUNT_LAUNCHES(1);
    PL_CUDA(cudaGetLastError());
    return PL_OK;
}

template <typename T, bool PACKED, int MB, int NB>
static int launch_narrow(MixBackArgs a, const pl_mix_gradients& d, cudaStream_t st) {
    // in 8 bits: one stage, and as many blocks of rows as give 32 headers of each array (see mix_backward)
    const int widest = std::max(a.n, std::max(a.k, a.k2));
    const MixLaunch l = mix_launch(a.rows, 32, 32 * sizeof(T) * (2 * a.n + 2 * (a.k + a.k2)), MB * NB > 12 ? 2 : BACK_CTAS, PACKED ? 1 : MIX_STAGES,
                                   PACKED ? std::max(1, 32 / widest) : 8, [&](int warps, int stages, int blocks) {
                                       MixBackArgs b = a;
                                       b.blocks = blocks, b.stages = stages;
                                       return std::max(MixBackSmem(b, warps, NB, sizeof(T), PACKED).bytes(warps), mix_share_bytes(warps, MB, NB));
                                   });
    a.stages = l.stages, a.blocks = l.blocks;
    PL_TRY((ensure_dynamic_smem<mix_backward<T, PACKED, MB, NB>>(l.smem)));
    mix_backward<T, PACKED, MB, NB><<<l.ctas, 32 * l.warps, l.smem, st>>>(a);
    PL_COUNT_LAUNCHES(1);
    PL_CUDA(cudaGetLastError());
    return a.shares ? add_shares(a, d, l.ctas, st) : PL_OK;
}
// dW in blocks of eight channels: rows an even number of them in all (what narrow() allows is at most 80), columns as many as there are.  A warp
// sums all blocks that are compiled, there or not, so that few rows of dW have kernels of their own.  us of dW and dx at 16, 48 and 80 rows of dW:
// four million rows of 8 channels to 8 134, 181 and 236, of 8 + 8 151, 199 and 251; two million of 24 to 16 with 48 and 80 133 and 183, of 21 + 21 to
// 21 213 and 336.  (With four blocks of columns only 80: 24 to 32 349 us, where 80 to 32 takes 470.)
template <typename T, bool PACKED>
static int narrow_any(const MixBackArgs& a, const pl_mix_gradients& d, cudaStream_t st) {
    const int rows = up8(a.k) + up8(a.k2), blocks = up8(a.n) / 8;
    if (rows <= 16 && blocks == 1) return launch_narrow<T, PACKED, 1, 1>(a, d, st);
    if (rows <= 48 && blocks <= 3)
        return blocks == 1   ? launch_narrow<T, PACKED, 3, 1>(a, d, st)
               : blocks == 2 ? launch_narrow<T, PACKED, 3, 2>(a, d, st)
                             : launch_narrow<T, PACKED, 3, 3>(a, d, st);
    return blocks == 1   ? launch_narrow<T, PACKED, 5, 1>(a, d, st)
           : blocks == 2 ? launch_narrow<T, PACKED, 5, 2>(a, d, st)
           : blocks == 3 ? launch_narrow<T, PACKED, 5, 3>(a, d, st)
                         : launch_narrow<T, PACKED, 5, 4>(a, d, st);
}

template <typename T>
static int launch_wide(const MixBackArgs& a, const pl_mix_gradients& d, cudaStream_t st) {
    mix_dz<T><<<grid_for(a.rows, 8, 8), 256, 0, st>>>(a);
    PL_COUNT_LAUNCHES(1);
    PL_CUDA(cudaGetLastError());
    for (int second = 0; second < 2; second++) {
        void* to = second ? a.dx2 : a.dx;
        if (!to) continue;
        MixArgs f = {};
        f.rows = a.rows;
        f.k = a.n, f.n = second ? a.k2 : a.k;
        f.activation = PL_ACT_NONE;
        f.x = a.dz, f.out = to;
        f.weight = second ? a.weight2 : a.weight;
        f.weight_dtype = a.weight_dtype, f.transposed = 1;
        PL_TRY(mix_forward_floats(f, dtype_of<T>(), st));
    }
    if (!a.shares) return PL_OK;
    PL_TRY((ensure_dynamic_smem<mix_backward_weights<T>>(WIDE_SMEM)));
    const unsigned ctas = grid_for(a.rows, WIDE_ROWS, 1);
    mix_backward_weights<T><<<dim3(ctas, a.want_x2 ? 2 : 1), 256, WIDE_SMEM, st>>>(a);
    PL_COUNT_LAUNCHES(1);
    PL_CUDA(cudaGetLastError());
    return add_shares(a, d, (int)ctas, st);
}

template <typename T>
static int launch_back(const MixBackArgs& a, const pl_mix_gradients& d, cudaStream_t st) {
    if (!mix_narrow(a.k, a.k2, a.n)) return launch_wide<T>(a, d, st);
    if (tiny(a.k, a.k2, a.n)) {
        const unsigned ctas = grid_for(a.rows, 256 * TINY_BACK_ROWS, 2);
        const void* rows[] = {a.grad, a.out.full, a.x.full, a.x2.full, a.dx, a.dx2, a.dresidual};
        const int v = tiny_channels(a.k, a.k2, a.n, sizeof(T), rows, 7);
        if (v == 4) mix_tiny_backward<T, 4><<<ctas, 256, 0, st>>>(a);
        else if (v == 2) mix_tiny_backward<T, 2><<<ctas, 256, 0, st>>>(a);
        else mix_tiny_backward<T, 0><<<ctas, 256, 0, st>>>(a);
        PL_COUNT_LAUNCHES(1);
        PL_CUDA(cudaGetLastError());
        return a.shares ? add_shares(a, d, (int)ctas, st) : PL_OK;
    }
    return a.out.codes || a.x.codes || a.x2.codes ? narrow_any<T, true>(a, d, st) : narrow_any<T, false>(a, d, st);
}

}  // namespace pl
