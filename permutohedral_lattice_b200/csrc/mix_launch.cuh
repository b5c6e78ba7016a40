// The launches of the forward kernels, for the translation units that compile them.
#pragma once
#include "mix_host.h"
#include "mix_tiny.cuh"

namespace pl {

template <typename TI, typename TO, int NT, int MT, int WAY>
static int launch_forward(MixArgs a, cudaStream_t st) {
    // Rows lie apart where that is of use (see RowsApart); what is packed from there has aligned codes, and whole blocks, which 32 rows
    // and a last block of rows of a multiple of 32 values are.
    auto may = [&](int c, const void* p, const void* q, const void* codes) {
        return aligned(p, 16) && aligned(q, 16) && (!codes || (aligned(codes, 4) && (c % PACK_BLOCK == 0 || a.rows % 32 == 0)));
    };
    a.x_apart = may(a.k, a.x, nullptr, a.x_codes), a.x2_apart = may(a.k2, a.x2, nullptr, a.x2_codes);
    a.out_apart = may(a.n, a.out, a.residual, a.out_codes);
    const MixLaunch l = mix_launch(a.rows, 16 * MT, 16 * MT * (sizeof(TI) * (a.k + a.k2 + (a.residual ? a.n : 0)) + sizeof(TO) * a.n),
                                   mix_forward_ctas(NT, WAY), 1, 8,
                                   [&](int warps, int, int blocks) { return MixSmem<TI, TO>(a, 16 * MT * blocks, NT, WAY).bytes(warps); });
    a.blocks = l.blocks;
    if constexpr (MT == 2 && std::is_same<TI, TO>::value) {
        if (a.x_codes || a.x2_codes || a.out_codes) {
            PL_TRY((ensure_dynamic_smem<mix_forward<TI, TO, NT, MT, WAY, true>>(l.smem)));
            mix_forward<TI, TO, NT, MT, WAY, true><<<l.ctas, 32 * l.warps, l.smem, st>>>(a);
            PL_COUNT_LAUNCHES(1);
            PL_CUDA(cudaGetLastError());
            return PL_OK;
        }
    }
    PL_TRY((ensure_dynamic_smem<mix_forward<TI, TO, NT, MT, WAY, false>>(l.smem)));
    mix_forward<TI, TO, NT, MT, WAY, false><<<l.ctas, 32 * l.warps, l.smem, st>>>(a);
    PL_COUNT_LAUNCHES(1);
    PL_CUDA(cudaGetLastError());
    return PL_OK;
}
// Output channels in steps of 8: the accumulators of a warp's rows are in registers.  From 65 channels on a warp takes
// 16 rows in place of 32, of 16-bit values: rows of floats have kernels of their own there (see forward_floats).
template <typename TI, typename TO, int WAY>
static int forward_of(const MixArgs& a, cudaStream_t st) {
    if (a.n <= 8) return launch_forward<TI, TO, 1, 2, WAY>(a, st);
    if (a.n <= 16) return launch_forward<TI, TO, 2, 2, WAY>(a, st);
    if (a.n <= 24) return launch_forward<TI, TO, 3, 2, WAY>(a, st);
    if (a.n <= 32) return launch_forward<TI, TO, 4, 2, WAY>(a, st);
    if constexpr (WAY != MIX_PLAIN) {
        if (a.n <= 40) return launch_forward<TI, TO, 5, 2, WAY>(a, st);
        if (a.n <= 48) return launch_forward<TI, TO, 6, 2, WAY>(a, st);
        if (a.n <= 56) return launch_forward<TI, TO, 7, 2, WAY>(a, st);
        if (a.n <= 64) return launch_forward<TI, TO, 8, 2, WAY>(a, st);
        if constexpr (sizeof(TI) == 2) return launch_forward<TI, TO, 16, 1, WAY>(a, st);
    }
    return PL_INTERNAL_ERROR;
}

// Channels of every operand where they are the same, 2 or 4, and all rows begin at multiples of their size; else 0.
static int tiny_channels(int k, int k2, int n, size_t size, const void* const* rows, int count) {
    if (k != n || (k2 && k2 != n) || (n != 2 && n != 4)) return 0;
    for (int i = 0; i < count; i++)
        if (!aligned(rows[i], n * size)) return 0;
    return n;
}
static bool tiny(int k, int k2, int n) { return k <= TINY && k2 <= TINY && n <= TINY; }

template <typename T>
static int launch_tiny(const MixArgs& a, cudaStream_t st) {
    const unsigned grid = grid_for(a.rows, 256 * TINY_ROWS, 4);
    const void* rows[] = {a.x, a.x2, a.residual, a.out};
    const int v = tiny_channels(a.k, a.k2, a.n, sizeof(T), rows, 4);
    if (v == 4) mix_tiny<T, 4><<<grid, 256, 0, st>>>(a);
    else if (v == 2) mix_tiny<T, 2><<<grid, 256, 0, st>>>(a);
    else mix_tiny<T, 0><<<grid, 256, 0, st>>>(a);
    PL_COUNT_LAUNCHES(1);
    PL_CUDA(cudaGetLastError());
    return PL_OK;
}

}  // namespace pl
