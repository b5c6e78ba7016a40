// Host side that the translation units of the channel products share: launch shapes, and what one calls of another.
#pragma once
#include <algorithm>
#include <stdint.h>

#include "host_calls.h"
#include "mix_backward.cuh"
#include "mix_forward.cuh"

namespace pl {

static unsigned grid_for(long long items, long long per_cta, int ctas_per_sm) {
    return (unsigned)std::max(1ll, std::min((items + per_cta - 1) / per_cta, (long long)num_sms() * ctas_per_sm));
}
static size_t size_of(int dtype) { return dtype == PL_F32 ? 4 : 2; }
static bool aligned(const void* p, size_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

// act(x W ...) of rows of floats (the output of any type), and of 16-bit values (the output alike).
int mix_forward_floats(const MixArgs& a, int out_dtype, cudaStream_t st);
int mix_forward_halves(const MixArgs& a, int dtype, cudaStream_t st);
// All gradients that `a` asks for; d: where those of the weights go.
int mix_backward_floats(const MixBackArgs& a, const pl_mix_gradients& d, cudaStream_t st);
int mix_backward_halves(const MixBackArgs& a, int dtype, const pl_mix_gradients& d, cudaStream_t st);
inline bool mix_narrow(int k, int k2, int n) { return up8(k) + up8(k2) <= 80 && n <= 32; }
constexpr int BACK_CTAS = 3;   // of an SM, at most: as many shares of dW there may be
// Whether the forward pass packs what is kept in 8 bits itself: up to 64 channels out, in blocks of 32 rows.
inline bool mix_keeps_in_forward(int n) { return n <= 64; }

constexpr size_t SMEM_SM = 228 * 1024, SMEM_CTA = 227 * 1024;   // shared memory of an SM, and the most that a CTA may have
// How a kernel runs whose warps have tiles of their own, smem(warps, stages, blocks) bytes a CTA: blocks of rows in a tile, stages of
// a warp, warps of a CTA, CTAs.
struct MixLaunch {
    int warps, stages, blocks, ctas;
    size_t smem;
};
template <typename Smem>
static MixLaunch mix_launch(long long rows, int block_rows, size_t block_bytes, int most_ctas, int most_stages, int most_blocks, Smem smem) {
    MixLaunch l;
    const long long all = (rows + block_rows - 1) / block_rows;
    // A tile of some 4 KB, as long as there are tiles for four warps of every SM.  (Four warps a CTA however few rows there are: they share
    // the work of reading the weights.)
    l.blocks = (int)std::max<size_t>(1, std::min<size_t>(most_blocks, 4096 / block_bytes));
    while (l.blocks > 1 && all < (long long)l.blocks * 4 * num_sms()) l.blocks--;
    const long long tiles = (all + l.blocks - 1) / l.blocks;
    l.warps = MIX_WARPS;
    // Two stages where three CTAs of an SM have room for them: what a warp waits for a tile is otherwise better hidden by other warps
    // (the gradients of 21 labels: 700 us with two stages and eight warps an SM, 602 with one and twelve).
    l.stages = tiles > (long long)l.warps * num_sms() ? most_stages : 1;
    if (l.stages == 2 && 3 * (smem(l.warps, 2, l.blocks) + 1024) > SMEM_SM) l.stages = 1;
    while (l.stages > 1 && smem(l.warps, l.stages, l.blocks) > SMEM_CTA) l.stages--;
    while (l.blocks > 1 && smem(l.warps, l.stages, l.blocks) > SMEM_CTA) l.blocks--;
    while (l.warps > 1 && smem(l.warps, l.stages, l.blocks) > SMEM_CTA) l.warps--;
    l.smem = smem(l.warps, l.stages, l.blocks);
    const int fit = (int)std::max<size_t>(1, SMEM_SM / (l.smem + 1024));
    const long long per_cta = (long long)block_rows * l.blocks * l.warps;
    l.ctas = (int)std::min<long long>((rows + per_cta - 1) / per_cta, (long long)num_sms() * std::min(most_ctas, fit));
    return l;
}

}  // namespace pl
