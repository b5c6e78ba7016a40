// The launches of the gated block's kernels, for the translation units that compile them.
#pragma once
#include <algorithm>

#include "gated.cuh"
#include "host_calls.h"

namespace pl {

int gated_floats(GatedArgs p, GatedPass pass, cudaStream_t st);
int gated_halves(GatedArgs p, int dtype, GatedPass pass, cudaStream_t st);

constexpr size_t GATED_SMEM = 227 * 1024;   // of a CTA, at most

// CTAs of a chunk of hidden channels when the weights' gradients are summed up.
inline int gated_splits(int chunks, long long rows, int sms) { return (int)std::max(1ll, std::min<long long>(std::max(1, sms / chunks), (rows + 127) / 128)); }

// Buffers, as far as there is room: the weights of all chunks where they fit (else they come anew for every tile), of everything else two, so
// that what comes next is fetched while products run.
template <typename T, GatedPass PASS, int ROWS>
static bool gated_plan(GatedArgs& p) {
    const int chunks = PASS == GATED_DW ? 1 : p.chunks;
    auto fits = [&](int w) {
        for (int left : {0, 1, 2, 3}) {
            p.w_buffers = w, p.x_buffers = left & 2 ? 1 : 2, p.a_buffers = left & 1 ? 1 : 2;
            if (PASS == GATED_DW && p.a_buffers == 2) continue;   // (its second products take as long as its first: nothing waits for them)
            if (GatedSmem<T, PASS, ROWS>(p).total <= (int)GATED_SMEM) return true;
        }
        return false;
    };
    if (!fits(chunks) && !fits(std::min(2, chunks)) && !fits(1)) return false;
    auto columns = [&](int s, int d) {
        p.s_buffers = s, p.d_buffers = d;
        return GatedColumns<T, PASS>(p).total <= 512;
    };
    return (PASS != GATED_DW && columns(2, 2)) || columns(2, 1) || columns(1, 1);
}

template <typename T, GatedPass PASS, int ROWS>
static int launch_gated_rows(GatedArgs& p, cudaStream_t st) {
    const int smem = GatedSmem<T, PASS, ROWS>(p).total;
    const long long tiles = (p.rows + ROWS - 1) / ROWS;
    const unsigned grid = PASS == GATED_DW ? p.chunks * p.splits : (unsigned)std::min<long long>(tiles, num_sms());
    PL_TRY((ensure_dynamic_smem<gated_kernel<T, PASS, ROWS>>(smem)));
    gated_kernel<T, PASS, ROWS><<<grid, GATED_THREADS, smem, st>>>(p);
    PL_COUNT_LAUNCHES(1);
    PL_CUDA(cudaGetLastError());
    return PL_OK;
}
template <typename T, GatedPass PASS>
static int launch_gated(GatedArgs& p, cudaStream_t st) {
    if (gated_plan<T, PASS, 128>(p)) return launch_gated_rows<T, PASS, 128>(p, st);
    if constexpr (sizeof(T) == 4)   // three terms of everything, from some 90 channels on: tiles of half as many rows, the other half of a product idle
        if (gated_plan<T, PASS, 64>(p)) return launch_gated_rows<T, PASS, 64>(p, st);
    return PL_INTERNAL_ERROR;
}
template <typename T>
static int gated_of(GatedArgs& p, GatedPass pass, cudaStream_t st) {
    p.chunks = (p.h + gated_chunk<T>() - 1) / gated_chunk<T>();
    p.splits = gated_splits(p.chunks, p.rows, num_sms());
    p.drain = sizeof(T) == 4 ? 2 : 64;
    return pass == GATED_OUT ? launch_gated<T, GATED_OUT>(p, st) : pass == GATED_DX ? launch_gated<T, GATED_DX>(p, st) : launch_gated<T, GATED_DW>(p, st);
}

}  // namespace pl
