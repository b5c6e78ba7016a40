// The launches of the norms' kernels, for the translation units that compile them.
#pragma once
#include <algorithm>

#include "channel_norm.cuh"
#include "host_calls.h"

namespace pl {

int norm_of_floats(NormArgs& a, bool backward, int ctas, cudaStream_t st);
int norm_of_halves(NormArgs& a, bool backward, int ctas, cudaStream_t st);
int norm_of_bfloats(NormArgs& a, bool backward, int ctas, cudaStream_t st);

static bool norm_aligned(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

template <typename T, bool WIDE, int E, int LANES>
static int launch_norm(NormArgs& a, bool backward, int ctas, cudaStream_t st) {
    const long long per_cta = (long long)NORM_WARPS * (32 / LANES), all = (a.rows + per_cta - 1) / per_cta;
    const unsigned grid = (unsigned)std::max(1ll, std::min(all, (long long)ctas));
    if (!backward && a.drop.threshold) norm_forward<T, WIDE, E, LANES, true><<<grid, NORM_THREADS, 0, st>>>(a);
    else if (!backward) norm_forward<T, WIDE, E, LANES, false><<<grid, NORM_THREADS, 0, st>>>(a);
    else if (a.after && a.before) norm_backward<T, WIDE, E, LANES, true, true><<<grid, NORM_THREADS, 0, st>>>(a);
    else if (a.after) norm_backward<T, WIDE, E, LANES, true, false><<<grid, NORM_THREADS, 0, st>>>(a);
    else if (a.before) norm_backward<T, WIDE, E, LANES, false, true><<<grid, NORM_THREADS, 0, st>>>(a);
    else norm_backward<T, WIDE, E, LANES, false, false><<<grid, NORM_THREADS, 0, st>>>(a);
    PL_COUNT_LAUNCHES(1);
    PL_CUDA(cudaGetLastError());
    a.ctas = (int)grid;
    return PL_OK;
}

template <typename T, bool WIDE, int E>
static int launch_norm_lanes(NormArgs& a, int lanes, bool backward, int ctas, cudaStream_t st) {
    if (lanes == 1) return launch_norm<T, WIDE, E, 1>(a, backward, ctas, st);
    if (lanes == 2) return launch_norm<T, WIDE, E, 2>(a, backward, ctas, st);
    if (lanes == 4) return launch_norm<T, WIDE, E, 4>(a, backward, ctas, st);
    if (lanes == 8) return launch_norm<T, WIDE, E, 8>(a, backward, ctas, st);
    if (lanes == 16) return launch_norm<T, WIDE, E, 16>(a, backward, ctas, st);
    return launch_norm<T, WIDE, E, 32>(a, backward, ctas, st);
}

// a.ctas: how many ran, and left a share of the sums each.  Up to 8 values a lane with as few lanes a row as that takes (16 where
// it is all lanes).  Single values: 6 where those do, as much again backward otherwise (3 380 000 rows of 21 floats, gate of every value, two norms: 247 us forward and 568 backward, 275 and
// 1162 with 8; bfloat16 217 and 590, 270 and 1302).
template <typename T>
static int norm_of(NormArgs& a, bool backward, int ctas, cudaStream_t st) {
    constexpr int V = 16 / sizeof(T);
    bool wide = a.c % V == 0;
    for (const void* p : {a.x, a.residual, a.gate, (const void*)a.h, (const void*)a.y, a.dh, a.dy, (const void*)a.dx, (const void*)a.dresidual, (const void*)a.dgate})
        wide = wide && norm_aligned(p);
    int lanes = 1;
    while (lanes < 32 && lanes * 8 < a.c) lanes *= 2;
    if (a.c > 256) return wide ? launch_norm<T, true, 16, 32>(a, backward, ctas, st) : launch_norm<T, false, 16, 32>(a, backward, ctas, st);
    if (wide) return launch_norm_lanes<T, true, 8>(a, lanes, backward, ctas, st);
    return a.c <= 6 * lanes ? launch_norm_lanes<T, false, 6>(a, lanes, backward, ctas, st) : launch_norm_lanes<T, false, 8>(a, lanes, backward, ctas, st);
}

}  // namespace pl
