// The launches of the norms' kernels, for the translation units that compile them.
#pragma once
#include <algorithm>

#include "channel_norm.cuh"
#include "host_calls.h"

namespace pl {

int norm_of_floats(NormArgs& a, bool backward, int ctas, cudaStream_t st);
int norm_of_halves(NormArgs& a, int dtype, bool backward, int ctas, cudaStream_t st);

static bool norm_aligned(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

template <typename T, bool WIDE, int E>
static int launch_norm(NormArgs& a, bool backward, int ctas, cudaStream_t st) {
    const int pieces = (a.c + Piece<T, WIDE>::V - 1) / Piece<T, WIDE>::V, per_lane = E / Piece<T, WIDE>::V;
    a.lanes = 1;
    while (a.lanes * per_lane < pieces) a.lanes *= 2;
    const long long per_cta = (long long)NORM_WARPS * (32 / a.lanes), all = (a.rows + per_cta - 1) / per_cta;
    const unsigned grid = (unsigned)std::max(1ll, std::min(all, (long long)ctas));
    if (!backward) norm_forward<T, WIDE, E><<<grid, NORM_THREADS, 0, st>>>(a);
    else if (a.after && a.before) norm_backward<T, WIDE, E, true, true><<<grid, NORM_THREADS, 0, st>>>(a);
    else if (a.after) norm_backward<T, WIDE, E, true, false><<<grid, NORM_THREADS, 0, st>>>(a);
    else if (a.before) norm_backward<T, WIDE, E, false, true><<<grid, NORM_THREADS, 0, st>>>(a);
    else norm_backward<T, WIDE, E, false, false><<<grid, NORM_THREADS, 0, st>>>(a);
    PL_COUNT_LAUNCHES(1);
    PL_CUDA(cudaGetLastError());
    a.ctas = (int)grid;
    return PL_OK;
}

// a.ctas: how many ran, and left a share of the sums each.
template <typename T>
static int norm_of(NormArgs& a, bool backward, int ctas, cudaStream_t st) {
    constexpr int V = 16 / sizeof(T);
    bool wide = a.c % V == 0;
    for (const void* p : {a.x, a.residual, a.gate, (const void*)a.h, (const void*)a.y, a.dh, a.dy, (const void*)a.dx, (const void*)a.dresidual, (const void*)a.dgate})
        wide = wide && norm_aligned(p);
    if (wide) return a.c <= 256 ? launch_norm<T, true, 8>(a, backward, ctas, st) : launch_norm<T, true, 16>(a, backward, ctas, st);
    if (a.c <= 4) return launch_norm<T, false, 4>(a, backward, ctas, st);
    return a.c <= 256 ? launch_norm<T, false, 8>(a, backward, ctas, st) : launch_norm<T, false, 16>(a, backward, ctas, st);
}

}  // namespace pl
