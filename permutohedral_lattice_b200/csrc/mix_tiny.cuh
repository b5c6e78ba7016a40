// The channel products with up to four channels of each input and of the output (two or three classes, a grey image): a thread
// a row, weights and sums in registers.  A row is some tens of bytes: bound by memory, and as matrix products of 8 x 8 blocks most of the
// work was on channels that are not there (volumes of two classes, 3.4 million rows, float: forward 93 -> 32 us, gradients 130 -> 44; their bytes
// take 17 and 29: the loops run over four channels whatever the number).  Two CTAs an SM are asked for, forward too: 35 us without.
#pragma once
#include "mix_backward.cuh"

namespace pl {

constexpr int TINY = 4, TINY_ROWS = 4, TINY_BACK_ROWS = 2;   // channels; rows that a thread has on their way at once, forward and backward

struct TinyWeights {
    float w[TINY][TINY], w2[TINY][TINY];
};
__device__ __forceinline__ void load_tiny_weights(TinyWeights& v, const void* weight, const void* weight2, int k, int k2, int n, int dtype) {
#pragma unroll
    for (int j = 0; j < TINY; j++)
#pragma unroll
        for (int c = 0; c < TINY; c++) {
            v.w[j][c] = weight && j < k && c < n ? load_weight(weight, j * n + c, dtype) : 0.f;
            v.w2[j][c] = weight2 && j < k2 && c < n ? load_weight(weight2, j * n + c, dtype) : 0.f;
        }
}
// V: channels of every operand's rows, 2 or 4, which then take one access each; 0: any number, an access a channel (behind the last
// one that one again: a weight of zero meets it).  Rows behind the last one are the last one again: nothing here branches, so that
// all loads are on their way together.
template <int V, typename T>
__device__ __forceinline__ void load_tiny_row(float (&v)[TINY], const T* rows, long long row, int channels) {
    if constexpr (V == 4) {
        load4(v, rows + 4 * row);
    } else if constexpr (V == 2) {
        v[2] = v[3] = 0.f;
        if constexpr (sizeof(T) == 4) {
            const float2 q = *reinterpret_cast<const float2*>(rows + 2 * row);
            v[0] = q.x, v[1] = q.y;
        } else {
            const u32 q = *reinterpret_cast<const u32*>(rows + 2 * row);
            v[0] = to_float(reinterpret_cast<const T*>(&q)[0]), v[1] = to_float(reinterpret_cast<const T*>(&q)[1]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < TINY; j++) v[j] = to_float(rows[row * channels + min(j, channels - 1)]);
    }
}
template <int V, typename T>
__device__ __forceinline__ void load_tiny_kept(float (&v)[TINY], const Kept& rows, long long row, int channels) {
    if (!rows.codes) {
        load_tiny_row<V>(v, static_cast<const T*>(rows.full), row, channels);
        return;
    }
#pragma unroll
    for (int j = 0; j < TINY; j++) {
        const long long i = row * channels + min(j, channels - 1);
        v[j] = decode_value(rows.codes[i], (u32)(u16)rows.scales[i / PACK_BLOCK]);
    }
}
template <int V, typename T>
__device__ __forceinline__ void store_tiny_row(T* rows, const float (&v)[TINY], long long row, int channels) {
    if constexpr (V == 4) {
        store4(rows + 4 * row, v);
    } else if constexpr (V == 2 && sizeof(T) == 4) {
        *reinterpret_cast<float2*>(rows + 2 * row) = make_float2(v[0], v[1]);
    } else if constexpr (V == 2) {
        u32 q;
        reinterpret_cast<T*>(&q)[0] = from_float<T>(v[0]), reinterpret_cast<T*>(&q)[1] = from_float<T>(v[1]);
        *reinterpret_cast<u32*>(rows + 2 * row) = q;
    } else {
#pragma unroll
        for (int j = 0; j < TINY; j++)
            if (j < channels) rows[row * channels + j] = from_float<T>(v[j]);
    }
}

template <typename T, int V>
__global__ void __launch_bounds__(256, 2) mix_tiny(MixArgs a) {
    __shared__ __align__(16) T pack_s[8][32 * TINY_ROWS * TINY];   // a warp's rows on their way to 8 bits
    const int k = a.k, k2 = a.k2, n = a.n, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    TinyWeights v;
    load_tiny_weights(v, a.weight, a.weight2, k, k2, n, a.weight_dtype);
    float bias[TINY];
#pragma unroll
    for (int c = 0; c < TINY; c++) bias[c] = a.bias && c < n ? load_weight(a.bias, c, a.weight_dtype) : 0.f;
    const T* residual = static_cast<const T*>(a.residual);
    const long long step = (long long)gridDim.x * 256 * TINY_ROWS;
    for (long long row0 = ((long long)blockIdx.x * 256 + warp * 32) * TINY_ROWS; row0 < a.rows; row0 += step) {
        float x[TINY_ROWS][TINY], x2[TINY_ROWS][TINY] = {}, r[TINY_ROWS][TINY] = {};
#pragma unroll
        for (int u = 0; u < TINY_ROWS; u++) {
            const long long row = min(row0 + 32 * u + lane, a.rows - 1);
            load_tiny_row<V>(x[u], static_cast<const T*>(a.x), row, k);
            if (k2) load_tiny_row<V>(x2[u], static_cast<const T*>(a.x2), row, k2);
            if (residual) load_tiny_row<V>(r[u], residual, row, n);
        }
#pragma unroll
        for (int u = 0; u < TINY_ROWS; u++) {
            float z[TINY];
            float top = -INFINITY, den = 0.f;
#pragma unroll
            for (int c = 0; c < TINY; c++) {
                z[c] = bias[c];
#pragma unroll
                for (int j = 0; j < TINY; j++) {
                    if (j < k) z[c] = fmaf(x[u][j], v.w[j][c], z[c]);
                    if (j < k2) z[c] = fmaf(x2[u][j], v.w2[j][c], z[c]);
                }
                if (residual) z[c] = fmaf(a.scale, r[u][c], z[c]);
                if (c >= n) z[c] = -INFINITY;
                top = fmaxf(top, z[c]);
            }
            if (a.activation == PL_ACT_SOFTMAX) {
                if (top == -INFINITY) top = 0.f;   // (see mix_activate)
#pragma unroll
                for (int c = 0; c < TINY; c++) {
                    z[c] = exp2_approx((z[c] - top) * 1.4426950408889634f);
                    den += z[c];
                }
                const float inv = den == 0.f ? 0.f : __fdividef(1.f, den);
#pragma unroll
                for (int c = 0; c < TINY; c++) z[c] *= inv;
            } else if (a.activation == PL_ACT_RELU) {
#pragma unroll
                for (int c = 0; c < TINY; c++) z[c] = z[c] < 0.f ? 0.f : z[c];
            }
            const long long row = row0 + 32 * u + lane;
            if (row < a.rows) store_tiny_row<V>(static_cast<T*>(a.out), z, row, n);
#pragma unroll
            for (int c = 0; c < TINY; c++) r[u][c] = z[c];   // (kept in 8 bits below)
        }
        auto keep = [&](const float (&values)[TINY_ROWS][TINY], int c, uint8_t* codes, int16_t* scales, bool nonzero) {
            const long long from = row0 * c;
            __syncwarp();
#pragma unroll
            for (int u = 0; u < TINY_ROWS; u++) store_tiny_row<0>(pack_s[warp], values[u], 32 * u + lane, c);
            __syncwarp();
            pack_by_warp(pack_s[warp], (int)min((long long)(32 * TINY_ROWS), a.rows - row0) * c, codes + from, scales + from / PACK_BLOCK, nonzero,
                         (reinterpret_cast<uintptr_t>(codes) & 3) == 0);
        };
        if (a.x_codes) keep(x, k, a.x_codes, a.x_scales, false);
        if (a.x2_codes) keep(x2, k2, a.x2_codes, a.x2_scales, false);
        if (a.out_codes) keep(r, n, a.out_codes, a.out_scales, a.activation == PL_ACT_RELU);
    }
}

template <typename T, int V>
__global__ void __launch_bounds__(256, 2) mix_tiny_backward(MixBackArgs a) {
    constexpr int SUMS = (2 * TINY + 1) * TINY;
    __shared__ float sums_s[8][SUMS];
    const int k = a.k, k2 = a.k2, n = a.n, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    TinyWeights v;
    load_tiny_weights(v, a.weight, a.weight2, k, k2, n, a.weight_dtype);
    float sums[2 * TINY + 1][TINY];   // dW, dW2, dbias
#pragma unroll
    for (int j = 0; j <= 2 * TINY; j++)
#pragma unroll
        for (int c = 0; c < TINY; c++) sums[j][c] = 0.f;
    const bool reads_y = a.activation != PL_ACT_NONE;
    const long long step = (long long)gridDim.x * 256 * TINY_BACK_ROWS;
    for (long long row0 = ((long long)blockIdx.x * 256 + warp * 32) * TINY_BACK_ROWS; row0 < a.rows; row0 += step) {
        float g[TINY_BACK_ROWS][TINY], y[TINY_BACK_ROWS][TINY] = {}, x[TINY_BACK_ROWS][TINY] = {}, x2[TINY_BACK_ROWS][TINY] = {};
#pragma unroll
        for (int u = 0; u < TINY_BACK_ROWS; u++) {
            const long long row = min(row0 + 32 * u + lane, a.rows - 1);
            load_tiny_row<V>(g[u], static_cast<const T*>(a.grad), row, n);
            if (reads_y) load_tiny_kept<V, T>(y[u], a.out, row, n);
            if (a.want_x) load_tiny_kept<V, T>(x[u], a.x, row, k);
            if (a.want_x2) load_tiny_kept<V, T>(x2[u], a.x2, row, k2);
        }
#pragma unroll
        for (int u = 0; u < TINY_BACK_ROWS; u++) {
            const long long row = row0 + 32 * u + lane;
            if (row >= a.rows) continue;
            float s = 0.f, dz[TINY], dr[TINY], dx[TINY], dx2[TINY];
#pragma unroll
            for (int c = 0; c < TINY; c++)
                if (c < n) s = fmaf(y[u][c], g[u][c], s);
            const bool empty = y[u][0] == 0.f && y[u][1] == 0.f && y[u][2] == 0.f && y[u][3] == 0.f;   // of a softmax: no gradient (see mix_backward)
#pragma unroll
            for (int c = 0; c < TINY; c++) {
                dz[c] = a.activation == PL_ACT_SOFTMAX ? (empty ? 0.f : y[u][c] * (g[u][c] - s)) : a.activation == PL_ACT_RELU ? relu_gradient(y[u][c], g[u][c]) : g[u][c];
                dr[c] = a.scale * dz[c];
                sums[2 * TINY][c] += dz[c];
            }
#pragma unroll
            for (int j = 0; j < TINY; j++) {
                dx[j] = dx2[j] = 0.f;
#pragma unroll
                for (int c = 0; c < TINY; c++)
                    if (c < n) {
                        dx[j] = fmaf(dz[c], v.w[j][c], dx[j]);
                        dx2[j] = fmaf(dz[c], v.w2[j][c], dx2[j]);
                        sums[j][c] = fmaf(x[u][j], dz[c], sums[j][c]);
                        sums[TINY + j][c] = fmaf(x2[u][j], dz[c], sums[TINY + j][c]);
                    }
            }
            if (a.dresidual) store_tiny_row<V>(static_cast<T*>(a.dresidual), dr, row, n);
            if (a.dx) store_tiny_row<V>(static_cast<T*>(a.dx), dx, row, k);
            if (a.dx2) store_tiny_row<V>(static_cast<T*>(a.dx2), dx2, row, k2);
        }
    }
    if (!a.shares) return;
#pragma unroll
    for (int j = 0; j <= 2 * TINY; j++)
#pragma unroll
        for (int c = 0; c < TINY; c++) {
            float w = sums[j][c];
#pragma unroll
            for (int o = 16; o; o >>= 1) w += __shfl_xor_sync(~0u, w, o);
            if (lane == 0) sums_s[warp][j * TINY + c] = w;
        }
    __syncthreads();
    const int count = (k + k2 + 1) * n, i = threadIdx.x;
    if (i >= count) return;
    const int r = i / n, c = i - r * n, from = (r < k ? r : r < k + k2 ? TINY + r - k : 2 * TINY) * TINY + c;
    float w = 0.f;
    for (int q = 0; q < 8; q++) w += sums_s[q][from];
    a.shares[(size_t)blockIdx.x * count + i] = w;
}

}  // namespace pl
