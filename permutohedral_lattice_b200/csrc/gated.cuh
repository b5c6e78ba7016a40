// The gated feed-forward block of rows of points, and its gradients:
//
//   g = x Wg + bg,  u = x Wu + bu,  a = act(g) u,  out = a Wd + bd + s residual
//   da = dout Wd^T,  dg = da u act'(g),  du = da act(g),  dx = dg Wg^T + du Wu^T
//   dWg = x^T dg,  dWu = x^T du,  dWd = a^T dout,  dbg, dbu, dbd: sums over rows of dg, du, dout
//
// The hidden values (g, u, a and their gradients) never leave the SM: a CTA takes a tile of rows through the hidden channels a chunk
// at a time.  A chunk's g and u (and da) are products in tensor memory, its a (dg, du) go to shared memory as the next products' operand.
// The biases of g and u are a row more of the weights beside a column of ones.  The backward pass makes g and u again, in two
// kernels: gated_kernel<DX> sums dx over the chunks of a tile as the forward pass does out, gated_kernel<DW> sums the weights' gradients
// over the tiles of a chunk, a chunk a CTA, and adds them to a share of its own in the workspace now and then (`drain`, see
// gated_launch.cuh); gated_sums adds up the shares in order.  gated_pack first lays out the weights as the products read them.
//
// Warps: workers turn the first products into the second's operand, and take out the sums, one half of them every other step, so that one half
// computes while the other waits, loads or stores; two warps ask for the first and the second
// products, and for the weights that only theirs read; loaders fetch rows.  They meet at barriers in shared memory; every wait is bounded.
// If one runs out (two seconds: it should not happen), all give up and what the CTA was to write is NaN, which nothing else reports.
//
// Tiles of 128 rows, the rows of a product; chunks of 64 hidden channels (floats: 32), so that g and u of two chunks and the sums fit into tensor memory and
// the weights of all chunks, mostly, into shared memory.  2 097 152 rows of 64 to 256 to 64 bfloat16 channels: 528 us (390 TFLOP/s, 1.5 TB/s), gradients of
// rows 1001, of weights 1349; 154 401 of 128 to 512 to 128 float16 152, 330, 395 (400 TFLOP/s forward); a million of 32 to 128 to 32 floats 277, 650, 1521.  The tensor
// pipe is busy 17 to 24 % of it, memory less: what bounds them are the workers' instructions (40 to 58 % of the issue slots), half of these at barriers.
#pragma once
#include <cuda.h>
#include "gated_give_up.h"
#include "gated_tensor.cuh"

namespace pl {

constexpr int GATED_HIDDEN = 512;   // channels in between, at most
enum GatedPass { GATED_OUT, GATED_DX, GATED_DW };
// Warps: 20 leave 96 registers a thread, 16 leave 128.  Floats, whose products are six, need fewer workers, and more loaders: three terms of every value.
template <typename T>
struct GatedWarps {
    static constexpr int WORKERS = sizeof(T) == 4 ? 8 : 16, LOADERS = sizeof(T) == 4 ? 6 : 2, THREADS = 32 * (WORKERS + 2 + LOADERS);
};

struct GatedArgs {
    long long rows;
    int k, h, n, activation, round_hidden;
    int kx, kp, np;                  // columns of a tile of x, with the ones (if there are biases of g or u), and of out
    int chunks, splits;              // of the hidden channels; CTAs of a chunk (DW)
    int x_buffers, w_buffers[2], a_buffers, s_buffers, d_buffers, io_buffers, drain;
    float scale;
    const void *x, *gate_weight, *up_weight, *down_weight, *gate_bias, *up_bias, *down_bias, *residual, *grad;
    int biased, wide_x, wide_grad, wide_out;          // wide: rows of whole 16 bytes on 16-byte boundaries
    int box_x, box_grad;                              // rows that the TMA brings: wide ones of 16-bit values
    int wide_dresidual, down_bias_wanted;             // (DX: dout and dresidual begin on 16-byte boundaries; DW)
    int split;                       // (OUT, DX, floats) the sums of every other chunk apart: over more than 256 hidden channels too much would be cut
    int stacked;                     // (DW, floats) the terms of a product's second operand side by side: a sum for every order of magnitude
    const u32* peaks;                // (float16 gradients) the largest |dout| of its parts, see gated_peak
    int peak_count;
    unsigned char* packed;           // the weights, a chunk after another: Wd, Wg and Wu as tiles
    void *out, *dresidual;           // out: or dx
    float* shares;                   // [chunks][splits][columns of sums][128]
};

// float16: dg and du hold nothing below 2^-25, and a mean's gradients over a million points are 1e-6.  Where the largest |dout| of a call is below 2^-6, they are made of
// dout times the power of two that takes it there, and what is summed up of them is divided by that on its way out.  (2^-6: some 2^19 below that
// they hold, and 2^22 above it.)  What is not finite counts for nothing, so that it does not change other rows.  A pass over dout, and one more launch: a training
// step of 154 401 rows of 128 to 512 to 128 takes 925 us with it, 900 without.
constexpr int GATED_PEAK_EXPONENT = -6;
static __global__ void __launch_bounds__(256) gated_peak(const __half* grad, long long count, u32* peaks) {
    __shared__ u32 peak_s[8];
    u32 peak = 0;   // of even and of odd values
    auto take = [&](u32 v) {
        v &= 0x7FFF7FFFu;
        peak = __vmaxu2(peak, v & __vcmpltu2(v, 0x7C007C00u));
    };
    const unsigned short* values = reinterpret_cast<const unsigned short*>(grad);
    const long long head = min(count, (long long)((16 - reinterpret_cast<uintptr_t>(grad) % 16) % 16 / 2)), pieces = (count - head) / 8;
    const uint4* whole = reinterpret_cast<const uint4*>(values + head);
    const long long thread = (long long)blockIdx.x * 256 + threadIdx.x, threads = (long long)gridDim.x * 256;
#pragma unroll 4
    for (long long i = thread; i < pieces; i += threads) {
        const uint4 q = whole[i];
        take(q.x), take(q.y), take(q.z), take(q.w);
    }
    if (thread < head) take(values[thread]);
    if (thread < count - head - 8 * pieces) take(values[head + 8 * pieces + thread]);
    peak = __reduce_max_sync(~0u, max(peak & 0xFFFFu, peak >> 16));
    if ((threadIdx.x & 31) == 0) peak_s[threadIdx.x >> 5] = peak;
    __syncthreads();
    if (threadIdx.x) return;
    for (int w = 1; w < 8; w++) peak = max(peak, peak_s[w]);
    peaks[blockIdx.x] = peak;
}
// The exponent of that power of two; peak: of a float16 number.
__device__ __forceinline__ int gated_scale_exponent(u32 peak) {
    if (peak == 0) return 0;
    const u32 bits = __float_as_uint(__half2float(__ushort_as_half((unsigned short)peak)));
    return max(0, GATED_PEAK_EXPONENT + 127 - (int)(bits >> 23));
}

struct GatedMaps {   // of x, dout, the residual and out (or dx) as matrices, where they go by the TMA
    CUtensorMap x, grad, residual, out;
};

template <typename T>
__host__ __device__ constexpr int gated_chunk() { return sizeof(T) == 4 ? 32 : 64; }   // hidden channels
// Bytes of a chunk's Wd, and of its Wg and Wu (side by side in one tile).
template <typename T>
__host__ __device__ inline int gated_down_bytes(int np) { return Tensor<T>::TERMS * tile_bytes(gated_chunk<T>(), np); }
template <typename T>
__host__ __device__ inline int gated_up_bytes(int kp) { return Tensor<T>::TERMS * tile_bytes(kp, 2 * gated_chunk<T>()); }

// Terms of a hidden value on its way to the second products.  FINE: 16-bit types take two, and results are off by their own rounding alone.  Else (who
// calls says so) it is rounded once more, which makes results 1.4 times as far off (sums of a few values up to 1.7).  Two million rows of 64 to 256 to
// 64 bfloat16 channels, forward, gradients of rows, of weights: 528, 1001, 1349 us with two terms, 461, 708, 715 with one.
template <typename T, bool FINE>
__host__ __device__ constexpr int hidden_terms() { return sizeof(T) == 4 ? 3 : FINE ? 2 : 1; }

// Where things lie in shared memory: offsets, bytes of a buffer, in all.
template <typename T, GatedPass PASS, int ROWS, bool FINE>
struct GatedSmem {
    static constexpr int C = gated_chunk<T>(), TERMS = Tensor<T>::TERMS, HIDDEN = hidden_terms<T, FINE>();
    static constexpr int A = HIDDEN * tile_bytes(ROWS, PASS == GATED_OUT ? C : 2 * C), ACT = PASS == GATED_DW ? HIDDEN * tile_bytes(ROWS, C) : 0;
    static constexpr int BARRIERS = 2048;
    __host__ __device__ static int rows_bytes(int columns) { return TERMS == 1 ? swizzled_bytes(ROWS, 2 * columns) : TERMS * tile_bytes(ROWS, columns); }
    int grad, x, io;                 // bytes: a tile of dout, of x with it, of rows on their way out
    int w[2];                        // of the weights that the first products alone read (OUT: Wg and Wu, DX and DW: Wd), and of the others
    int at_x, at_w[2], at_a, at_io, at_ones, total;
    __host__ __device__ GatedSmem(const GatedArgs& p) {
        grad = PASS == GATED_OUT ? 0 : rows_bytes(p.np);
        x = grad + rows_bytes(p.kx);
        const int down = gated_down_bytes<T>(p.np), up = gated_up_bytes<T>(p.kp);
        w[0] = PASS == GATED_OUT ? up : down, w[1] = PASS == GATED_OUT ? down : up;
        io = swizzled_bytes(ROWS, (PASS == GATED_OUT ? p.n : p.k) * (int)sizeof(T));
        at_x = BARRIERS;
        at_io = at_x + p.x_buffers * x;
        at_io = (at_io + 1023) / 1024 * 1024;
        at_w[0] = at_io + p.io_buffers * io;
        at_w[1] = at_w[0] + p.w_buffers[0] * w[0];
        at_a = at_w[1] + p.w_buffers[1] * w[1];
        at_ones = at_a + p.a_buffers * (A + ACT);
        // (products of 128 rows read on behind a tile of 64, and of 128 columns behind one of fewer: what they make of it nobody takes)
        total = at_ones + (p.biased || p.down_bias_wanted ? tile_bytes(ROWS, 16) : 0) + (ROWS < 128 ? 1024 : 0);
    }
};
// Columns of tensor memory: of g and u (and da), and of the sums.  Those of DW are, in this order, of dWg and dWu, dbg and dbu, dWd, and dbd.
template <typename T, GatedPass PASS>
struct GatedColumns {
    static constexpr int C = gated_chunk<T>(), WIDE = PASS == GATED_OUT ? 2 * C : 3 * C, SUMS = Tensor<T>::TERMS == 3 ? 2 : 1;
    int d, d_one, d_all, total;         // from there on; of the values, of all their parts
    int up_bias, down, down_bias;       // (DW) where those sums begin
    int up_part, down_part, bias_part;  // from one part of a value (float32: of its products' small terms, by size) to the next
    __host__ __device__ GatedColumns(const GatedArgs& p) {
        d = p.s_buffers * WIDE;
        d_one = PASS == GATED_DW ? p.kp + C + (p.down_bias_wanted ? 16 : 0) : PASS == GATED_OUT ? p.np : p.kx;
        d_all = SUMS * d_one;
        up_bias = p.kx, down = p.kp, down_bias = p.kp + C;
        up_part = down_part = bias_part = SUMS == 2 ? d_one : 0;
        if (p.split) d_all = 3 * d_one;
        if (p.stacked) {
            const int biases = p.kp - p.kx + (p.down_bias_wanted ? 16 : 0);
            down = 3 * p.kx, up_bias = down + 3 * C, down_bias = up_bias + p.kp - p.kx;
            up_part = p.kx, down_part = C, bias_part = biases;
            d_all = up_bias + 2 * biases;
        }
        total = d + p.d_buffers * d_all;
    }
    // Where value c's first part is, how far the next, and how many.
    __device__ __forceinline__ int place(const GatedArgs& p, int c, int& part, int& parts) const {
        part = up_part, parts = p.stacked || p.split ? 3 : SUMS;
        if (PASS != GATED_DW || c < p.kx) return c;
        if (c >= p.kp && c < p.kp + C) {
            part = down_part;
            return down + c - p.kp;
        }
        part = bias_part, parts = SUMS;
        return c < p.kp ? up_bias + c - p.kx : down_bias + c - p.kp - C;
    }
};

// Eight sigmoids of g and (REST) what is left to one.  16-bit types: by e = exp(-|g|), at most one, of which 1 / (1 + e) and e / (1 + e) are the two, whichever way
// round, so that neither loses its bits where a gate is shut or open.  A quarter of the reciprocals, the other three by products, which stay below 16: the
// exponentials and reciprocals of all, two an element, took longer than their other instructions.  Floats, whose products take longer, do without.
template <typename T, bool REST>
__device__ __forceinline__ void gated_sigmoids(const float2 (&g)[4], float2 (&s)[4], float2 (&rest)[4]) {
    const float2 one = make_float2(1.f, 1.f);
    if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
            float2 e[2], d[2];
#pragma unroll
            for (int j = 0; j < 2; j++) {
                e[j] = make_float2(exp2_approx(-1.4426950408889634f * fabsf(g[i + j].x)), exp2_approx(-1.4426950408889634f * fabsf(g[i + j].y)));
                d[j] = add2(e[j], one);
            }
            const float2 pairs = mul2(d[0], d[1]);                     // x, y: of two each
            float all;
            asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(all) : "f"(pairs.x * pairs.y));
            const float2 of_pairs = mul2(make_float2(all, all), make_float2(pairs.y, pairs.x));
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const float2 large = mul2(of_pairs, d[1 - j]), small = mul2(large, e[j]);
                const bool x = g[i + j].x < 0.f, y = g[i + j].y < 0.f;
                s[i + j] = make_float2(x ? small.x : large.x, y ? small.y : large.y);
                if constexpr (REST) rest[i + j] = make_float2(x ? large.x : small.x, y ? large.y : small.y);
            }
        }
    } else {
        const float2 minus = make_float2(-1.4426950408889634f, -1.4426950408889634f);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 q = mul2(g[i], minus), d = add2(make_float2(exp2_approx(q.x), exp2_approx(q.y)), one);
            s[i] = make_float2(__fdividef(1.f, d.x), __fdividef(1.f, d.y));
            if constexpr (REST) rest[i] = fma2(s[i], make_float2(-1.f, -1.f), one);
        }
    }
}
// act(g) of eight values; SLOPE: act'(g) too
template <typename T, int ACT, bool SLOPE>
__device__ __forceinline__ void gated_act(const float2 (&g)[4], float2 (&act)[4], float2 (&slope)[4]) {
    const float2 one = make_float2(1.f, 1.f), minus = make_float2(-1.f, -1.f);
    if constexpr (ACT == PL_GATE_SILU || ACT == PL_GATE_SIGMOID) {
        float2 s[4], rest[4];
        gated_sigmoids<T, SLOPE && ACT == PL_GATE_SIGMOID>(g, s, rest);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            act[i] = ACT == PL_GATE_SILU ? mul2(g[i], s[i]) : s[i];
            if constexpr (SLOPE && ACT == PL_GATE_SILU) slope[i] = fma2(act[i], fma2(s[i], minus, one), s[i]);   // s (1 + g (1 - s)): of 1 - s nothing small is wanted
            if constexpr (SLOPE && ACT == PL_GATE_SIGMOID) slope[i] = mul2(s[i], rest[i]);
        }
    } else if constexpr (ACT == PL_GATE_GELU) {
        // g Phi(g).  With t = 1 / (1 + p |g|) and e = exp(-g^2 / 2), which the slope takes anyway, the smaller of Phi and 1 - Phi is e times a polynomial of t,
        // fitted to erfcx(|g| / sqrt 2) / 2 for the least relative error, which holds however small Phi is.  Floats: nine terms, 0.6 2^-24 off and evaluated
        // 6 2^-24 (erfcf's registers took 5 % of every activation's time).  16-bit types: six, 2^-18 (erff took as long as all the rest).
        auto both = [](float v) { return make_float2(v, v); };
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 q = mul2(mul2(g[i], g[i]), both(-0.72134752044448170f));
            const float2 e = make_float2(exp2_approx(q.x), exp2_approx(q.y));
            const float2 d = fma2(make_float2(fabsf(g[i].x), fabsf(g[i].y)), both(sizeof(T) == 4 ? 0.35f : 0.30816703f), one);
            const float2 t = make_float2(__fdividef(1.f, d.x), __fdividef(1.f, d.y));
            float2 p;
            if constexpr (sizeof(T) == 4) {
                p = fma2(t, both(-0.02914591133594513f), both(0.14397162199020386f));
                p = fma2(t, p, both(-0.25571408867836f));
                p = fma2(t, p, both(0.15917399525642395f));
                p = fma2(t, p, both(-0.02310972847044468f));
                p = fma2(t, p, both(0.10550796240568161f));
                p = fma2(t, p, both(0.11983287334442139f));
                p = fma2(t, p, both(0.13986186683177948f));
                p = fma2(t, p, both(0.13962140679359436f));
            } else {
                p = fma2(t, both(-0.07539591193199158f), both(0.1891007274389267f));
                p = fma2(t, p, both(0.00772145064547658f));
                p = fma2(t, p, both(0.1364033967256546f));
                p = fma2(t, p, both(0.11898145079612732f));
                p = fma2(t, p, both(0.12318693846464157f));
            }
            p = mul2(mul2(p, t), e);
            const float2 rest = fma2(p, minus, one);
            const float2 cdf = make_float2(g[i].x < 0.f ? p.x : rest.x, g[i].y < 0.f ? p.y : rest.y);
            act[i] = mul2(g[i], cdf);
            if constexpr (SLOPE) slope[i] = fma2(mul2(g[i], both(0.3989422804014327f)), e, cdf);
        }
    } else {
        auto relu = [](float v) { return v < 0.f ? 0.f : v; };
        auto step = [](float v) { return v > 0.f ? 1.f : v <= 0.f ? 0.f : v; };   // (NaN: itself)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            act[i] = make_float2(relu(g[i].x), relu(g[i].y));
            if constexpr (SLOPE) slope[i] = make_float2(step(g[i].x), step(g[i].y));
        }
    }
}

template <typename T>
struct Piece16 {   // 16 bytes of values
    static constexpr int V = 16 / sizeof(T);
    __device__ __forceinline__ static void store(void* to, const float* v) {
        uint4 q;
        T* e = reinterpret_cast<T*>(&q);
#pragma unroll
        for (int i = 0; i < V; i++) e[i] = from_float<T>(v[i]);
        *static_cast<uint4*>(to) = q;
    }
    __device__ __forceinline__ static void load(float* v, const void* from) {
        const uint4 q = *static_cast<const uint4*>(from);
        const T* e = reinterpret_cast<const T*>(&q);
#pragma unroll
        for (int i = 0; i < V; i++) v[i] = to_float(e[i]);
    }
};
// Rows of `width` values to a tile of `blocks` blocks of columns by some warps: `valid` rows, zeros behind and beside.  wide: read by 16 bytes (floats;
// wide 16-bit rows come by the TMA).  Eight rows of four blocks a warp at a time: whole sectors of memory, all banks of shared memory.  (16-bit values
// by words of 4 bytes, shifted where rows begin between them, took half as long again as one by one.)
template <typename T, int ROWS>
__device__ __forceinline__ void stage(unsigned char* to, int blocks, const T* src, int width, int valid, bool wide, int warp, int warps) {
    const int lane = threadIdx.x & 31, r8 = lane & 7, b0 = lane >> 3, plane = tile_bytes(ROWS, 8 * blocks);
    for (int b = b0; b < (blocks + 3) / 4 * 4; b += 4) {
        constexpr int U = 4;
        for (int g0 = warp; g0 < ROWS / 8; g0 += U * warps) {
            float v[U][8];
#pragma unroll
            for (int i = 0; i < U; i++) {
                const int r = 8 * (g0 + i * warps) + r8;
                const T* from = src + (long long)r * width + 8 * b;
                const bool there = r < valid && r < ROWS && 8 * b < width;
                if (sizeof(T) == 4 && wide) {
                    float q[4] = {0.f, 0.f, 0.f, 0.f};
                    if (there) load4(q, from);
#pragma unroll
                    for (int e = 0; e < 4; e++) v[i][e] = q[e], q[e] = 0.f;
                    if (there) load4(q, from + 4);
#pragma unroll
                    for (int e = 0; e < 4; e++) v[i][4 + e] = q[e];
                } else {
#pragma unroll
                    for (int e = 0; e < 8; e++) v[i][e] = there && 8 * b + e < width ? to_float(from[e]) : 0.f;
                }
            }
#pragma unroll
            for (int i = 0; i < U; i++) {
                const int r = 8 * (g0 + i * warps) + r8;
                if (r < ROWS && b < blocks) store_terms8<T>(to + (sizeof(T) == 2 ? swizzled_at(ROWS, r, b) : b * column_blocks(ROWS) + 16 * r), plane, v[i]);
            }
        }
    }
}

// The weights of all chunks as the products' operands, terms made: a row's eight columns a thread.
template <typename T>
__global__ void __launch_bounds__(256) gated_pack(const __grid_constant__ GatedArgs p) {
    constexpr int C = gated_chunk<T>();
    const int down_items = C * (p.np / 8), up_items = p.kp * (2 * C / 8), items = down_items + up_items;
    const int down_bytes = gated_down_bytes<T>(p.np), up_bytes = gated_up_bytes<T>(p.kp);
    const int chunk = blockIdx.y, h0 = chunk * C;
    unsigned char* to = p.packed + (long long)chunk * (down_bytes + up_bytes);
    const int i = blockIdx.x * 256 + threadIdx.x;
    if (i >= items) return;
    const bool down = i < down_items;
    const int blocks = down ? p.np / 8 : 2 * C / 8, j = down ? i : i - down_items, r = j / blocks, b = j - r * blocks;
    const bool up = !down && b >= C / 8;
    const int c0 = down ? 8 * b : h0 + 8 * (up ? b - C / 8 : b), width = down ? p.n : p.h, row = down ? h0 + r : r, rows = down ? p.h : p.k;
    const T* from = static_cast<const T*>(down ? p.down_weight : up ? p.up_weight : p.gate_weight) + (long long)row * width + c0;
    bool there = row < rows;
    if (!down && row == p.kx) {   // the biases' row
        const T* bias = static_cast<const T*>(up ? p.up_bias : p.gate_bias);
        there = p.biased && bias;
        from = bias + c0;
    }
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = there && c0 + e < width ? to_float(from[e]) : 0.f;
    const int tile_rows = down ? C : p.kp;
    store_terms8<T>(to + (down ? 0 : down_bytes) + b * column_blocks(tile_rows) + 16 * r, tile_bytes(tile_rows, 8 * blocks), v);
}

struct GatedBarriers {
    u64 x_full[4], x_free[4], w_full[2][16], w_free[2][16], s_full[2], s_free[2], a_full[2], a_free[2], d_full[2], d_free[2], io_full[2], io_done[2], end[2];
    u32 tensor, dead;
};
static_assert(sizeof(GatedBarriers) <= 1024);
__device__ __forceinline__ bool b_dead(const GatedBarriers& b) { return *static_cast<const volatile u32*>(&b.dead) != 0; }

// Where one of a ring of buffers is in its turns.
struct Turn {
    int at = 0, turns = 0;
    __device__ __forceinline__ void next(int buffers) {
        if (++at == buffers) at = 0, turns++;
    }
};
struct Waits {
    volatile u32* dead;
    bool alive = true;
    // Gives up two seconds after it began, or (unless it is `last`) when others have.
    __device__ __forceinline__ bool on(u64* bar, int parity, bool last = false) {
        if (!alive || mbar_done(bar, parity & 1)) return alive;
        const u64 began = global_timer();
        for (int i = 1; !mbar_done(bar, parity & 1); i++)
            if ((*dead && !last) || i >= 1 << 26 || ((i & 63) == 0 && global_timer() - began > 2000000000ull)) {
                *dead = 1;
                return alive = false;
            }
        return true;
    }
    // Barriers of even and of odd steps: one half of the workers meets one of them, and sees each of its phases.
    __device__ __forceinline__ bool step(u64* bars, long long q) { return on(bars + (q & 1), (int)(q >> 1)); }
    __device__ __forceinline__ bool full(u64* bars, const Turn& t) { return on(bars + t.at, t.turns); }
    __device__ __forceinline__ bool free(u64* bars, const Turn& t) { return t.turns == 0 ? alive : on(bars + t.at, t.turns - 1); }
};

template <typename T>
__device__ __forceinline__ void store16(T* to, const float (&v)[16], int left, bool wide) {
    constexpr int V = 16 / sizeof(T);
    if (wide) {
#pragma unroll
        for (int j = 0; j < 16; j += V)
            if (j < left) {
                float q[4] = {v[j], v[j + 1], v[j + 2], v[j + 3]};
                if constexpr (V == 4) {
                    store4(to + j, q);
                } else {
                    uint4 p;
                    T* e = reinterpret_cast<T*>(&p);
#pragma unroll
                    for (int i = 0; i < 8; i++) e[i] = from_float<T>(v[j + i]);
                    *reinterpret_cast<uint4*>(to + j) = p;
                }
            }
    } else {
#pragma unroll
        for (int j = 0; j < 16; j++)
            if (j < left) to[j] = from_float<T>(v[j]);
    }
}
template <typename T>
__device__ __forceinline__ void load16(float (&v)[16], const T* from, int left, bool wide) {
    constexpr int V = 16 / sizeof(T);
    if (wide) {
#pragma unroll
        for (int j = 0; j < 16; j += 4) {
            float q[4] = {0.f, 0.f, 0.f, 0.f};
            if (j < left) load4(q, from + j);      // (left is a multiple of V)
#pragma unroll
            for (int e = 0; e < 4; e++) v[j + e] = q[e];
        }
    } else {
#pragma unroll
        for (int j = 0; j < 16; j++) v[j] = j < left ? to_float(from[j]) : 0.f;
    }
    static_assert(V >= 4);
}

// 16 columns of a row on its way in or out; pieces of 16 bytes behind the last column are not touched.
template <typename T, int ROWS>
__device__ __forceinline__ void io_store16(unsigned char* io, int row, int c, const float (&v)[16], int width) {
    constexpr int V = 16 / sizeof(T);
#pragma unroll
    for (int j = 0; j < 16; j += V)
        if (c + j < width) Piece16<T>::store(io + swizzled_at(ROWS, row, (c + j) / V), v + j);
}
template <typename T, int ROWS>
__device__ __forceinline__ void io_load16(float (&v)[16], const unsigned char* io, int row, int c, int width) {
    constexpr int V = 16 / sizeof(T);
#pragma unroll
    for (int j = 0; j < 16; j += V) {
        if (c + j < width) Piece16<T>::load(v + j, io + swizzled_at(ROWS, row, (c + j) / V));
        else
#pragma unroll
            for (int e = 0; e < V; e++) v[j + e] = 0.f;
    }
}
// to = s times the rows of a tile of 16-bit values (swizzled), by a warp.
template <typename T, int ROWS, typename = typename std::enable_if<sizeof(T) == 2>::type>
__device__ __forceinline__ void scale_tile(T* to, const unsigned char* tile, int rows, int pieces, float s) {
    const int lane = threadIdx.x & 31, count = rows * pieces, per = (65536 + pieces - 1) / pieces;   // (i per >> 16 is i / pieces for i < 2048)
#pragma unroll 4
    for (int i = lane; i < count; i += 32) {
        const int r = i * per >> 16;
        float v[8];
        Piece16<T>::load(v, tile + swizzled_at(ROWS, r, i - r * pieces));
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] *= s;
        Piece16<T>::store(to + 8 * i, v);
    }
}
// to = s from, `count` values, by a warp.  aligned: both begin on 16-byte boundaries, which tiles of contiguous rows do wherever the first one does.
template <typename T>
__device__ __forceinline__ void scale_rows(T* to, const T* from, int count, float s, bool aligned) {
    constexpr int V = 16 / sizeof(T), U = 8;
    const int lane = threadIdx.x & 31, whole = aligned ? count / V * V : 0;
    for (int i0 = V * lane; i0 < whole; i0 += 32 * V * U) {
        uint4 q[U];
#pragma unroll
        for (int u = 0; u < U; u++)
            if (i0 + 32 * V * u < whole) q[u] = *reinterpret_cast<const uint4*>(from + i0 + 32 * V * u);
#pragma unroll
        for (int u = 0; u < U; u++)
            if (i0 + 32 * V * u < whole) {
                T* e = reinterpret_cast<T*>(&q[u]);
#pragma unroll
                for (int i = 0; i < V; i++) e[i] = from_float<T>(s * to_float(e[i]));
                *reinterpret_cast<uint4*>(to + i0 + 32 * V * u) = q[u];
            }
    }
#pragma unroll 8
    for (int i = whole + lane; i < count; i += 32) to[i] = from_float<T>(s * to_float(from[i]));
}

// Some hidden channels of a row: from g, u (and da, times scale) to what the second products take.
template <typename T, GatedPass PASS, int ACT, int ROWS, int HIDDEN, int W>
__device__ __forceinline__ void gated_work(const float (&g)[W], const float (&u)[W], const float (&da)[W], float scale, unsigned char* a, int row, int column) {
    constexpr int C = gated_chunk<T>(), CB = column_blocks(ROWS), PLANE = tile_bytes(ROWS, PASS == GATED_OUT ? C : 2 * C);
#pragma unroll
    for (int j = 0; j < W; j += 8) {
        float2 g2[4], u2[4], d2[4], act[4], slope[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            g2[i] = make_float2(g[j + 2 * i], g[j + 2 * i + 1]);
            u2[i] = make_float2(u[j + 2 * i], u[j + 2 * i + 1]);
            if (PASS != GATED_OUT) d2[i] = make_float2(da[j + 2 * i], da[j + 2 * i + 1]);
            if (PASS != GATED_OUT && std::is_same<T, __half>::value) d2[i] = mul2(d2[i], make_float2(scale, scale));
        }
        gated_act<T, ACT, PASS != GATED_OUT>(g2, act, slope);
        unsigned char* to = a + (column + j) / 8 * CB + row * 16;
        auto put = [&](unsigned char* where, int plane, auto value) {
            float v[8];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float2 q = value(i);
                v[2 * i] = q.x, v[2 * i + 1] = q.y;
            }
            store_terms8<T, HIDDEN>(where, plane, v);
        };
        if constexpr (PASS == GATED_OUT) {
            put(to, PLANE, [&](int i) { return mul2(act[i], u2[i]); });
        } else {
            put(to, PLANE, [&](int i) { return mul2(mul2(d2[i], u2[i]), slope[i]); });
            put(to + C / 8 * CB, PLANE, [&](int i) { return mul2(d2[i], act[i]); });
            if constexpr (PASS == GATED_DW) put(to + HIDDEN * PLANE, tile_bytes(ROWS, C), [&](int i) { return mul2(act[i], u2[i]); });
        }
    }
}

// The weights that one of the two warps of products fetches for itself: a chunk of one kind for every step, or (all of them there) once.
struct WeightRing {
    unsigned char* buffers;
    const unsigned char* from;   // of the first chunk
    u64 *full, *free;
    int count, bytes, chunks, chunk0;
    long long pitch;             // from a chunk to the next in memory
    bool resident;
    long long asked = 0, all;
    int next = 0;                // the chunk to ask for
    Turn use, load, freed;
    __device__ __forceinline__ void ask() {
        mbar_expect_tx(&full[load.at], bytes);
        bulk_load(buffers + load.at * bytes, from + (chunk0 + next) * pitch, bytes, &full[load.at]);
        load.next(count);
        asked++;
        if (++next == chunks) next = 0;
    }
    __device__ __forceinline__ void begin() {
        if (resident) all = min(all, (long long)chunks);
        while (asked < min(all, (long long)count)) ask();
    }
    // After the products of step q have been asked for: the buffer of the step before (or, of one buffer, its own) gets what comes next.
    __device__ __forceinline__ void used(Waits& wait, long long q) {
        if (resident) return;
        tensor_commit(&free[use.at]);
        use.next(count);
        if ((q == 0 && count > 1) || asked == all) return;
        if (!wait.on(&free[freed.at], freed.turns)) return;
        freed.next(count);
        ask();
    }
    __device__ __forceinline__ void end(Waits& wait) {   // nothing on its way when others have given up
        if (wait.alive && !*wait.dead) return;
        for (long long i = max(0ll, asked - count); i < asked; i++) Waits{wait.dead}.on(&full[i % count], (int)(i / count), true);
    }
};

template <typename T, GatedPass PASS, int ROWS, bool FINE>
__global__ void __launch_bounds__(GatedWarps<T>::THREADS, 1) gated_kernel(const __grid_constant__ GatedArgs p, const __grid_constant__ GatedMaps maps) {
    extern __shared__ __align__(1024) unsigned char smem[];
    using Smem = GatedSmem<T, PASS, ROWS, FINE>;
    using Columns = GatedColumns<T, PASS>;
    constexpr int C = gated_chunk<T>(), TERMS = Tensor<T>::TERMS, HIDDEN = Smem::HIDDEN;
    constexpr int WORKERS = GatedWarps<T>::WORKERS, LOADERS = GatedWarps<T>::LOADERS, THREADS = GatedWarps<T>::THREADS;
    const Smem at(p);
    const Columns col(p);
    GatedBarriers& b = *reinterpret_cast<GatedBarriers*>(smem);
    float* bias_s = reinterpret_cast<float*>(smem + 1024);   // of out
    const int warp = __shfl_sync(~0u, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    // The last of the loaders brings the residual and takes the output away, and takes dout to the residual's gradient.
    const bool scales = PASS == GATED_DX && p.dresidual && p.box_x && p.box_grad && p.wide_dresidual;   // by the first of them, from the tile of dout: another that reads it
    const bool beside = p.io_buffers || (PASS == GATED_DX && p.dresidual && !scales);
    const int row_loaders = LOADERS - (beside ? 1 : 0);
    const bool boxes = p.box_x || p.box_grad, staged_rows = !p.box_x || (PASS != GATED_OUT && !p.box_grad);
    if (threadIdx.x == 0) {
        for (int i = 0; i < p.x_buffers; i++) mbar_init(&b.x_full[i], (boxes ? 1 : 0) + (staged_rows ? 32 * row_loaders : 0)), mbar_init(&b.x_free[i], scales ? 2 : 1);
        for (int i = 0; i < 2; i++) {
            mbar_init(&b.s_full[i], 1), mbar_init(&b.s_free[i], WORKERS / 2);
            mbar_init(&b.a_full[i], WORKERS / 2), mbar_init(&b.a_free[i], 1);
            mbar_init(&b.d_full[i], 1), mbar_init(&b.d_free[i], WORKERS);
            for (int j = 0; j < p.w_buffers[i]; j++) mbar_init(&b.w_full[i][j], 1), mbar_init(&b.w_free[i][j], 1);
            mbar_init(&b.end[i], 1);
        }
        for (int i = 0; i < p.io_buffers; i++) mbar_init(&b.io_full[i], 1), mbar_init(&b.io_done[i], WORKERS);
        b.dead = 0;
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(shared_address(&b.tensor)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    if (p.biased || p.down_bias_wanted) {   // a column of ones
        float one[8] = {1.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, none[8] = {};
        using Term = typename Tensor<T>::Term;
        for (int i = threadIdx.x; i < 2 * ROWS; i += THREADS) store_terms8<Term>(smem + at.at_ones + 16 * i, 0, i < ROWS ? one : none);
    }
    fence_async_proxy();
    wait_for_previous_kernel();
    if constexpr (PASS == GATED_OUT)
        for (int i = threadIdx.x; i < p.np; i += THREADS) bias_s[i] = p.down_bias && i < p.n ? to_float(static_cast<const T*>(p.down_bias)[i]) : 0.f;
    constexpr bool SCALED = PASS != GATED_OUT && std::is_same<T, __half>::value;   // dg and du by a power of two
    u32* peaks_s = reinterpret_cast<u32*>(smem + 1024);   // a warp's
    if constexpr (SCALED) {
        u32 peak = 0;
        for (int i = threadIdx.x; i < p.peak_count; i += THREADS) peak = max(peak, p.peaks[i]);
        peak = __reduce_max_sync(~0u, peak);
        if (lane == 0) peaks_s[warp] = peak;
    }
    tensor_before_sync();
    __syncthreads();
    tensor_after_sync();
    const u32 tensor = __shfl_sync(~0u, b.tensor, 0);
    Waits wait{&b.dead};

    // What this CTA does: tiles from `split` on, every `step`-th, each through `chunks` chunks from `chunk0` on.
    const long long tiles = (p.rows + ROWS - 1) / ROWS;
    const int split = PASS == GATED_DW ? blockIdx.x / p.chunks : blockIdx.x, step = PASS == GATED_DW ? p.splits : gridDim.x;
    const int chunk0 = PASS == GATED_DW ? blockIdx.x % p.chunks : 0, chunks = PASS == GATED_DW ? 1 : p.chunks;
    const long long mine = split < tiles ? (tiles - split + step - 1) / step : 0;
    const long long all = mine * chunks;                                  // steps: chunks of tiles
    const int group = PASS == GATED_DW ? p.drain : chunks;                // steps whose sums are one
    auto rows_over_columns = [](u32 a, int columns) { return TERMS == 1 ? swizzled_over_columns(a, ROWS) : over_columns(a, ROWS, columns); };
    auto rows_over_rows = [](u32 a, int columns) { return TERMS == 1 ? swizzled_over_rows(a, ROWS) : over_rows(a, ROWS, columns); };
    auto ring = [&](int which) {
        const bool down = (which == 0) != (PASS == GATED_OUT);
        const int down_bytes = gated_down_bytes<T>(p.np);
        WeightRing r{smem + at.at_w[which], p.packed + (down ? 0 : down_bytes), b.w_full[which], b.w_free[which], p.w_buffers[which], at.w[which], chunks,
                     chunk0, (long long)down_bytes + gated_up_bytes<T>(p.kp), p.w_buffers[which] >= chunks};
        r.all = all;
        return r;
    };

    if (warp >= WORKERS + 2) {   // loaders
        const int loader = warp - WORKERS - 2;
        if (beside && loader == LOADERS - 1) {
            constexpr int BOX = 128 / sizeof(T);
            const int width = PASS == GATED_OUT ? p.n : p.k;
            const bool one = one_of_warp(), loads = PASS == GATED_OUT && p.residual;
            long long arrived = 0;      // tiles whose buffer has been given to the workers
            Turn out, given;
            auto give = [&]() {         // the next tile's, with its residual
                u64* bar = &b.io_full[given.at];
                unsigned char* io = smem + at.at_io + given.at * at.io;
                given.next(p.io_buffers);
                if (loads) {
                    mbar_expect_tx(bar, at.io);
                    for (int c = 0; c < width; c += BOX) box_load(io + c / BOX * ROWS * 128, &maps.residual, c, (int)((split + arrived * step) * ROWS), bar);
                } else {
                    mbar_arrive(bar);
                }
                arrived++;
            };
            if (one)
                while (arrived < min(mine, (long long)p.io_buffers)) give();
            for (long long t = 0; t < mine && wait.alive; t++) {
                const long long row0 = (split + t * step) * ROWS;
                if (PASS == GATED_DX && p.dresidual && !scales)
                    scale_rows<T>(static_cast<T*>(p.dresidual) + row0 * p.n, static_cast<const T*>(p.grad) + row0 * p.n,
                                  (int)min((long long)ROWS, p.rows - row0) * p.n, p.scale, p.wide_dresidual);
                if (p.io_buffers) {
                    if (!wait.full(b.io_done, out)) break;
                    if (one) {
                        const unsigned char* io = smem + at.at_io + out.at * at.io;
                        for (int c = 0; c < width; c += BOX) box_store(&maps.out, c, (int)row0, io + c / BOX * ROWS * 128);
                        bulk_commit();
                        bulk_wait_read();
                        if (arrived < mine) give();
                    }
                    __syncwarp();
                    out.next(p.io_buffers);
                }
            }
            if (one) {
                bulk_wait_all();
                if (loads && b_dead(b))     // nothing on its way when others have given up
                    for (long long i = max(0ll, arrived - p.io_buffers); i < arrived; i++)
                        Waits{&b.dead}.on(&b.io_full[i % p.io_buffers], (int)(i / p.io_buffers), true);
            }
        } else if (!boxes) {
            // (by themselves: beside the boxes' code in one loop these took half as long again)
            Turn xt;
            for (long long t = 0; t < mine && wait.alive; t++) {
                const long long row0 = (split + t * step) * ROWS;
                const int valid = (int)min((long long)ROWS, p.rows - row0);
                if (!wait.free(b.x_free, xt)) break;
                unsigned char* x = smem + at.at_x + xt.at * at.x;
                if constexpr (PASS != GATED_OUT)
                    stage<T, ROWS>(x, p.np / 8, static_cast<const T*>(p.grad) + row0 * p.n, p.n, valid, p.wide_grad, loader, row_loaders);
                stage<T, ROWS>(x + at.grad, p.kx / 8, static_cast<const T*>(p.x) + row0 * p.k, p.k, valid, p.wide_x, loader, row_loaders);
                fence_async_proxy();
                mbar_arrive(&b.x_full[xt.at]);
                xt.next(p.x_buffers);
            }
        } else if (staged_rows || loader == 0) {
            const bool one = loader == 0 && one_of_warp();
            const int box_bytes = (p.box_x ? at.x - at.grad : 0) + (p.box_grad ? at.grad : 0);
            Turn xt, st;
            auto scale = [&](long long t) {
                if constexpr (sizeof(T) == 2) {
                    if (!wait.full(b.x_full, st)) return;
                    const long long row0 = (split + t * step) * ROWS;
                    scale_tile<T, ROWS>(static_cast<T*>(p.dresidual) + row0 * p.n, smem + at.at_x + st.at * at.x, (int)min((long long)ROWS, p.rows - row0),
                                        p.n / 8, p.scale);
                    __syncwarp();
                    if (one) mbar_arrive(&b.x_free[st.at]);
                    st.next(p.x_buffers);
                }
            };
            const int behind = p.x_buffers >= 2 ? 1 : 0;      // a tile is scaled when the next one has been asked for
            for (long long t = 0; t < mine; t++) {
                const long long row0 = (split + t * step) * ROWS;
                const int valid = (int)min((long long)ROWS, p.rows - row0);
                if (!wait.free(b.x_free, xt)) break;
                unsigned char* x = smem + at.at_x + xt.at * at.x;
                u64* full = &b.x_full[xt.at];
                if (one) {
                    mbar_expect_tx(full, box_bytes);
                    if (p.box_grad)
                        for (int c = 0; c < p.n; c += 64) box_load(x + c * ROWS * 2, &maps.grad, c, (int)row0, full);
                    if (p.box_x)
                        for (int c = 0; c < p.k; c += 64) box_load(x + at.grad + c * ROWS * 2, &maps.x, c, (int)row0, full);
                }
                __syncwarp();
                if (staged_rows) {
                    if (PASS != GATED_OUT && !p.box_grad)
                        stage<T, ROWS>(x, p.np / 8, static_cast<const T*>(p.grad) + row0 * p.n, p.n, valid, p.wide_grad, loader, row_loaders);
                    if (!p.box_x)
                        stage<T, ROWS>(x + at.grad, p.kx / 8, static_cast<const T*>(p.x) + row0 * p.k, p.k, valid, p.wide_x, loader, row_loaders);
                    fence_async_proxy();
                    mbar_arrive(full);
                }
                xt.next(p.x_buffers);
                if (scales && t >= behind) scale(t - behind);
            }
            if (scales && behind && mine > 0 && wait.alive) scale(mine - 1);
            // nothing on its way when others have given up
            if (one && b_dead(b))
                for (int i = 0; i < p.x_buffers; i++) {
                    const int turns = xt.turns - (i >= xt.at ? 1 : 0);
                    if (turns >= 0) Waits{&b.dead}.on(&b.x_full[i], turns, true);
                }
        }
    } else if (warp == WORKERS) {   // the first products: g, u (, da) of a step
        if (one_of_warp()) {
            WeightRing w = ring(0);
            w.begin();
            Turn xt, wt, w2t;
            int c = 0;
            for (long long q = 0; q < all; q++) {
                if (c == 0 && !wait.full(b.x_full, xt)) break;
                if (!(w.resident && q >= chunks) && !wait.full(b.w_full[0], wt)) break;
                if (PASS != GATED_OUT && !(p.w_buffers[1] >= chunks && q >= chunks) && !wait.full(b.w_full[1], w2t)) break;
                if (q >= p.s_buffers && !wait.step(b.s_free, q - p.s_buffers)) break;
                tensor_after_sync();
                const u32 x = shared_address(smem + at.at_x + xt.at * at.x), s = tensor + ((int)q & (p.s_buffers - 1)) * Columns::WIDE;
                const u32 w0 = shared_address(w.buffers + wt.at * w.bytes), w1 = shared_address(smem + at.at_w[1] + w2t.at * at.w[1]);
                const Operand up = over_rows(PASS == GATED_OUT ? w0 : w1, p.kp, 2 * C);
                // Ones times the biases' row: its small terms with the small products, the large one last.  (Ahead of all, what was cut of every later
                // product was a part of the bias: sums of 128 floats and one were 1.8e-6 off, 3e-7 now.)
                const Operand one = over_columns(shared_address(smem + at.at_ones), ROWS, 16);
                const u32 shape = product_shape<T>(one, up, 2 * C);
                if (p.biased)
                    for (int t = TERMS - 1; t >= 1; t--) tensor_product(s, one.first, up.at(p.kx / 16, t), shape, t < TERMS - 1);
                products<T>(s, s, rows_over_columns(x + at.grad, p.kx), up, 2 * C, p.kx / 16, p.biased && TERMS > 1, p.biased && TERMS > 1);
                if (p.biased) tensor_product(s, one.first, up.at(p.kx / 16, 0), shape, true);
                if constexpr (PASS != GATED_OUT) products<T>(s + 2 * C, s + 2 * C, rows_over_columns(x, p.np), over_columns(w0, C, p.np), C, p.np / 16, false, false);
                tensor_commit(&b.s_full[q & 1]);
                wt.next(w.count), w2t.next(p.w_buffers[1]);
                if (++c == chunks) {
                    c = 0;
                    if (PASS != GATED_DW) tensor_commit(&b.x_free[xt.at]);
                    xt.next(p.x_buffers);
                }
                w.used(wait, q);
                if (!wait.alive) break;
            }
            w.end(wait);
            tensor_commit(&b.end[0]);
        }
    } else if (warp == WORKERS + 1) {   // the second products
        if (one_of_warp()) {
            WeightRing w = ring(1);
            w.begin();
            Turn wt, xt, dt;
            int in_group = 0;
            for (long long q = 0; q < all; q++) {
                if (PASS == GATED_OUT && !(w.resident && q >= chunks) && !wait.full(b.w_full[1], wt)) break;   // (the first products have waited for the others)
                if (!wait.step(b.a_full, q)) break;
                if (in_group == 0 && !wait.free(b.d_free, dt)) break;
                tensor_after_sync();
                const u32 x = shared_address(smem + at.at_x + xt.at * at.x), w1 = shared_address(w.buffers + wt.at * w.bytes);
                const u32 a = shared_address(smem + at.at_a + ((int)q & (p.a_buffers - 1)) * (Smem::A + Smem::ACT));
                const u32 d = tensor + col.d + dt.at * col.d_all;
                const bool add = in_group > 0, add_main = p.split ? in_group > 1 : add;
                const u32 main = d + (p.split ? (in_group & 1) * col.up_part : 0), small = d + (p.split ? 2 : 1) * col.up_part;
                if constexpr (PASS == GATED_OUT && TERMS == 1) {
                    few_products<T, HIDDEN, 1>(d, over_columns(a, ROWS, C), over_rows(w1, C, p.np), p.np, C / 16, add);
                } else if constexpr (PASS == GATED_DX && TERMS == 1) {
                    few_products<T, HIDDEN, 1>(d, over_columns(a, ROWS, 2 * C), over_columns(w1, p.kp, 2 * C), p.kx, 2 * C / 16, add);
                } else if constexpr (PASS == GATED_OUT) {
                    products<T>(main, small, over_columns(a, ROWS, C), over_rows(w1, C, p.np), p.np, C / 16, add_main, add);
                } else if constexpr (PASS == GATED_DX) {
                    products<T>(main, small, over_columns(a, ROWS, 2 * C), over_columns(w1, p.kp, 2 * C), p.kx, 2 * C / 16, add_main, add);
                } else {
                    const Operand hidden = over_rows(a, ROWS, 2 * C), grad = rows_over_rows(x, p.np);
                    const Operand rows = rows_over_rows(x + at.grad, p.kx), act = over_rows(a + Smem::A, ROWS, C);
                    if constexpr (TERMS == 1) {
                        few_products<T, HIDDEN, 1>(d, hidden, rows, p.kx, ROWS / 16, add);
                        few_products<T, 1, HIDDEN>(d + col.down, grad, act, C, ROWS / 16, add);
                    } else if (p.stacked) {
                        stacked_products<T>(d, hidden, rows, p.kx, ROWS / 16, add);
                        stacked_products<T>(d + col.down, grad, act, C, ROWS / 16, add);
                    } else {
                        products<T>(d, d + col.up_part, hidden, rows, p.kx, ROWS / 16, add, add);
                        products<T>(d + col.down, d + col.down + col.down_part, grad, act, C, ROWS / 16, add, add);
                    }
                    // the biases': times ones (which have one term)
                    const Operand one = over_rows(shared_address(smem + at.at_ones), ROWS, 16);
                    auto column_sums = [&](const Operand& of, u32 to, int terms) {   // (16-bit: small terms in the same place, before)
                        const u32 shape = product_shape<T>(of, one, 16);
                        for (int t = terms - 1; t >= 0; t--)
                            for (int s = 0; s < ROWS / 16; s++)
                                tensor_product(to + (t ? col.bias_part : 0), of.at(s, t), one.at(s, 0), shape,
                                               add || s > 0 || (TERMS == 3 ? t == 1 : t < terms - 1));
                    };
                    if (p.biased) column_sums(hidden, d + col.up_bias, HIDDEN);
                    if (p.down_bias_wanted) column_sums(grad, d + col.down_bias, TERMS);
                    tensor_commit(&b.x_free[xt.at]);
                    xt.next(p.x_buffers);
                }
                tensor_commit(&b.a_free[q & 1]);
                wt.next(w.count);
                if (++in_group == group || q + 1 == all) {
                    in_group = 0;
                    tensor_commit(&b.d_full[dt.at]);
                    dt.next(p.d_buffers);
                }
                w.used(wait, q);
                if (!wait.alive) break;
            }
            w.end(wait);
            tensor_commit(&b.end[1]);
        }
    } else {   // workers
        constexpr int PARTS = WORKERS / 8, W = C / PARTS;   // of one half: warps of 32 rows, hidden channels of each
        const int quarter = warp & 3, part = (warp >> 2) % PARTS, half = warp / (WORKERS / 2), row = 32 * quarter + lane;
        const bool works = 32 * quarter < ROWS;
        const u32 lanes = tensor + ((u32)(32 * quarter) << 16);
        Turn dt;
        Turn io_turn;
        float scale = 1.f, unscale = 1.f;
        if constexpr (SCALED) {
            u32 peak = 0;
            for (int w = 0; w < THREADS / 32; w++) peak = max(peak, peaks_s[w]);
            const u32 exponent = gated_scale_exponent(peak);
            scale = __uint_as_float((127 + exponent) << 23), unscale = __uint_as_float((127 - exponent) << 23);
        }
        // The finished sums: of this CTA's index-th tile, or group of tiles.
        auto take_out = [&](long long index) {
            if (!wait.full(b.d_full, dt)) return;
            tensor_after_sync();
            const u32 d = lanes + col.d + dt.at * col.d_all;
            const long long row0 = PASS == GATED_DW ? 0 : (split + index * step) * ROWS, at_row = row0 + row;
            const bool there = works && at_row < p.rows, staged = PASS != GATED_DW && p.io_buffers;
            const int width = PASS == GATED_OUT ? p.n : p.k;
            float* share = PASS == GATED_DW ? p.shares + ((long long)chunk0 * p.splits + split) * col.d_one * 128 + row : nullptr;
            unsigned char* io = smem + at.at_io + io_turn.at * at.io;
            if (staged && !wait.full(b.io_full, io_turn)) return;   // the residual is there, and the rows before have left
            for (int c = 16 * (2 * part + half); c < col.d_one; c += 32 * PARTS) {
                float v[16], low[16];
                __syncwarp();
                int part, parts;
                const u32 from = d + col.place(p, c, part, parts);
                tensor_load(v, from);
                if (Columns::SUMS == 2) tensor_load(low, from + part);
                tensor_loaded();
                if (Columns::SUMS == 2) {
                    if (parts == 3) {   // the smallest first
                        float third[16];
                        tensor_load(third, from + 2 * part);
                        tensor_loaded();
#pragma unroll
                        for (int j = 0; j < 16; j++) low[j] += third[j];
                    }
#pragma unroll
                    for (int j = 0; j < 16; j++) v[j] += low[j];
                }
                if (SCALED && (PASS == GATED_DX || c < p.kp)) {   // (dWd and dbd are of dout as it is)
#pragma unroll
                    for (int j = 0; j < 16; j++) v[j] *= unscale;
                }
                if constexpr (PASS == GATED_DW) {
                    float* to = share + (long long)c * 128;
                    if (index) {
#pragma unroll
                        for (int j = 0; j < 16; j++) v[j] += to[j * 128];
                    }
#pragma unroll
                    for (int j = 0; j < 16; j++) to[j * 128] = v[j];
                } else if (there) {
                    if constexpr (PASS == GATED_OUT) {
                        if (p.down_bias) {
#pragma unroll
                            for (int j = 0; j < 16; j += 4) {
                                const float4 q = *reinterpret_cast<const float4*>(bias_s + c + j);
                                v[j] += q.x, v[j + 1] += q.y, v[j + 2] += q.z, v[j + 3] += q.w;
                            }
                        }
                        if (p.residual) {
                            float r[16];
                            if (staged) io_load16<T, ROWS>(r, io, row, c, width);
                            else load16(r, static_cast<const T*>(p.residual) + at_row * width + c, width - c, p.wide_out);
#pragma unroll
                            for (int j = 0; j < 16; j++) v[j] = fmaf(p.scale, r[j], v[j]);
                        }
                    }
                    if (staged) io_store16<T, ROWS>(io, row, c, v, width);
                    else store16(static_cast<T*>(p.out) + at_row * width + c, v, width - c, p.wide_out);
                }
            }
            tensor_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(&b.d_free[dt.at]);
            dt.next(p.d_buffers);
            if (!staged) return;
            fence_async_proxy();
            __syncwarp();
            if (lane == 0) mbar_arrive(&b.io_done[io_turn.at]);
            io_turn.next(p.io_buffers);
        };
        // Sums are taken out after the half's next step, when their last products have had time; amid it where that step's operand may have to wait for
        // second products, which wait for the sums' place; before it where its first products may, too (for weights or, in DW, for rows).
        const bool late = p.d_buffers == 2 || (PASS == GATED_OUT && p.a_buffers == 2);
        const bool amid = !late && (PASS == GATED_DW ? p.x_buffers >= 2 : PASS == GATED_DX && (p.w_buffers[1] >= chunks || p.w_buffers[1] >= 3));
        long long taken = 0, before = 0;      // groups of steps: whose sums have been taken out, that are done
        int in_group = half;
        for (long long q = half; q < all && wait.alive; q += 2, in_group += 2) {
            for (; in_group >= group; in_group -= group) before++;
            if (!late && !amid)
                while (taken < before && wait.alive) take_out(taken++);
            if (!wait.step(b.s_full, q)) break;
            if (amid)
                while (taken < before && wait.alive) take_out(taken++);
            tensor_after_sync();
            const u32 s = lanes + ((int)q & (p.s_buffers - 1)) * Columns::WIDE + W * part;
            unsigned char* a = smem + at.at_a + ((int)q & (p.a_buffers - 1)) * (Smem::A + Smem::ACT);
            const bool behind = PASS == GATED_DW && (split + q * step) * ROWS + row >= p.rows;
#pragma unroll 1
            for (int j = 0; j < W; j += 16) {
                float g[16], u[16], da[16];
                tensor_load(g, s + j);
                tensor_load(u, s + C + j);
                if (PASS != GATED_OUT) tensor_load(da, s + 2 * C + j);
                tensor_loaded();
                if (j + 16 == W) {
                    tensor_before_sync();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&b.s_free[half]);
                }
                if (j == 0 && q >= p.a_buffers && !wait.step(b.a_free, q - p.a_buffers)) break;
                // Rows behind the last one have zeros for x and dout, but g and u are the biases: a must be zero too, since infinity (float16: biases of some 300)
                // times a zero of dout is not.
                if (PASS == GATED_DW && behind) {
#pragma unroll
                    for (int i = 0; i < 16; i++) u[i] = 0.f;
                }
                if (works) {
                    if (p.activation == PL_GATE_SILU) gated_work<T, PASS, PL_GATE_SILU, ROWS, HIDDEN>(g, u, da, scale, a, row, W * part + j);
                    else if (p.activation == PL_GATE_GELU) gated_work<T, PASS, PL_GATE_GELU, ROWS, HIDDEN>(g, u, da, scale, a, row, W * part + j);
                    else if (p.activation == PL_GATE_SIGMOID) gated_work<T, PASS, PL_GATE_SIGMOID, ROWS, HIDDEN>(g, u, da, scale, a, row, W * part + j);
                    else gated_work<T, PASS, PL_GATE_RELU, ROWS, HIDDEN>(g, u, da, scale, a, row, W * part + j);
                }
                __syncwarp();
            }
            if (!wait.alive) break;
            fence_async_proxy();
            __syncwarp();
            if (lane == 0) mbar_arrive(&b.a_full[half]);
            while (taken < before && wait.alive) take_out(taken++);
        }
        const long long groups = (all + group - 1) / group;
        while (taken < groups && wait.alive) take_out(taken++);
    }
    // All products are done, or a wait has run out: then nothing that could pass for a result.
    __syncwarp();
    if (warp == WORKERS || warp == WORKERS + 1) Waits{&b.dead}.on(&b.end[warp - WORKERS], 0, true);
    __syncthreads();
    if (b.dead) {
        if constexpr (PASS == GATED_DW) {
            float* share = p.shares + ((long long)chunk0 * p.splits + split) * col.d_one * 128;
            for (int i = threadIdx.x; i < col.d_one * 128; i += THREADS) share[i] = NAN;
        } else {
            const GatedRows<T> outputs[2] = {{static_cast<T*>(p.out), PASS == GATED_OUT ? p.n : p.k}, {PASS == GATED_DX ? static_cast<T*>(p.dresidual) : nullptr, p.n}};
            give_up(outputs, GatedTiles{p.rows, split, step, ROWS}, from_float<T>(NAN), (int)threadIdx.x, THREADS);
        }
    }
    tensor_before_sync();
    __syncthreads();
    tensor_after_sync();
    if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tensor) : "memory");
}

// The gradients of weights and biases from the shares: a value a thread, those of consecutive hidden channels (of dWg, dWu, dbg, dbu) or of
// consecutive channels out (dWd, dbd) side by side in a share.
struct GatedSums {
    const float* shares;
    int k, h, n, kx, chunk, chunks, splits, columns, down, bias;
    void *gate_weight, *up_weight, *down_weight, *gate_bias, *up_bias, *down_bias;
};
template <typename T>
__global__ void __launch_bounds__(256) gated_sums(const __grid_constant__ GatedSums p) {
    // rows of the grid: k rows of dWg, (one of dbg,) as many of up, h rows of dWd, (one of dbd)
    int r = blockIdx.y;
    const int i = blockIdx.x * 256 + threadIdx.x;
    const bool first = r < 2 * (p.k + 1), up = first && r > p.k;
    int chunk, column, line;
    T* to;
    if (first) {
        if (up) r -= p.k + 1;
        if (i >= p.h) return;
        void* bias = up ? p.up_bias : p.gate_bias;
        void* weight = up ? p.up_weight : p.gate_weight;
        if (r == p.k ? !bias : !weight) return;
        to = r == p.k ? static_cast<T*>(bias) + i : static_cast<T*>(weight) + (long long)r * p.h + i;
        chunk = i / p.chunk, column = r == p.k ? p.kx : r, line = i % p.chunk + (up ? p.chunk : 0);
    } else {
        r -= 2 * (p.k + 1);
        if (i >= p.n) return;
        if (r == p.h ? !p.down_bias : !p.down_weight) return;
        to = r == p.h ? static_cast<T*>(p.down_bias) + i : static_cast<T*>(p.down_weight) + (long long)r * p.n + i;
        chunk = r == p.h ? 0 : r / p.chunk, column = r == p.h ? p.bias : p.down + r % p.chunk, line = i;
    }
    const float* from = p.shares + ((long long)chunk * p.splits * p.columns + column) * 128 + line;
    double sum = 0.0;   // (its place in the time is not seen; a float was 1e-7 off)
#pragma unroll 8
    for (int s = 0; s < p.splits; s++) sum += (double)from[(long long)s * p.columns * 128];
    *to = from_float<T>((float)sum);
}

}  // namespace pl
