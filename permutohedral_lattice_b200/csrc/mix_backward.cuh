// The gradients of act(x W [+ x2 W2] + ...): dz from the upstream gradient and the output, dx = dz W^T, dW = x^T dz.
//
// mix_backward (up to 80 input and 32 output channels): everything in one pass over memory, by tiles of a warp's own (see
// mix_common.cuh).  A warp takes 32 rows at a time: dz to the place where the output came in, their share of dW into registers
// that last for the whole kernel, dx into the place where x came in.  At the end a CTA's warps add their shares of dW up,
// mix_add_shares those of the CTAs, in double and in a fixed order.
//
// 16 x 512x512 rows of 21 + 21 channels to 21, floats: 496 us, 5.0 TB/s of what has to be moved (358 without dW); from activations in 8
// bits 618, a fifth of it their decoding.  Three CTAs of four warps an SM, 168 registers: bound by issue slots (1920 instructions for 32
// rows, in 8 bits 2530, at 2 of 4 a cycle).
//
// Beyond that dW does not fit a warp's registers: mix_dz writes dz to the workspace, mix_forward multiplies it by the
// transposed weights, mix_backward_weights gives a CTA's warps blocks of dW to sum over all its rows.
#pragma once
#include <type_traits>
#include "mix_common.cuh"
#include "mix_forward.cuh"

namespace pl {

struct Kept {   // an activation as it was, or in 8 bits
    const void* full;
    const uint8_t* codes;
    const int16_t* scales;
};
struct MixBackArgs {
    long long rows;
    int k, k2, n, activation;
    float scale;                       // of the residual
    const void* grad;
    Kept out, x, x2;
    const void *weight, *weight2;
    int weight_dtype;
    void *dx, *dx2, *dresidual;        // NULL: not wanted
    float* shares;                     // [CTAs][(k + k2 + 1) n]: dW, dW2 and dbias; NULL: none of them wanted
    int bias;                          // dbias is wanted
    float* dz;                         // the wide way: [rows][n]
    int want_x, want_x2;               // its product with dz is wanted
    int stages, blocks;                // blocks of 32 rows in a tile
};

// W^T and dz in shared memory: blocks of 8 x 8 as the lanes take them, both terms of W^T (see mix_common.cuh), dz as it is; nb of them
// for eight rows.
constexpr int MIX_BLOCK = 512, MIX_DZ_BLOCK = 256;

// Shared memory, in bytes.  A stage holds a tile's rows of the gradient (dresidual leaves from there), the output, x and x2 (dx and
// dx2 leave from there); a warp's own memory dz of the 32 rows that it works on and, where some of them come in 8 bits, the output,
// then x and x2 as floats (dx and dx2 leave from there then).
struct MixBackSmem {
    size_t weights, stage0, stage_bytes, own0, own_bytes;
    size_t y_at, x_at, x2_at;   // of a stage
    size_t work_at, work2_at;   // of a warp's own memory, dz before
    __host__ __device__ MixBackSmem(const MixBackArgs& a, int warps, int nb, int size /* of a value */, bool packed) {
        const size_t rows = 32 * (size_t)a.blocks;
        const int k = a.k, k2 = a.k2, n = a.n;
        weights = up16(sizeof(u64) * MIX_WARPS * MIX_STAGES);   // barriers before
        stage0 = weights + (size_t)(up8(k) + up8(k2)) / 8 * nb * MIX_BLOCK;
        y_at = up16(rows * n * size);
        x_at = y_at + (a.activation == PL_ACT_NONE ? 0 : up16(rows * n * (a.out.codes ? 1 : size)));
        x2_at = x_at + (packed && !a.want_x ? 0 : up16(rows * k * (a.x.codes ? 1 : size)));
        stage_bytes = x2_at + (packed && !a.want_x2 ? 0 : up16(rows * k2 * (a.x2.codes ? 1 : size)));
        work_at = 4 * nb * MIX_DZ_BLOCK;
        work2_at = work_at + (packed ? up16(sizeof(float) * 32 * (size_t)k) : 0);
        own_bytes = work2_at + (packed ? up16(sizeof(float) * 32 * (size_t)(k + k2 > n ? k2 : n - k)) : 0);
        own0 = stage0 + stage_bytes * a.stages * warps;
    }
    __host__ __device__ size_t bytes(int warps) const { return own0 + own_bytes * warps + 128; }   // (reads of eight channels pass the last one)
};

// 0 where the output is zero, NaN where it is: of a block in 8 bits that held an infinity nothing is known but that.
__device__ __forceinline__ float relu_gradient(float y, float g) { return y > 0.f ? g : y * 0.f; }

// PACKED: some of the output, x and x2 come in 8 bits; all are then read from floats of the warp's own memory.  One stage, and the
// headers of its blocks in registers: there are at most 32 of the output and 96 of x or x2 in a tile (see narrow_any).
template <typename T, bool PACKED, int MB, int NB>
__global__ void __launch_bounds__(32 * MIX_WARPS, MB * NB > 12 ? 2 : 3) mix_backward(MixBackArgs a) {
    extern __shared__ __align__(128) unsigned char smem[];
    typedef typename std::conditional<PACKED, float, T>::type TX;   // of the rows that are worked on
    const int warps = (int)blockDim.x / 32, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int tile_rows = 32 * a.blocks, k = a.k, k2 = a.k2, n = a.n, stages = PACKED ? 1 : a.stages;
    const MixBackSmem at(a, warps, NB, sizeof(T), PACKED);
    const bool reads_y = a.activation != PL_ACT_NONE;
    u64* bars = reinterpret_cast<u64*>(smem) + MIX_STAGES * warp;
    unsigned char* stage0 = smem + at.stage0 + at.stage_bytes * stages * warp;
    const T* grad = static_cast<const T*>(a.grad);
    const long long tiles = (a.rows + tile_rows - 1) / tile_rows, step = (long long)gridDim.x * warps;
    const long long first = (long long)blockIdx.x * warps + warp;
    if (lane == 0)
        for (int s = 0; s < stages; s++) mbar_init(&bars[s], 1);
    __syncwarp();
    auto kept_aligned = [](const Kept& p) { return p.codes ? aligned16(p.codes) : aligned16(p.full); };
    auto kept_bytes = [&](const Kept& p, int c) { return (u32)(tile_rows * c * (p.codes ? 1 : sizeof(T))); };
    // (codes of an odd number of 32-row blocks of an odd number of channels: 32 c bytes, a multiple of 16 all the same)
    const bool bulk_in = aligned16(grad) && (!reads_y || kept_aligned(a.out)) && (!a.want_x || kept_aligned(a.x)) && (!a.want_x2 || kept_aligned(a.x2));
    const u32 tile_bytes = (u32)(tile_rows * n * sizeof(T)) + (reads_y ? kept_bytes(a.out, n) : 0) + (a.want_x ? kept_bytes(a.x, k) : 0) +
                           (a.want_x2 ? kept_bytes(a.x2, k2) : 0);
    u32 heads_y = 0, heads_x[3] = {0, 0, 0}, heads_x2[3] = {0, 0, 0};
    auto fetch = [&](long long tile, int s) {
        unsigned char* stage = stage0 + at.stage_bytes * s;
        const long long row0 = tile * tile_rows;
        if (row0 >= a.rows) return;
        const int here = (int)min((long long)tile_rows, a.rows - row0);
        if constexpr (PACKED) {
            auto heads_in = [&](u32* heads, int most, const Kept& p, int c) {
                if (!p.codes) return;
                const int count = (here * c + PACK_BLOCK - 1) / PACK_BLOCK;
                const int16_t* from = p.scales + row0 * c / PACK_BLOCK;
#pragma unroll
                for (int i = 0; i < most; i++)
                    if (32 * i + lane < count) heads[i] = (u32)(u16)from[32 * i + lane];
            };
            if (reads_y) heads_in(&heads_y, 1, a.out, n);
            if (a.want_x) heads_in(heads_x, 3, a.x, k);
            if (a.want_x2) heads_in(heads_x2, 3, a.x2, k2);
        }
        auto from = [&](const Kept& p, int c) -> const void* {
            return p.codes ? static_cast<const void*>(p.codes + row0 * c) : static_cast<const void*>(static_cast<const T*>(p.full) + row0 * c);
        };
        if (bulk_in && here == tile_rows) {
            if (lane == 0) {
                mbar_expect_tx(&bars[s], tile_bytes);
                bulk_load(stage, grad + row0 * n, (u32)(tile_rows * n * sizeof(T)), &bars[s]);
                if (reads_y) bulk_load(stage + at.y_at, from(a.out, n), kept_bytes(a.out, n), &bars[s]);
                if (a.want_x) bulk_load(stage + at.x_at, from(a.x, k), kept_bytes(a.x, k), &bars[s]);
                if (a.want_x2) bulk_load(stage + at.x2_at, from(a.x2, k2), kept_bytes(a.x2, k2), &bars[s]);
            }
        } else {
            auto rows_in = [&](size_t place, const Kept& p, int c) {
                if (p.codes) {
                    copy_in(stage + place, p.codes + row0 * c, here * c);
                    return;
                }
                copy_in(stage + place, static_cast<const T*>(p.full) + row0 * c, here * c);
                // rows of a block that are not there: their dz is zero, their x must not be NaN
                T* to = reinterpret_cast<T*>(stage + place);
                for (int i = here * c + lane; i < (here + 31) / 32 * 32 * c; i += 32) to[i] = from_float<T>(0.f);
            };
            copy_in(stage, grad + row0 * n, here * n);
            if (reads_y) rows_in(at.y_at, a.out, n);
            if (a.want_x) rows_in(at.x_at, a.x, k);
            if (a.want_x2) rows_in(at.x2_at, a.x2, k2);
            if (lane == 0) mbar_expect_tx(&bars[s], 0);
        }
    };
    for (int s = 0; s < stages; s++) fetch(first + s * step, s);

    // W^T: a row an input channel, zeros behind the last channel of either side
    const int kp = up8(k), all_p = kp + up8(k2);
    for_weights<8 * NB>(all_p, kp, k, k2, n, a.weight, a.weight2, 0, a.weight_dtype, [&](int r, int c, float v) {
        u32 hi, lo;
        split(v, hi, lo);
        // the product's rows are the output channels c, its columns the input channels r
        u32* to = reinterpret_cast<u32*>(smem + at.weights + ((r >> 3) * NB + (c >> 3)) * MIX_BLOCK + (4 * (r & 7) + (c & 3)) * 16 + 4 * (c >> 2 & 1));
        to[0] = hi, to[2] = lo;
    });
    __syncthreads();

    const int g = lane >> 2, t = lane & 3;
    const bool split_w = a.weight_dtype == PL_F32;
    // 8-bit codes times a power of two need no second term, nor do 16 bits
    const bool split_x = sizeof(T) == 4 && !(PACKED && (!a.want_x || a.x.codes) && (!a.want_x2 || a.x2.codes));
    const bool bulk_out = aligned16(a.dx) && aligned16(a.dx2) && aligned16(a.dresidual);   // (NULL counts as aligned)
    unsigned char* own = smem + at.own0 + at.own_bytes * warp;
    const u32 dz_at = shared_address(own), w_at = shared_address(smem + at.weights);
    float acc[MB][NB][4], sums[NB];
#pragma unroll
    for (int i = 0; i < MB; i++)
#pragma unroll
        for (int j = 0; j < NB; j++)
#pragma unroll
            for (int e = 0; e < 4; e++) acc[i][j][e] = 0.f;
#pragma unroll
    for (int j = 0; j < NB; j++) sums[j] = 0.f;

    constexpr int J = 2 * NB, FULL = 2 * NB - 2;   // channels of a row that a lane looks at: every fourth; those that are there whatever n is
    bool alive = true;
    int s = 0, parity = 0;
    for (long long tile = first; tile < tiles; tile += step) {
        unsigned char* stage = stage0 + at.stage_bytes * s;
        cp_async_wait_all();
        alive = alive && mbar_wait(&bars[s], parity);
        alive = __all_sync(~0u, alive);
        __syncwarp();   // what the lanes copied is there for all
        const long long tile0 = tile * tile_rows;
        const int rows_here = (int)min((long long)tile_rows, a.rows - tile0);
#pragma unroll 1
        for (int r0 = 0; r0 < rows_here; r0 += 32) {
            const int here = min(32, rows_here - r0);
            // 32 rows to floats, four lanes a block; rows that are not there to zeros.  Every other block's lanes take their two halves the
            // other way round, so that lanes which write together write to different banks.
            auto decode = [&](float* to, const Kept& p, const unsigned char* place, const u32* heads, int most, int c) {
                const int from = 32 * (lane >> 2) + 8 * (lane & 3), swap = lane & 4;
                float* w = to + from;
                int left = c - (lane >> 2);   // blocks, from this lane's on
                if (p.codes) {
                    const uint2* codes = reinterpret_cast<const uint2*>(place + r0 * c + from);
                    int b = r0 / 32 * c + (lane >> 2);
                    for (int i = 0; i < c; i += 8, left -= 8, b += 8, w += 256, codes += 32) {
                        u32 head = __shfl_sync(~0u, heads[0], b);
                        if (most > 1 && c > 32) {
                            const u32 second = __shfl_sync(~0u, heads[most > 1 ? 1 : 0], b), third = __shfl_sync(~0u, heads[most > 2 ? 2 : 0], b);
                            head = b < 32 ? head : b < 64 ? second : third;
                        }
                        if (left > 0) {
                            const uint2 q = *codes;
                            float v[4];
                            decode4(v, swap ? q.y : q.x, head);
                            store4(w + swap, v);
                            decode4(v, swap ? q.x : q.y, head);
                            store4(w + 4 - swap, v);
                        }
                    }
                } else {
                    const T* values = reinterpret_cast<const T*>(place) + r0 * c + from;
                    for (int i = 0; i < c; i += 8, left -= 8, w += 256, values += 256)
                        if (left > 0) {
                            float v[4];
                            load4(v, values + swap);
                            store4(w + swap, v);
                            load4(v, values + 4 - swap);
                            store4(w + 4 - swap, v);
                        }
                }
                if (here < 32) {
                    __syncwarp();
                    for (int i = here * c + lane; i < 32 * c; i += 32) to[i] = 0.f;
                }
            };
            float* work = reinterpret_cast<float*>(own + at.work_at);
            float* work2 = reinterpret_cast<float*>(own + at.work2_at);
            if constexpr (PACKED) {
                if (reads_y) decode(work, a.out, stage + at.y_at, &heads_y, 1, n);
                __syncwarp();
            }
            // dz: four lanes a row, rows 8 p + g.  A lane's values are just what it takes of dz as the left side of dz W^T; for x^T dz, where
            // others take them, they go to shared memory.
            const u32 g_at = shared_address(stage) + r0 * n * sizeof(T);
            const u32 y_at = PACKED ? shared_address(work) : shared_address(stage + at.y_at) + r0 * n * sizeof(T);
            float d[4][J], y[4][J];
            const u32 g_row = g_at + (g * n + t) * sizeof(T), y_row = y_at + (g * n + t) * sizeof(TX);
#pragma unroll
            for (int p = 0; p < 4; p++)
#pragma unroll
                for (int j = 0; j < J; j++) {
                    const u32 at = g_row + (8 * p * n + 4 * j) * sizeof(T);
                    d[p][j] = j < FULL ? lds_value<T>(at) : lds_value_if<T>(4 * j + t < n, at);
                    y[p][j] = 0.f;
                }
            if (reads_y) {
#pragma unroll
                for (int p = 0; p < 4; p++)
#pragma unroll
                    for (int j = 0; j < J; j++) {
                        const u32 at = y_row + (8 * p * n + 4 * j) * sizeof(TX);
                        y[p][j] = j < FULL ? lds_value<TX>(at) : lds_value_if<TX>(4 * j + t < n, at);
                    }
            }
            if (a.activation == PL_ACT_SOFTMAX) {
                float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int j = 0; j < J; j++)
#pragma unroll
                    for (int p = 0; p < 4; p++) sum[p] = fmaf(y[p][j], d[p][j], sum[p]);
#pragma unroll
                for (int o = 1; o < 4; o <<= 1)
#pragma unroll
                    for (int p = 0; p < 4; p++) sum[p] += __shfl_xor_sync(~0u, sum[p], o);
                // A row that came out as zeros has no gradient, whatever comes from above: -1 / 0 of a logarithm, say.  (One vote, where all
                // sums are finite.)
                bool odd = false;
#pragma unroll
                for (int p = 0; p < 4; p++) odd |= !(fabsf(sum[p]) < INFINITY);
                if (__any_sync(~0u, odd)) {
#pragma unroll
                    for (int p = 0; p < 4; p++) {
                        bool any = false;
#pragma unroll
                        for (int j = 0; j < J; j++) any |= y[p][j] != 0.f;
                        if (__ballot_sync(~0u, any) >> (lane & 28) & 15u) continue;
                        sum[p] = 0.f;
#pragma unroll
                        for (int j = 0; j < J; j++) d[p][j] = 0.f;
                    }
                }
#pragma unroll
                for (int p = 0; p < 4; p++)
#pragma unroll
                    for (int j = 0; j < J; j++) d[p][j] = y[p][j] * (d[p][j] - sum[p]);   // (behind the last channel: see below)
            } else if (a.activation == PL_ACT_RELU) {
#pragma unroll
                for (int p = 0; p < 4; p++)
#pragma unroll
                    for (int j = 0; j < J; j++) d[p][j] = relu_gradient(y[p][j], d[p][j]);
            }
            if (!alive || here < 32) {
#pragma unroll
                for (int p = 0; p < 4; p++)
#pragma unroll
                    for (int j = 0; j < J; j++)
                        if (8 * p + g >= here || 4 * j + t >= n) d[p][j] = 0.f;   // rows that are not there may hold anything
                        else if (!alive) d[p][j] = NAN;                           // gave up: nothing that could pass for a result
            }
            // Behind the last channel dz is zero, or NaN in a row that is NaN throughout: as good for dx, and in columns of dW that nobody reads.
            if (a.shares) {
#pragma unroll
                for (int p = 0; p < 4; p++)
#pragma unroll
                    for (int j = 0; j < J; j++)
                        sts(dz_at + (p * NB + j / 2) * MIX_DZ_BLOCK + (4 * (4 * (j & 1) + t) + (g & 3)) * 8 + 4 * (g >> 2), d[p][j]);
            }
            if (a.dresidual) {
#pragma unroll
                for (int j = 0; j < J; j++)
#pragma unroll
                    for (int p = 0; p < 4; p++) {   // (where this lane has read)
                        const u32 at = g_row + (8 * p * n + 4 * j) * sizeof(T);
                        if (j < FULL) sts_value<T>(at, a.scale * d[p][j]);
                        else sts_value_if<T>(4 * j + t < n, at, a.scale * d[p][j]);
                    }
            }
            if constexpr (PACKED) {
                __syncwarp();
                if (a.want_x) decode(work, a.x, stage + at.x_at, heads_x, 3, k);
                if (a.want_x2) decode(work2, a.x2, stage + at.x2_at, heads_x2, 3, k2);
            }
            __syncwarp();
            const u32 x_at = PACKED ? shared_address(work) : shared_address(stage + at.x_at) + r0 * k * sizeof(T);
            const u32 x2_at = PACKED ? shared_address(work2) : shared_address(stage + at.x2_at) + r0 * k2 * sizeof(T);
            if (a.shares) {
                // dW in blocks of eight channels of x, then of x2: channels behind the last give rows of dW that nobody reads.  32 rows'
                // products by themselves, then added to the sums as floats are: the tensor cores cut what they add to, and a sum over
                // many rows would drift.  (Eight rows' where there are too few registers.)
                constexpr bool LONG = MB * NB <= 9;
                float part[LONG ? MB : 1][NB][4];
                if constexpr (LONG) {
#pragma unroll
                    for (int i = 0; i < MB; i++)
#pragma unroll
                        for (int j = 0; j < NB; j++)
#pragma unroll
                            for (int e = 0; e < 4; e++) part[i][j][e] = 0.f;
                }
                u32 from[2 * MB];
#pragma unroll
                for (int i = 0; i < 2 * MB; i++) {
                    const bool second = 8 * i >= kp && 8 * i < all_p;
                    from[i] = second ? x2_at + (t * k2 + g + 8 * i - kp) * sizeof(TX) : x_at + (t * k + g + (8 * i < kp ? 8 * i : 0)) * sizeof(TX);
                }
                u32 dz_from = dz_at + lane * 8;
#pragma unroll (LONG ? 4 : 1)
                for (int r = 0; r < 32; r += 8, dz_from += NB * MIX_DZ_BLOCK) {
                    u32 b_hi[NB][2], b_lo[NB][2];
#pragma unroll
                    for (int j = 0; j < NB; j++) {
                        const uint2 b = lds2(dz_from + MIX_DZ_BLOCK * j);
                        split(__uint_as_float(b.x), b_hi[j][0], b_lo[j][0]);
                        split(__uint_as_float(b.y), b_hi[j][1], b_lo[j][1]);
                        if (a.bias) sums[j] += __uint_as_float(b.x) + __uint_as_float(b.y);
                    }
#pragma unroll
                    for (int i = 0; i < MB; i++) {
                        u32 a_hi[4], a_lo[4];
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            const bool second = 8 * (2 * i + h) >= kp && 8 * (2 * i + h) < all_p;
                            const u32 four = (second ? k2 : k) * 4 * (u32)sizeof(TX);
                            u32& p = from[2 * i + h];
                            const float v0 = lds_value<TX>(p), v1 = lds_value<TX>(p + four);
                            p += 2 * four;
                            if (split_x) {
                                split(v0, a_hi[h], a_lo[h]);
                                split(v1, a_hi[2 + h], a_lo[2 + h]);
                            } else {
                                a_hi[h] = __float_as_uint(v0), a_hi[2 + h] = __float_as_uint(v1);
                            }
                        }
                        float (&to)[NB][4] = part[LONG ? i : 0];
#pragma unroll
                        for (int j = 0; j < NB; j++) {
                            if constexpr (LONG) mma8(to[j], a_hi, b_hi[j]);
                            else mma8_first(to[j], a_hi, b_hi[j]);
                        }
#pragma unroll
                        for (int j = 0; j < NB; j++) mma8(to[j], a_hi, b_lo[j]);
                        if (split_x) {
#pragma unroll
                            for (int j = 0; j < NB; j++) mma8(to[j], a_lo, b_hi[j]);
                        }
                        if constexpr (!LONG) {
#pragma unroll
                            for (int j = 0; j < NB; j++)
#pragma unroll
                                for (int e = 0; e < 4; e++) acc[i][j][e] += to[j][e];
                        }
                    }
                }
                if constexpr (LONG) {
#pragma unroll
                    for (int i = 0; i < MB; i++)
#pragma unroll
                        for (int j = 0; j < NB; j++)
#pragma unroll
                            for (int e = 0; e < 4; e++) acc[i][j][e] += part[i][j][e];
                }
                __syncwarp();   // x has been read: dx may take its place
            }
            // dx and dx2, CH blocks of eight channels at a time, to where x and x2 were
            if (a.dx || a.dx2) {
                constexpr int CH = MB == 3 ? 3 : MB == 1 ? 2 : 5;
                const int blocks = all_p / 8;
#pragma unroll 1
                for (int c0 = a.dx ? 0 : kp / 8; c0 < (a.dx2 ? blocks : kp / 8); c0 += CH) {
                    float part[2][CH][4];
#pragma unroll
                    for (int q = 0; q < NB; q++) {
                        u32 a_hi[2][4], a_lo[2][4], b_hi[CH][2], b_lo[CH][2];
#pragma unroll
                        for (int m = 0; m < 2; m++)
#pragma unroll
                            for (int e = 0; e < 4; e++) split(d[2 * m + (e & 1)][2 * q + (e >> 1)], a_hi[m][e], a_lo[m][e]);
#pragma unroll
                        for (int j = 0; j < CH; j++) {   // (behind the last block: that block again, and results that nobody keeps)
                            const uint4 b = lds4(w_at + (min(c0 + j, blocks - 1) * NB + q) * MIX_BLOCK + lane * 16);
                            b_hi[j][0] = b.x, b_hi[j][1] = b.y, b_lo[j][0] = b.z, b_lo[j][1] = b.w;
                        }
#pragma unroll
                        for (int j = 0; j < CH; j++)
#pragma unroll
                            for (int m = 0; m < 2; m++) {
                                if (q == 0) mma8_first(part[m][j], a_hi[m], b_hi[j]);
                                else mma8(part[m][j], a_hi[m], b_hi[j]);
                            }
#pragma unroll
                        for (int j = 0; j < CH; j++)
#pragma unroll
                            for (int m = 0; m < 2; m++) mma8(part[m][j], a_lo[m], b_hi[j]);
                        if (split_w) {
#pragma unroll
                            for (int j = 0; j < CH; j++)
#pragma unroll
                                for (int m = 0; m < 2; m++) mma8(part[m][j], a_hi[m], b_lo[j]);
                        }
                    }
#pragma unroll
                    for (int j = 0; j < CH; j++) {
                        const bool second = c0 + j >= kp / 8;
                        const int width = second ? k2 : k, c = 8 * (c0 + j) - (second ? kp : 0) + 2 * t;
                        if (c0 + j >= blocks || !(second ? a.dx2 : a.dx)) continue;
                        const u32 to = (second ? x2_at : x_at) + (g * width + c) * sizeof(T);
#pragma unroll
                        for (int e = 0; e < 2; e++)
#pragma unroll
                            for (int m = 0; m < 4; m++)
                                sts_value_if<T>(c + e < width, to + (8 * m * width + e) * sizeof(T), part[m / 2][j][2 * (m & 1) + e]);
                    }
                }
            }
            fence_async_proxy();
            __syncwarp();
            const bool bulk = bulk_out && here == 32;
            const long long row0 = tile0 + r0;
            const T* dx_s = PACKED ? reinterpret_cast<T*>(work) : reinterpret_cast<T*>(stage + at.x_at) + r0 * k;
            const T* dx2_s = PACKED ? reinterpret_cast<T*>(work2) : reinterpret_cast<T*>(stage + at.x2_at) + r0 * k2;
            if (a.dresidual) copy_out(static_cast<T*>(a.dresidual) + row0 * n, reinterpret_cast<T*>(stage) + r0 * n, here * n, bulk);
            if (a.dx) copy_out(static_cast<T*>(a.dx) + row0 * k, dx_s, here * k, bulk);
            if (a.dx2) copy_out(static_cast<T*>(a.dx2) + row0 * k2, dx2_s, here * k2, bulk);
            if (lane == 0) bulk_commit();
            if (lane == 0 && (PACKED || r0 + 32 >= rows_here)) bulk_wait_read();   // (work rows are written again by the next block)
            __syncwarp();
        }
        if (alive) fetch(tile + stages * step, s);
        if (++s == stages) s = 0, parity ^= 1;
    }
    if (!alive)   // gave up once: no copy may be in flight when the CTA goes on
        for (int i = 0; i < stages; i++) mbar_wait(&bars[i], 0), mbar_wait(&bars[i], 1);

    // the CTA's share of dW and dbias: the warps' sums through shared memory, in place of all that was there
    if (!a.shares) return;
    constexpr int PER = MB * 16 * NB * 8 + NB * 8;
    float* mine = reinterpret_cast<float*>(smem + at.weights);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < MB; i++)
#pragma unroll
        for (int j = 0; j < NB; j++)
#pragma unroll
            for (int e = 0; e < 4; e++)
                mine[warp * PER + (16 * i + g + (e & 2 ? 8 : 0)) * 8 * NB + 8 * j + 2 * t + (e & 1)] = acc[i][j][e];
#pragma unroll
    for (int j = 0; j < NB; j++) {
        float v = sums[j];
        v += __shfl_xor_sync(~0u, v, 1);
        v += __shfl_xor_sync(~0u, v, 2);
        if (t == 0) mine[warp * PER + MB * 16 * 8 * NB + 8 * j + g] = v;
    }
    __syncthreads();
    const int count = (k + k2 + 1) * n;
    float* share = a.shares + (size_t)blockIdx.x * count;
    for (int i = threadIdx.x; i < count; i += blockDim.x) {
        const int r = i / n, c = i - r * n, from = (r < k ? r : r < k + k2 ? r - k + kp : MB * 16) * 8 * NB + c;
        float v = 0.f;
        for (int w = 0; w < warps; w++) v += mine[w * PER + from];
        share[i] = v;
    }
}
// Shared memory that the sum of the shares takes, from the weights on.
__host__ __device__ constexpr size_t mix_share_bytes(int warps, int mb, int nb) {
    return up16(sizeof(u64) * MIX_WARPS * MIX_STAGES) + sizeof(float) * (size_t)warps * (mb * 16 * nb * 8 + nb * 8);
}

// Sums of the CTAs' shares, in double, in the order of the CTAs: eight threads an element.
template <typename W>
__global__ void __launch_bounds__(256)
mix_add_shares(const float* __restrict__ shares, int ctas, int k, int k2, int n, W* __restrict__ dw, W* __restrict__ dw2, W* __restrict__ db) {
    __shared__ double part[8][32];
    const int count = (k + k2 + 1) * n, i = blockIdx.x * 32 + (threadIdx.x & 31), slice = threadIdx.x >> 5;
    double sum = 0.0;
    if (i < count)
        for (int c = slice; c < ctas; c += 8) sum += (double)shares[(size_t)c * count + i];
    part[slice][threadIdx.x & 31] = sum;
    __syncthreads();
    if (slice || i >= count) return;
    for (int q = 1; q < 8; q++) sum += part[q][threadIdx.x];
    W* to = i < k * n ? (dw ? dw + i : nullptr) : i < (k + k2) * n ? (dw2 ? dw2 + (i - k * n) : nullptr) : (db ? db + (i - (k + k2) * n) : nullptr);
    if (to) *to = from_float<W>((float)sum);
}

// ---------------------------------------------------------------------------------------------
// The wide way
// ---------------------------------------------------------------------------------------------
// dz of every row, a warp a row.
template <typename T>
__global__ void __launch_bounds__(256) mix_dz(MixBackArgs a) {
    const int lane = threadIdx.x & 31, n = a.n;
    const T* grad = static_cast<const T*>(a.grad);
    const T* out = static_cast<const T*>(a.out.full);
    for (long long row = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); row < a.rows; row += (long long)gridDim.x * 8) {
        float y[4], g[4], s = 0.f;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int c = lane + 32 * j;
            const long long i = row * n + c;
            g[j] = c < n ? to_float(grad[i]) : 0.f;
            y[j] = 0.f;
            if (c < n && a.activation != PL_ACT_NONE)
                y[j] = a.out.codes ? decode_value(a.out.codes[i], (u32)(u16)a.out.scales[i / PACK_BLOCK]) : to_float(out[i]);
            s = fmaf(y[j], g[j], s);
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
        if (a.activation == PL_ACT_SOFTMAX && !__any_sync(~0u, y[0] != 0.f || y[1] != 0.f || y[2] != 0.f || y[3] != 0.f))
            s = g[0] = g[1] = g[2] = g[3] = 0.f;   // a row of zeros has no gradient (see mix_backward)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int c = lane + 32 * j;
            if (c >= n) continue;
            const float dz = a.activation == PL_ACT_SOFTMAX ? y[j] * (g[j] - s) : a.activation == PL_ACT_RELU ? relu_gradient(y[j], g[j]) : g[j];
            a.dz[row * n + c] = dz;
            if (a.dresidual) static_cast<T*>(a.dresidual)[row * n + c] = from_float<T>(a.scale * dz);
        }
    }
}

// dW of one input (blockIdx.y: x or x2) and, with the first, dbias: a CTA's eight warps each sum blocks of 64 x 32 of it over all the
// CTA's rows, 32 rows at a time through shared memory; the next 32 are on their way in registers meanwhile.  154 401 rows of 128 + 128 x
// 128: 329 us, the tensor cores busy a third of them (110 us is their floor); 680 with loads and products in turn.
constexpr int WIDE_ROWS = 32, WIDE_DS = MIX_MOST + 8;   // (rows of 136 floats: 4 rows by 8 channels in 32 banks)
constexpr size_t WIDE_SMEM = sizeof(float) * 2 * 2 * WIDE_ROWS * WIDE_DS;
template <typename T>
__global__ void __launch_bounds__(256, 1) mix_backward_weights(MixBackArgs a) {
    extern __shared__ __align__(16) float wide_s[];   // [2][dz, x][32][WIDE_DS]
    const bool second = blockIdx.y != 0;
    const int n = a.n, k = second ? a.k2 : a.k, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int m0 = 64 * (warp & 1), c0 = 32 * (warp >> 1);
    const bool want = second ? a.want_x2 != 0 : a.want_x != 0;
    const Kept& from = second ? a.x2 : a.x;
    const bool split_x = sizeof(T) == 4 && !from.codes;
    const bool works = c0 < n && (m0 == 0 || m0 < k);   // (the first half of the rows of dW sums dbias, too)
    float acc[4][4][4], sums[4];
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            sums[j] = 0.f;
#pragma unroll
            for (int e = 0; e < 4; e++) acc[i][j][e] = 0.f;
        }
    const long long tiles = (a.rows + WIDE_ROWS - 1) / WIDE_ROWS;
    const int c = threadIdx.x & 127, r_first = threadIdx.x >> 7;   // this thread's channel, and the first of its rows: every second
    // In 8 bits, rows of whole words: four channels at a time, of every eighth row.
    const bool words = from.codes && k % 4 == 0 && (reinterpret_cast<uintptr_t>(from.codes) & 3) == 0;
    float next_d[16], next_x[16];
    u32 next_c[4], next_h[4];
    auto fetch = [&](long long tile) {
        const long long row0 = tile * WIDE_ROWS + r_first;
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const long long row = row0 + 2 * i;
            const bool there = row < a.rows;
            next_d[i] = there && c < n ? a.dz[row * n + c] : 0.f;
            next_x[i] = 0.f;
            if (!words && there && want && c < k) {
                const long long at = row * k + c;
                next_x[i] = from.codes ? decode_value(from.codes[at], (u32)(u16)from.scales[at / PACK_BLOCK]) : to_float(static_cast<const T*>(from.full)[at]);
            }
        }
        if (words) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const long long row = tile * WIDE_ROWS + warp + 8 * i, at = row * k + 4 * lane;
                const bool there = row < a.rows && want && 4 * lane < k;
                next_c[i] = there ? *reinterpret_cast<const u32*>(from.codes + at) : 0;
                next_h[i] = there ? (u32)(u16)from.scales[at / PACK_BLOCK] : 1;
            }
        }
    };
    fetch(blockIdx.x);
    int buffer = 0;
    for (long long tile = blockIdx.x; tile < tiles; tile += gridDim.x, buffer ^= 1) {
        float* dz_s = wide_s + buffer * 2 * WIDE_ROWS * WIDE_DS;
        float* x_s = dz_s + WIDE_ROWS * WIDE_DS;
#pragma unroll
        for (int i = 0; i < 16; i++) {
            dz_s[(r_first + 2 * i) * WIDE_DS + c] = next_d[i];
            if (!words) x_s[(r_first + 2 * i) * WIDE_DS + c] = next_x[i];
        }
        if (words) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                float v[4];
                decode4(v, next_c[i], next_h[i]);
                store4(x_s + (warp + 8 * i) * WIDE_DS + 4 * lane, v);
            }
        }
        __syncthreads();   // (nobody writes this buffer again before everybody has passed the next barrier)
        fetch(tile + gridDim.x);
        if (!works) continue;
        u32 d_at = shared_address(dz_s) + (t * WIDE_DS + c0 + g) * 4, x_at = shared_address(x_s) + (t * WIDE_DS + m0 + g) * 4;
#pragma unroll 1
        for (int r = 0; r < WIDE_ROWS; r += 8, d_at += 8 * WIDE_DS * 4, x_at += 8 * WIDE_DS * 4) {
            u32 b_hi[4][2], b_lo[4][2];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float v0 = lds(d_at + 32 * j), v1 = lds(d_at + 4 * WIDE_DS * 4 + 32 * j);
                sums[j] += v0 + v1;
                split(v0, b_hi[j][0], b_lo[j][0]);
                split(v1, b_hi[j][1], b_lo[j][1]);
            }
            if (!want) continue;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                if (m0 + 16 * i >= k) break;
                u32 a_hi[4], a_lo[4];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float v = lds(x_at + (e & 2 ? 4 : 0) * WIDE_DS * 4 + 64 * i + (e & 1 ? 32 : 0));
                    if (split_x) split(v, a_hi[e], a_lo[e]);
                    else a_hi[e] = __float_as_uint(v);
                }
                float part[4][4];
#pragma unroll
                for (int j = 0; j < 4; j++) mma8_first(part[j], a_hi, b_hi[j]);
#pragma unroll
                for (int j = 0; j < 4; j++) mma8(part[j], a_hi, b_lo[j]);
                if (split_x) {
#pragma unroll
                    for (int j = 0; j < 4; j++) mma8(part[j], a_lo, b_hi[j]);
                }
#pragma unroll
                for (int j = 0; j < 4; j++)
#pragma unroll
                    for (int e = 0; e < 4; e++) acc[i][j][e] += part[j][e];   // (see mix_backward)
            }
        }
    }
    const int count = (a.k + a.k2 + 1) * n;
    float* share = a.shares + (size_t)blockIdx.x * count;
    float* rows = share + (second ? a.k * n : 0);
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int row = m0 + 16 * i + g + (e & 2 ? 8 : 0), col = c0 + 8 * j + 2 * t + (e & 1);
                if (row < k && col < n) rows[row * n + col] = acc[i][j][e];
            }
    if (second || m0) return;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        float v = sums[j];
        v += __shfl_xor_sync(~0u, v, 1);
        v += __shfl_xor_sync(~0u, v, 2);
        const int col = c0 + 8 * j + g;
        if (t == 0 && col < n) share[(size_t)(a.k + a.k2) * n + col] = v;
    }
}

}  // namespace pl
