// The gradients of act(x W [+ x2 W2] + ...): dz from the upstream gradient and the output, dx = dz W^T, dW = x^T dz.
//
// mix_backward (up to 80 input and 32 output channels): everything in one pass over memory.  A consumer warp takes 32 rows:
// dz in registers and to shared memory, its share of dW into registers that last for the whole kernel, dx into the place
// where x came in, and bulk copies out.  At the end a CTA's warps add their shares of dW up, mix_add_shares those of the
// CTAs, in double and in a fixed order.
//
// Beyond that dW does not fit a warp's registers: mix_dz writes dz to the workspace, mix_forward multiplies it by the
// transposed weights, mix_backward_weights gives a CTA's warps blocks of dW to sum over all its rows.
#pragma once
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
    float* dz;                         // the wide way: [rows][n]
    int want_x, want_x2, stages;       // want: its product with dz
};

// Rows of dz and of W^T in shared memory: 8 rows by 4 columns in 32 banks.
__host__ __device__ constexpr int mix_dz_stride(int nt) { return 8 * nt + 4; }

// What a consumer warp's 32 rows take of a stage and of its own memory, in bytes.
struct MixBackSmem {
    size_t weights, own, stage0;
    size_t dz, work, own_bytes;                          // of a warp: dz, then x and x2 as floats
    size_t y_at, ys_at, x_at, xs_at, x2_at, x2s_at, stage_bytes;   // of a stage: the gradient first
    __host__ __device__ MixBackSmem(int warps, int k, int k2, int n, int nb, int size /* of a value */, bool work_rows, bool y, bool y_packed,
                                    bool x, bool x_packed, bool x2, bool x2_packed) {
        const size_t tp = 32 * warps;
        weights = 128;
        own = up16(weights + sizeof(float) * (size_t)(up8(k) + up8(k2)) * mix_dz_stride(nb));
        dz = 0;
        work = up16(sizeof(float) * 32 * mix_dz_stride(nb));
        own_bytes = work + (work_rows ? sizeof(float) * 32 * (size_t)(k + k2) : 0);
        stage0 = own + own_bytes * warps;
        auto room = [&](bool there, bool packed, size_t c) { return !there ? (size_t)0 : up16(packed ? tp * c : tp * c * size); };
        auto heads = [&](bool there, bool packed, size_t c) { return there && packed ? up16(2 * tp * c / PACK_BLOCK) : (size_t)0; };
        y_at = up16(tp * n * size);
        ys_at = y_at + room(y, y_packed, n);
        x_at = ys_at + heads(y, y_packed, n);
        // without work rows dx leaves from where x came in, or would have
        xs_at = x_at + room(x || !work_rows, x_packed && work_rows, k);
        x2_at = xs_at + heads(x, x_packed, k);
        x2s_at = x2_at + room((x2 || !work_rows) && k2, x2_packed && work_rows, k2);
        stage_bytes = up16(x2s_at + heads(x2, x2_packed, k2));
    }
    __host__ __device__ size_t bytes(int stages) const { return stage0 + stage_bytes * stages; }
};
__host__ __device__ inline MixBackSmem mix_back_smem(const MixBackArgs& a, int warps, int nb, int size, bool work) {
    return MixBackSmem(warps, a.k, a.k2, a.n, nb, size, work, a.activation != PL_ACT_NONE, a.out.codes != nullptr, a.want_x != 0,
                       a.x.codes != nullptr, a.want_x2 != 0, a.x2.codes != nullptr);
}

// WORK: x or x2 comes in 8 bits; both are then multiplied from floats of the warp's own memory.
template <typename T, bool WORK, int MB, int NB>
__global__ void __launch_bounds__(160, MB * NB > 12 ? 2 : 3) mix_backward(MixBackArgs a) {
    extern __shared__ __align__(128) unsigned char smem[];
    const int warps = (int)blockDim.x / 32 - 1, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int tp = 32 * warps, k = a.k, k2 = a.k2, n = a.n, stages = a.stages;
    const MixBackSmem at = mix_back_smem(a, warps, NB, sizeof(T), WORK);
    const bool reads_y = a.activation != PL_ACT_NONE, y_packed = a.out.codes != nullptr;
    u64* full = reinterpret_cast<u64*>(smem);
    u64* empty = full + MIX_STAGES;
    float* w_s = reinterpret_cast<float*>(smem + at.weights);
    if (threadIdx.x == 0)
        for (int s = 0; s < stages; s++) {
            mbar_init(&full[s], 32);
            mbar_init(&empty[s], warps);
        }
    __syncthreads();
    const long long tiles = (a.rows + tp - 1) / tp;
    const T* grad = static_cast<const T*>(a.grad);

    if (warp == warps) {   // the producer
        int s = 0, round = 0;
        for (long long tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
            if (round && !mbar_wait(&empty[s], (round - 1) & 1)) break;
            unsigned char* stage = smem + at.stage0 + at.stage_bytes * s;
            const long long row0 = tile * tp;
            const int here = (int)min((long long)tp, a.rows - row0);
            const bool whole = here == tp;
            unsigned bytes = 0;
            const void* from[4];
            unsigned char* to[4];
            unsigned size[4];
            int copies = 0;
            auto values_in = [&](size_t place, const T* p, int c) {
                p += row0 * c;
                if (whole && aligned16(p)) {
                    from[copies] = p, to[copies] = stage + place, size[copies] = (unsigned)(tp * c * sizeof(T));
                    bytes += size[copies++];
                } else {
                    copy_in<sizeof(T)>(stage + place, p, here * c);
                }
            };
            auto codes_in = [&](size_t place, size_t heads_place, const Kept& p, int c) {
                const uint8_t* q = p.codes + row0 * c;
                if (whole && aligned16(q)) {
                    from[copies] = q, to[copies] = stage + place, size[copies] = (unsigned)(tp * c);
                    bytes += size[copies++];
                } else {
                    copy_in<1>(stage + place, q, here * c);
                }
                copy_in<2>(stage + heads_place, p.scales + row0 * c / PACK_BLOCK, (here * c + PACK_BLOCK - 1) / PACK_BLOCK);
            };
            auto kept_in = [&](size_t place, size_t heads_place, const Kept& p, int c) {
                if (p.codes) codes_in(place, heads_place, p, c);
                else values_in(place, static_cast<const T*>(p.full), c);
            };
            values_in(0, grad, n);
            if (reads_y) kept_in(at.y_at, at.ys_at, a.out, n);
            if (a.want_x) kept_in(at.x_at, at.xs_at, a.x, k);
            if (a.want_x2) kept_in(at.x2_at, at.x2s_at, a.x2, k2);
            if (!whole) {   // rows that are not there: their dz is zero, their x must not be NaN
                auto zero = [&](size_t place, bool packed, int c) {
                    if (packed) return;   // (the decoding writes zeros)
                    T* p = reinterpret_cast<T*>(stage + place);
                    for (int i = here * c + lane; i < tp * c; i += 32) p[i] = from_float<T>(0.f);
                };
                if (a.want_x) zero(at.x_at, a.x.codes != nullptr, k);
                if (a.want_x2) zero(at.x2_at, a.x2.codes != nullptr, k2);
            }
            cp_async_wait_all();
            if (lane == 0 && bytes) {
                mbar_expect_tx(&full[s], bytes);   // (lane 0's arrival)
                for (int i = 0; i < copies; i++) bulk_load(to[i], from[i], size[i], &full[s]);
            } else {
                mbar_arrive(&full[s]);
            }
            if (++s == stages) s = 0, round++;
        }
        return;
    }

    // W^T: a row an input channel, zeros behind the last channel of either side
    constexpr int DS = mix_dz_stride(NB);
    const int kp = up8(k), threads = 32 * warps;
    for (int i = threadIdx.x; i < (kp + up8(k2)) * DS; i += threads) {
        const int r = i / DS, c = i - r * DS;
        const bool second = r >= kp;
        const int j = second ? r - kp : r;
        const void* w = second ? a.weight2 : a.weight;
        w_s[i] = c < n && j < (second ? k2 : k) && w ? load_weight(w, j * n + c, a.weight_dtype) : 0.f;
    }
    asm volatile("bar.sync 1, %0;" ::"r"(threads) : "memory");

    const int g = lane >> 2, t = lane & 3, r0 = 32 * warp;
    const bool split_w = a.weight_dtype == PL_F32;
    // 8-bit codes times a power of two need no second term, nor do 16 bits
    const bool split_x = sizeof(T) == 4 && !(WORK && (!a.want_x || a.x.codes) && (!a.want_x2 || a.x2.codes));
    const bool bulk_x = a.dx && aligned16(a.dx), bulk_x2 = a.dx2 && aligned16(a.dx2), bulk_r = a.dresidual && aligned16(a.dresidual);
    unsigned char* own = smem + at.own + at.own_bytes * warp;
    float* dz_s = reinterpret_cast<float*>(own + at.dz);      // [32][DS]
    float* work = reinterpret_cast<float*>(own + at.work);    // [32][k], [32][k2]
    float acc[MB][NB][4], sums[NB];
#pragma unroll
    for (int i = 0; i < MB; i++)
#pragma unroll
        for (int j = 0; j < NB; j++)
#pragma unroll
            for (int e = 0; e < 4; e++) acc[i][j][e] = 0.f;
#pragma unroll
    for (int j = 0; j < NB; j++) sums[j] = 0.f;

    int s = 0, parity = 0;
    for (long long tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
        unsigned char* stage = smem + at.stage0 + at.stage_bytes * s;
        const bool arrived = mbar_wait(&full[s], parity);
        const long long row0 = tile * tp + r0;
        const int here = (int)max(0ll, min(32ll, a.rows - row0));
        if (here > 0) {
            T* g_s = reinterpret_cast<T*>(stage) + r0 * n;
            // dz: four lanes a row, each every fourth channel, from another one on in every row so that banks differ
            constexpr int J = 2 * NB;
            const T* y_s = reinterpret_cast<const T*>(stage + at.y_at) + r0 * n;
            const uint8_t* yc_s = stage + at.y_at + r0 * n;
            const int16_t* ys_s = reinterpret_cast<const int16_t*>(stage + at.ys_at) + warp * n;   // 32 rows: n blocks
#pragma unroll
            for (int p = 0; p < 4; p++) {
                const int row = 8 * p + g;
                float y[J], d[J], sum = 0.f;
#pragma unroll
                for (int j = 0; j < J; j++) {
                    const int c = 4 * ((j + g) % J) + t, i = row * n + c;
                    const bool there = c < n && row < here;
                    d[j] = there ? to_float(g_s[i]) : 0.f;
                    y[j] = 0.f;
                    if (there && reads_y) y[j] = y_packed ? decode_value(yc_s[i], (u32)(u16)ys_s[i >> 5]) : to_float(y_s[i]);
                    sum = fmaf(y[j], d[j], sum);
                }
                if (a.activation == PL_ACT_SOFTMAX) {
                    sum += __shfl_xor_sync(~0u, sum, 1);
                    sum += __shfl_xor_sync(~0u, sum, 2);
                }
#pragma unroll
                for (int j = 0; j < J; j++) {
                    const int c = 4 * ((j + g) % J) + t;
                    float z = a.activation == PL_ACT_SOFTMAX ? y[j] * (d[j] - sum) : a.activation == PL_ACT_RELU ? (y[j] > 0.f ? d[j] : 0.f) : d[j];
                    if (!arrived) z = NAN;   // gave up: nothing that could pass for a result
                    if (c >= n || row >= here) z = 0.f;
                    dz_s[row * DS + c] = z;
                    if (a.dresidual && c < n) g_s[row * n + c] = from_float<T>(a.scale * z);
                }
            }
            const T* x_s = reinterpret_cast<const T*>(stage + at.x_at) + r0 * k;
            const T* x2_s = reinterpret_cast<const T*>(stage + at.x2_at) + r0 * k2;
            if constexpr (WORK) {
                auto decode = [&](float* to, const Kept& from, size_t place, size_t heads_place, int c) {
                    const int count = here * c;
                    const uint8_t* codes = stage + place + r0 * c;
                    const int16_t* heads = reinterpret_cast<const int16_t*>(stage + heads_place) + warp * c;
                    const T* values = reinterpret_cast<const T*>(stage + place) + r0 * c;
                    for (int i = 4 * lane; i < 32 * c; i += 128) {
                        float v[4];
                        if (from.codes) {
                            decode4(v, *reinterpret_cast<const u32*>(codes + i), (u32)(u16)heads[min(i, count - 1) >> 5]);
#pragma unroll
                            for (int e = 0; e < 4; e++)
                                if (i + e >= count) v[e] = 0.f;
                        } else {
                            load4(v, values + i);
                        }
                        store4(to + i, v);
                    }
                };
                if (a.want_x) decode(work, a.x, at.x_at, at.xs_at, k);
                if (a.want_x2) decode(work + 32 * k, a.x2, at.x2_at, at.x2s_at, k2);
            }
            __syncwarp();
            if (a.shares) {
                for (int r = 0; r < 32; r += 8) {
                    u32 b_hi[NB][2], b_lo[NB][2];
#pragma unroll
                    for (int j = 0; j < NB; j++) {
                        const float v0 = dz_s[(r + t) * DS + 8 * j + g], v1 = dz_s[(r + t + 4) * DS + 8 * j + g];
                        sums[j] += v0 + v1;
                        split(v0, b_hi[j][0], b_lo[j][0]);
                        split(v1, b_hi[j][1], b_lo[j][1]);
                    }
#pragma unroll
                    for (int i = 0; i < MB; i++) {
                        u32 a_hi[4], a_lo[4];
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const int c = 16 * i + g + (e & 1 ? 8 : 0), row = r + t + (e & 2 ? 4 : 0);
                            float v = 0.f;
                            if (c < k) {
                                if (a.want_x) v = WORK ? work[row * k + c] : to_float(x_s[row * k + c]);
                            } else if (c < k + k2) {
                                if (a.want_x2) v = WORK ? work[32 * k + row * k2 + c - k] : to_float(x2_s[row * k2 + c - k]);
                            }
                            split(v, a_hi[e], a_lo[e]);
                        }
                        // Eight rows' products by themselves, then added to the sums as floats are: the tensor cores cut what they
                        // add to, and a sum over many rows would drift.
                        float part[NB][4];
#pragma unroll
                        for (int j = 0; j < NB; j++)
#pragma unroll
                            for (int e = 0; e < 4; e++) part[j][e] = 0.f;
                        if (split_x) {
#pragma unroll
                            for (int j = 0; j < NB; j++) mma8(part[j], a_lo, b_hi[j]);
                        }
#pragma unroll
                        for (int j = 0; j < NB; j++) mma8(part[j], a_hi, b_lo[j]);
#pragma unroll
                        for (int j = 0; j < NB; j++) mma8(part[j], a_hi, b_hi[j]);
#pragma unroll
                        for (int j = 0; j < NB; j++)
#pragma unroll
                            for (int e = 0; e < 4; e++) acc[i][j][e] += part[j][e];
                    }
                }
            }
            __syncwarp();   // x has been read: dx may take its place
            auto product = [&](T* to, const float* w, int c_count) {
                for (int c0 = 0; c0 < c_count; c0 += 24) {
                    float part[2][3][4];
#pragma unroll
                    for (int m = 0; m < 2; m++)
#pragma unroll
                        for (int j = 0; j < 3; j++)
#pragma unroll
                            for (int e = 0; e < 4; e++) part[m][j][e] = 0.f;
#pragma unroll
                    for (int q = 0; q < NB; q++) {
                        u32 a_hi[2][4], a_lo[2][4];
#pragma unroll
                        for (int m = 0; m < 2; m++)
#pragma unroll
                            for (int e = 0; e < 4; e++)
                                split(dz_s[(16 * m + g + (e & 1 ? 8 : 0)) * DS + 8 * q + t + (e & 2 ? 4 : 0)], a_hi[m][e], a_lo[m][e]);
                        u32 b_hi[3][2], b_lo[3][2];
#pragma unroll
                        for (int j = 0; j < 3; j++) {
                            const bool there = c0 + 8 * j < c_count;   // rows behind belong to the second input, or to nobody
                            const float* wc = w + (size_t)(c0 + 8 * j + g) * DS + 8 * q + t;
                            split(there ? wc[0] : 0.f, b_hi[j][0], b_lo[j][0]);
                            split(there ? wc[4] : 0.f, b_hi[j][1], b_lo[j][1]);
                        }
#pragma unroll
                        for (int j = 0; j < 3; j++)
#pragma unroll
                            for (int m = 0; m < 2; m++) mma8(part[m][j], a_lo[m], b_hi[j]);
                        if (split_w) {
#pragma unroll
                            for (int j = 0; j < 3; j++)
#pragma unroll
                                for (int m = 0; m < 2; m++) mma8(part[m][j], a_hi[m], b_lo[j]);
                        }
#pragma unroll
                        for (int j = 0; j < 3; j++)
#pragma unroll
                            for (int m = 0; m < 2; m++) mma8(part[m][j], a_hi[m], b_hi[j]);
                    }
#pragma unroll
                    for (int m = 0; m < 2; m++)
#pragma unroll
                        for (int j = 0; j < 3; j++)
#pragma unroll
                            for (int e = 0; e < 4; e++) {
                                const int c = c0 + 8 * j + 2 * t + (e & 1), row = 16 * m + g + (e & 2 ? 8 : 0);
                                if (c < c_count) to[row * c_count + c] = from_float<T>(part[m][j][e]);
                            }
                }
            };
            T* dx_s = WORK ? reinterpret_cast<T*>(work) : const_cast<T*>(x_s);
            T* dx2_s = WORK ? reinterpret_cast<T*>(work + 32 * k) : const_cast<T*>(x2_s);
            if (a.dx) product(dx_s, w_s, k);
            if (a.dx2) product(dx2_s, w_s + (size_t)kp * DS, k2);
            fence_async_proxy();
            __syncwarp();
            const bool all = here == 32;
            if (a.dresidual) copy_out(static_cast<T*>(a.dresidual) + row0 * n, g_s, here * n, bulk_r && all);
            if (a.dx) copy_out(static_cast<T*>(a.dx) + row0 * k, dx_s, here * k, bulk_x && all);
            if (a.dx2) copy_out(static_cast<T*>(a.dx2) + row0 * k2, dx2_s, here * k2, bulk_x2 && all);
            if (lane == 0) {
                bulk_commit();
                bulk_wait_read();
            }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[s]);
        if (++s == stages) s = 0, parity ^= 1;
    }

    // the CTA's share of dW and dbias: the warps' sums through shared memory (dz's place and behind; every copy out has read its own)
    if (!a.shares) return;
    constexpr int PER = MB * 16 * NB * 8 + NB * 8;
    float* mine = reinterpret_cast<float*>(smem + at.weights);   // the weights are not needed any more, nor is what lies behind them
    asm volatile("bar.sync 1, %0;" ::"r"(threads) : "memory");
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
    asm volatile("bar.sync 1, %0;" ::"r"(threads) : "memory");
    const int count = (k + k2 + 1) * n;
    float* share = a.shares + (size_t)blockIdx.x * count;
    for (int i = threadIdx.x; i < count; i += threads) {
        const int r = i / n, c = i - r * n, from = (r < k + k2 ? r : MB * 16) * 8 * NB + c;
        float v = 0.f;
        for (int w = 0; w < warps; w++) v += mine[w * PER + from];
        share[i] = v;
    }
}
// Shared memory that the sum of the shares takes, from the weights on.
__host__ __device__ constexpr size_t mix_share_bytes(int warps, int mb, int nb) {
    return 128 + sizeof(float) * (size_t)warps * (mb * 16 * nb * 8 + nb * 8);
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
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int c = lane + 32 * j;
            if (c >= n) continue;
            const float dz = a.activation == PL_ACT_SOFTMAX ? y[j] * (g[j] - s) : a.activation == PL_ACT_RELU ? (y[j] > 0.f ? g[j] : 0.f) : g[j];
            a.dz[row * n + c] = dz;
            if (a.dresidual) static_cast<T*>(a.dresidual)[row * n + c] = from_float<T>(a.scale * dz);
        }
    }
}

// dW of one input (blockIdx.y: x or x2) and, with the first, dbias: a CTA's eight warps each sum blocks of 64 x 32 of it over all the
// CTA's rows, 32 rows at a time through shared memory.
constexpr int WIDE_ROWS = 32, WIDE_DS = MIX_MOST + 8, WIDE_XS = MIX_MOST + 8;
constexpr size_t WIDE_SMEM = sizeof(float) * WIDE_ROWS * (WIDE_DS + WIDE_XS);
template <typename T>
__global__ void __launch_bounds__(256) mix_backward_weights(MixBackArgs a) {
    extern __shared__ __align__(16) float wide_smem[];
    float* dz_s = wide_smem;                          // [32][WIDE_DS]
    float* x_s = dz_s + WIDE_ROWS * WIDE_DS;          // [32][WIDE_XS]
    const bool second = blockIdx.y != 0;
    const int n = a.n, k = second ? a.k2 : a.k, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int m0 = 64 * (warp & 1), c0 = 32 * (warp >> 1);
    const bool want = second ? a.want_x2 != 0 : a.want_x != 0;
    const Kept& from = second ? a.x2 : a.x;
    const bool split_x = sizeof(T) == 4 && !from.codes;
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
    for (long long tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
        __syncthreads();
        const long long row0 = tile * WIDE_ROWS;
        for (int r = warp; r < WIDE_ROWS; r += 8) {
            const bool there = row0 + r < a.rows;
            for (int c = lane; c < MIX_MOST; c += 32) {
                const long long i = (row0 + r) * n + c, ix = (row0 + r) * k + c;
                dz_s[r * WIDE_DS + c] = there && c < n ? a.dz[i] : 0.f;
                float v = 0.f;
                if (there && want && c < k)
                    v = from.codes ? decode_value(from.codes[ix], (u32)(u16)from.scales[ix / PACK_BLOCK]) : to_float(static_cast<const T*>(from.full)[ix]);
                x_s[r * WIDE_XS + c] = v;
            }
        }
        __syncthreads();
        if (c0 >= n || (m0 >= k && m0)) continue;   // (the first half of the rows of dW sums dbias, too)
        for (int r = 0; r < WIDE_ROWS; r += 8) {
            u32 b_hi[4][2], b_lo[4][2];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float v0 = dz_s[(r + t) * WIDE_DS + c0 + 8 * j + g], v1 = dz_s[(r + t + 4) * WIDE_DS + c0 + 8 * j + g];
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
                for (int e = 0; e < 4; e++)
                    split(x_s[(r + t + (e & 2 ? 4 : 0)) * WIDE_XS + m0 + 16 * i + g + (e & 1 ? 8 : 0)], a_hi[e], a_lo[e]);
                float part[4][4];
#pragma unroll
                for (int j = 0; j < 4; j++)
#pragma unroll
                    for (int e = 0; e < 4; e++) part[j][e] = 0.f;
                if (split_x) {
#pragma unroll
                    for (int j = 0; j < 4; j++) mma8(part[j], a_lo, b_hi[j]);
                }
#pragma unroll
                for (int j = 0; j < 4; j++) mma8(part[j], a_hi, b_lo[j]);
#pragma unroll
                for (int j = 0; j < 4; j++) mma8(part[j], a_hi, b_hi[j]);
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
                const int r = m0 + 16 * i + g + (e & 2 ? 8 : 0), c = c0 + 8 * j + 2 * t + (e & 1);
                if (r < k && c < n) rows[r * n + c] = acc[i][j][e];
            }
    if (second || m0) return;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        float v = sums[j];
        v += __shfl_xor_sync(~0u, v, 1);
        v += __shfl_xor_sync(~0u, v, 2);
        const int c = c0 + 8 * j + g;
        if (t == 0 && c < n) share[(size_t)(a.k + a.k2) * n + c] = v;
    }
}

}  // namespace pl
