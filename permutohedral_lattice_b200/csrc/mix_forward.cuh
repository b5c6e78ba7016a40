// out = act(x W [+ x2 W2] [+ bias] [+ s residual]) of rows of up to 128 channels.
//
// One pass over memory: a producer warp copies tiles of rows (contiguous in memory, whatever the number of channels) into
// stages of shared memory with bulk copies, consumer warps of 16 MT rows each multiply them by the weights, which stay in shared
// memory for all tiles of a CTA, finish the rows in registers (a row's logits lie in the registers of four lanes: the maximum
// and the sum of a softmax take two shuffles each) and send them out with a bulk copy from where the residual came in.  Warps
// work on rows of their own and meet nobody else at a tile.
#pragma once
#include "mix_common.cuh"

namespace pl {

struct MixArgs {
    long long rows;
    int k, k2, n, activation;
    float scale;                       // of the residual
    const void *x, *x2, *weight, *weight2, *bias, *residual;
    void* out;
    int weight_dtype, transposed;      // transposed: weight is [n][k] (no second input)
    int stages;
    uint8_t *x_codes, *x2_codes, *out_codes;
    int16_t *x_scales, *x2_scales, *out_scales;
};

__host__ __device__ constexpr int up8(int v) { return (v + 7) & ~7; }
__host__ __device__ constexpr size_t up16(size_t v) { return (v + 15) & ~(size_t)15; }
// Weight rows in shared memory: lanes read 4 rows by 8 columns, which have to lie in 32 banks.  Where a row is a multiple of 32
// floats, groups of 8 columns are exchanged by the row's number; else rows are 8 or 24 floats off that.
__host__ __device__ constexpr int mix_weight_stride(int nt) { return nt % 4 == 0 || nt % 2 == 1 ? 8 * nt : 8 * nt + 8; }
__host__ __device__ constexpr int mix_weight_at(int nt, int r, int c) {
    return r * mix_weight_stride(nt) + (nt % 4 == 0 ? c ^ ((r & 3) << 3) : c);
}

template <typename TI, typename TO>
struct MixSmem {   // byte offsets; a stage holds the rows of x, x2 and of the residual, in whose place the output leaves
    size_t weights, bias, stage0, x2_at, r_at, stage_bytes;
    __host__ __device__ MixSmem(int tp, int k, int k2, int n, int nt) {
        weights = 128;   // barriers before
        bias = weights + sizeof(float) * (size_t)(up8(k) + up8(k2)) * mix_weight_stride(nt);
        stage0 = up16(bias + sizeof(float) * 8 * nt);
        x2_at = up16(sizeof(TI) * (size_t)tp * k);
        r_at = x2_at + up16(sizeof(TI) * (size_t)tp * k2);
        stage_bytes = up16(r_at + (sizeof(TI) > sizeof(TO) ? sizeof(TI) : sizeof(TO)) * (size_t)tp * n);
    }
    __host__ __device__ size_t bytes(int stages) const { return stage0 + stage_bytes * stages; }
};
constexpr int MIX_STAGES = 4;   // at most

// acc += rows of `x` (k channels, from row r0 of the tile) times weight rows from w on.
template <typename TI, int NT, int MT>
__device__ __forceinline__ void mix_products(float (&acc)[MT][NT][4], const TI* x, int k, const float* w, int r0, bool split_w) {
    constexpr int WS = mix_weight_stride(NT), JG = NT < 4 ? NT : 4;   // (columns of one group of products)
    static_assert(NT % JG == 0);
    const int g = (threadIdx.x & 31) >> 2, t = threadIdx.x & 3;
    for (int kk = 0; kk < k; kk += 8) {
        u32 a_hi[MT][4], a_lo[MT][4];
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int c = kk + t + (i & 2 ? 4 : 0), r = r0 + 16 * m + g + (i & 1 ? 8 : 0);
                const float v = c < k ? to_float(x[r * k + c]) : 0.f;   // what lies behind is another row's, and may be NaN
                if constexpr (sizeof(TI) == 4) split(v, a_hi[m][i], a_lo[m][i]);
                else a_hi[m][i] = __float_as_uint(v);
            }
        const float* wk = w + (size_t)(kk + t) * WS + g;
#pragma unroll
        for (int j0 = 0; j0 < NT; j0 += JG) {
            u32 b_hi[JG][2], b_lo[JG][2];
#pragma unroll
            for (int j = 0; j < JG; j++) {
                const float* at = wk + 8 * (NT % 4 == 0 ? (j0 + j) ^ t : j0 + j);
                split(at[0], b_hi[j][0], b_lo[j][0]);
                split(at[4 * WS], b_hi[j][1], b_lo[j][1]);
            }
            if constexpr (sizeof(TI) == 4) {
#pragma unroll
                for (int j = 0; j < JG; j++)
#pragma unroll
                    for (int m = 0; m < MT; m++) mma8(acc[m][j0 + j], a_lo[m], b_hi[j]);
            }
            if (sizeof(TI) == 4 || split_w) {
#pragma unroll
                for (int j = 0; j < JG; j++)
#pragma unroll
                    for (int m = 0; m < MT; m++) mma8(acc[m][j0 + j], a_hi[m], b_lo[j]);
            }
#pragma unroll
            for (int j = 0; j < JG; j++)
#pragma unroll
                for (int m = 0; m < MT; m++) mma8(acc[m][j0 + j], a_hi[m], b_hi[j]);
        }
    }
}

template <typename TI, typename TO, int NT, int MT>
__global__ void __launch_bounds__(160) mix_forward(MixArgs a) {
    extern __shared__ __align__(128) unsigned char smem[];
    const int warps = (int)blockDim.x / 32 - 1, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int tp = 16 * MT * warps, k = a.k, k2 = a.k2, n = a.n, stages = a.stages;
    const MixSmem<TI, TO> at(tp, k, k2, n, NT);
    u64* full = reinterpret_cast<u64*>(smem);
    u64* empty = full + MIX_STAGES;
    float* w_s = reinterpret_cast<float*>(smem + at.weights);
    float* bias_s = reinterpret_cast<float*>(smem + at.bias);
    if (threadIdx.x == 0)
        for (int s = 0; s < stages; s++) {
            mbar_init(&full[s], 32);
            mbar_init(&empty[s], warps);
        }
    __syncthreads();
    const long long tiles = (a.rows + tp - 1) / tp;
    const TI* x = static_cast<const TI*>(a.x);
    const TI* x2 = static_cast<const TI*>(a.x2);
    const TI* residual = static_cast<const TI*>(a.residual);

    if (warp == warps) {   // the producer
        const bool bulk_x = aligned16(x), bulk_x2 = aligned16(x2), bulk_r = aligned16(residual);
        int s = 0, round = 0;
        for (long long tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
            if (round && !mbar_wait(&empty[s], (round - 1) & 1)) return;
            unsigned char* stage = smem + at.stage0 + at.stage_bytes * s;
            const long long row0 = tile * tp;
            const int here = (int)min((long long)tp, a.rows - row0);
            const bool whole = here == tp;
            unsigned bytes = 0;
            auto rows_in = [&](unsigned char* to, const TI* from, int c, bool bulk) {
                if (whole && bulk) bytes += (unsigned)(tp * c * sizeof(TI));
                else copy_in<sizeof(TI)>(to, from + row0 * c, here * c);
            };
            rows_in(stage, x, k, bulk_x);
            if (k2) rows_in(stage + at.x2_at, x2, k2, bulk_x2);
            if (residual) rows_in(stage + at.r_at, residual, n, bulk_r);
            cp_async_wait_all();
            if (lane == 0 && bytes) {
                mbar_expect_tx(&full[s], bytes);   // (lane 0's arrival)
                if (bulk_x) bulk_load(stage, x + row0 * k, (unsigned)(tp * k * sizeof(TI)), &full[s]);
                if (k2 && bulk_x2) bulk_load(stage + at.x2_at, x2 + row0 * k2, (unsigned)(tp * k2 * sizeof(TI)), &full[s]);
                if (residual && bulk_r) bulk_load(stage + at.r_at, residual + row0 * n, (unsigned)(tp * n * sizeof(TI)), &full[s]);
            } else {
                mbar_arrive(&full[s]);
            }
            if (++s == stages) s = 0, round++;
        }
        return;
    }

    // the weights, zeros behind the last channel of either side, by the consumers while the first tile arrives
    constexpr int WS = mix_weight_stride(NT);
    const int kp = up8(k), threads = 32 * warps;
    for (int i = threadIdx.x; i < (kp + up8(k2)) * WS; i += threads) {
        const int r = i / WS, c = i - r * WS;
        const bool second = r >= kp;
        const int j = second ? r - kp : r;
        float v = 0.f;
        if (c < n && j < (second ? k2 : k))
            v = load_weight(second ? a.weight2 : a.weight, a.transposed ? c * k + j : j * n + c, a.weight_dtype);
        w_s[mix_weight_at(NT, r, c)] = v;
    }
    for (int i = threadIdx.x; i < 8 * NT; i += threads) bias_s[i] = a.bias && i < n ? load_weight(a.bias, i, a.weight_dtype) : 0.f;
    asm volatile("bar.sync 1, %0;" ::"r"(threads) : "memory");

    const int g = lane >> 2, t = lane & 3, r0 = warp * 16 * MT;
    const bool split_w = a.weight_dtype == PL_F32, bulk_out = aligned16(a.out);
    int s = 0, parity = 0;
    for (long long tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
        unsigned char* stage = smem + at.stage0 + at.stage_bytes * s;
        const bool arrived = mbar_wait(&full[s], parity);
        const long long row0 = tile * tp + r0;
        const int here = (int)max(0ll, min((long long)(16 * MT), a.rows - row0));
        TO* o_s = reinterpret_cast<TO*>(stage + at.r_at);
        if (here > 0) {
            float acc[MT][NT][4];
#pragma unroll
            for (int m = 0; m < MT; m++)
#pragma unroll
                for (int j = 0; j < NT; j++)
#pragma unroll
                    for (int i = 0; i < 4; i++) acc[m][j][i] = arrived ? 0.f : NAN;   // gave up: nothing that could pass for a result
            mix_products<TI, NT, MT>(acc, reinterpret_cast<const TI*>(stage), k, w_s, r0, split_w);
            if (k2) mix_products<TI, NT, MT>(acc, reinterpret_cast<const TI*>(stage + at.x2_at), k2, w_s + (size_t)kp * WS, r0, split_w);
            const TI* r_s = reinterpret_cast<const TI*>(stage + at.r_at);
#pragma unroll
            for (int m = 0; m < MT; m++)
#pragma unroll
                for (int h = 0; h < 2; h++) {   // rows g and g + 8 of the sixteen
                    const int row = r0 + 16 * m + 8 * h + g;
                    float z[2 * NT];
#pragma unroll
                    for (int j = 0; j < 2 * NT; j++) {
                        const int c = 8 * (j / 2) + 2 * t + (j & 1);
                        z[j] = acc[m][j / 2][2 * h + (j & 1)] + bias_s[c];
                        if (a.residual && c < n) z[j] = fmaf(a.scale, to_float(r_s[row * n + c]), z[j]);
                    }
                    if (a.activation == PL_ACT_SOFTMAX) {
                        float top = -INFINITY, den = 0.f;
#pragma unroll
                        for (int j = 0; j < 2 * NT; j++)
                            if (8 * (j / 2) + 2 * t + (j & 1) < n) top = fmaxf(top, z[j]);
                        top = fmaxf(top, __shfl_xor_sync(~0u, top, 1));
                        top = fmaxf(top, __shfl_xor_sync(~0u, top, 2));
                        if (top == -INFINITY) top = 0.f;   // nothing allowed: zeros (a NaN among them stays one)
#pragma unroll
                        for (int j = 0; j < 2 * NT; j++) {
                            z[j] = 8 * (j / 2) + 2 * t + (j & 1) < n ? __expf(z[j] - top) : 0.f;
                            den += z[j];
                        }
                        den += __shfl_xor_sync(~0u, den, 1);
                        den += __shfl_xor_sync(~0u, den, 2);
                        const float inv = den == 0.f ? 0.f : 1.f / den;
#pragma unroll
                        for (int j = 0; j < 2 * NT; j++) z[j] *= inv;
                    } else if (a.activation == PL_ACT_RELU) {
#pragma unroll
                        for (int j = 0; j < 2 * NT; j++) z[j] = z[j] < 0.f ? 0.f : z[j];
                    }
                    // The output goes where the residual was.  Each lane has read the values at the places that it writes; with
                    // an output of fewer bytes than the input there is no residual.
#pragma unroll
                    for (int j = 0; j < 2 * NT; j++) {
                        const int c = 8 * (j / 2) + 2 * t + (j & 1);
                        if (c < n) o_s[row * n + c] = from_float<TO>(z[j]);
                    }
                }
            fence_async_proxy();
            __syncwarp();
            copy_out(static_cast<TO*>(a.out) + row0 * n, o_s + r0 * n, here * n, bulk_out && here == 16 * MT);
            if (lane == 0) bulk_commit();
            if constexpr (MT == 2) {   // whole blocks: 32 rows of any number of channels
                auto keep = [&](const auto* rows, int c, uint8_t* codes, int16_t* scales, bool nonzero) {
                    const long long first = row0 * c;
                    pack_by_warp(rows + r0 * c, here * c, codes + first, scales + first / PACK_BLOCK, nonzero,
                                 (reinterpret_cast<uintptr_t>(codes) & 3) == 0);
                };
                if (a.x_codes) keep(reinterpret_cast<const TI*>(stage), k, a.x_codes, a.x_scales, false);
                if (a.x2_codes) keep(reinterpret_cast<const TI*>(stage + at.x2_at), k2, a.x2_codes, a.x2_scales, false);
                if (a.out_codes) keep(o_s, n, a.out_codes, a.out_scales, a.activation == PL_ACT_RELU);
            }
            if (lane == 0) bulk_wait_read();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[s]);
        if (++s == stages) s = 0, parity ^= 1;
    }
}

}  // namespace pl
