// out = act(x W [+ x2 W2] [+ bias] [+ s residual]) of rows of up to 128 channels.
//
// One pass over memory: tiles of rows come and go by bulk copies (see mix_common.cuh), the weights stay in shared memory for
// all tiles of a CTA, a warp takes 16 MT rows at a time through the tensor cores and finishes them in registers (a row's logits lie in
// the registers of four lanes: the maximum and the sum of a softmax take two shuffles each); the output leaves from where the
// residual came in.
#pragma once
#include "mix_common.cuh"

namespace pl {

#ifndef MIXF_C
#define MIXF_C (NT <= 4 ? 4 : 2)
#endif
struct MixArgs {
    long long rows;
    int k, k2, n, activation;
    float scale;                       // of the residual
    const void *x, *x2, *weight, *weight2, *bias, *residual;
    void* out;
    int weight_dtype, transposed;      // transposed: weight is [n][k] (no second input)
    int stages, blocks;                // blocks of 16 MT rows in a tile
    uint8_t *x_codes, *x2_codes, *out_codes;
    int16_t *x_scales, *x2_scales, *out_scales;
};

__host__ __device__ constexpr int up8(int v) { return (v + 7) & ~7; }
__host__ __device__ constexpr size_t up16(size_t v) { return (v + 15) & ~(size_t)15; }
// Weights in shared memory: blocks of 8 x 8 as the lanes take them, with up to 32 output channels both terms of each (see mix_common.cuh).
__host__ __device__ constexpr bool mix_both_terms(int nt) { return nt <= 4; }
__host__ __device__ constexpr int mix_block_bytes(int nt) { return mix_both_terms(nt) ? 512 : 256; }
__host__ __device__ constexpr size_t mix_weight_bytes(int nt, int rows) { return (size_t)rows / 8 * nt * mix_block_bytes(nt); }
// The first of the bytes of row r, column c.
__host__ __device__ constexpr int mix_weight_at(int nt, int r, int c) {
    return ((r >> 3) * nt + (c >> 3)) * mix_block_bytes(nt) + (4 * (c & 7) + (r & 3)) * (mix_block_bytes(nt) / 32) + 4 * (r >> 2 & 1);
}
// Column blocks all of whose channels are there, whatever n: those of up to 64 channels are compiled one by one.
__host__ __device__ constexpr int mix_full_blocks(int nt) { return nt <= 8 ? nt - 1 : nt / 2; }

template <typename TI, typename TO>
struct MixSmem {   // byte offsets; a stage holds `rows` rows of x, x2 and of the residual, in whose place the output leaves
    size_t weights, bias, stage0, x2_at, r_at, stage_bytes;
    __host__ __device__ MixSmem(int rows, int k, int k2, int n, int nt) {
        weights = up16(sizeof(u64) * MIX_WARPS * MIX_STAGES);   // barriers before
        bias = up16(weights + mix_weight_bytes(nt, up8(k) + up8(k2)));
        stage0 = up16(bias + sizeof(float) * 8 * nt);
        x2_at = up16(sizeof(TI) * (size_t)rows * k);
        r_at = x2_at + up16(sizeof(TI) * (size_t)rows * k2);
        stage_bytes = up16(r_at + (sizeof(TI) > sizeof(TO) ? sizeof(TI) : sizeof(TO)) * (size_t)rows * n);
    }
    __host__ __device__ size_t bytes(int warps, int stages) const { return stage0 + stage_bytes * stages * warps; }
};

// acc += eight channels of a block's rows times eight weight rows, which begin at w.  rows: where the lane's rows begin at its channel.
// PARTS: their products by themselves, then added to the sums as floats are.  The tensor cores cut what they add to: of
// sums of more than a hundred terms that cancel (128 labels: dz W^T) it cost 1.6 bits.
template <typename TI, int NT, int MT, bool PARTS, bool EDGE>
__device__ __forceinline__ void mix_product8(float (&acc)[MT][NT][4], const u32 (&rows)[2 * MT], int left, u32 w, bool split_w) {
    constexpr int JG = NT % 4 == 0 ? 4 : NT % 3 == 0 ? 3 : NT % 2 == 0 ? 2 : NT == 1 ? 1 : NT;
    const int t = threadIdx.x & 3;
    u32 a_hi[MT][4], a_lo[MT][4];
#pragma unroll
    for (int m = 0; m < MT; m++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            float v = 0.f;
            if (!EDGE || t + (i & 2 ? 4 : 0) < left) v = lds_value<TI>(rows[2 * m + (i & 1)] + (i & 2 ? 4 : 0) * sizeof(TI));   // behind lies another row, which may hold NaN
            if constexpr (sizeof(TI) == 4) split(v, a_hi[m][i], a_lo[m][i]);
            else a_hi[m][i] = __float_as_uint(v);
        }
#pragma unroll
    for (int j0 = 0; j0 < NT; j0 += JG) {
        u32 b_hi[JG][2], b_lo[JG][2];
#pragma unroll
        for (int j = 0; j < JG; j++) {
            if constexpr (mix_both_terms(NT)) {
                const uint4 b = lds4(w + 512 * (j0 + j));
                b_hi[j][0] = b.x, b_hi[j][1] = b.y, b_lo[j][0] = b.z, b_lo[j][1] = b.w;
            } else {
                const uint2 b = lds2(w + 256 * (j0 + j));
                split(__uint_as_float(b.x), b_hi[j][0], b_lo[j][0]);
                split(__uint_as_float(b.y), b_hi[j][1], b_lo[j][1]);
            }
        }
        float part[PARTS ? MT : 1][PARTS ? JG : 1][4];
        auto all = [&](const u32 (&l)[MT][4], const u32 (&r)[JG][2], bool first) {
#pragma unroll
            for (int j = 0; j < JG; j++)
#pragma unroll
                for (int m = 0; m < MT; m++) {
                    if (PARTS && first) mma8_first(part[PARTS ? m : 0][PARTS ? j : 0], l[m], r[j]);
                    else if (PARTS) mma8(part[PARTS ? m : 0][PARTS ? j : 0], l[m], r[j]);
                    else mma8(acc[m][j0 + j], l[m], r[j]);
                }
        };
        all(a_hi, b_hi, true);
        if constexpr (sizeof(TI) == 4) all(a_lo, b_hi, false);
        if (sizeof(TI) == 4 || split_w) all(a_hi, b_lo, false);
        if constexpr (PARTS) {
#pragma unroll
            for (int j = 0; j < JG; j++)
#pragma unroll
                for (int m = 0; m < MT; m++)
#pragma unroll
                    for (int e = 0; e < 4; e++) acc[m][j0 + j][e] += part[m][j][e];
        }
    }
}
// All k channels of the rows that begin at x_at.
template <typename TI, int NT, int MT, bool PARTS>
__device__ __forceinline__ void mix_products(float (&acc)[MT][NT][4], u32 x_at, int k, u32 w, bool split_w) {
    const int g = (threadIdx.x & 31) >> 2, t = threadIdx.x & 3;
    u32 rows[2 * MT];
#pragma unroll
    for (int m = 0; m < 2 * MT; m++) rows[m] = x_at + ((8 * m + g) * k + t) * sizeof(TI);
    int left = k;
#pragma unroll 1
    for (; left >= 8; left -= 8, w += NT * mix_block_bytes(NT)) {
        mix_product8<TI, NT, MT, PARTS, false>(acc, rows, 8, w, split_w);
#pragma unroll
        for (int m = 0; m < 2 * MT; m++) rows[m] += 8 * sizeof(TI);
    }
    if (left) mix_product8<TI, NT, MT, PARTS, true>(acc, rows, left, w, split_w);
}

template <typename TI, typename TO, int NT, int MT, bool PARTS>
__global__ void __launch_bounds__(128, MIXF_C) mix_forward(MixArgs a) {
    extern __shared__ __align__(128) unsigned char smem[];
    constexpr int BLOCK = 16 * MT;
    const int warps = (int)blockDim.x / 32, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int tile_rows = BLOCK * a.blocks, k = a.k, k2 = a.k2, n = a.n, stages = a.stages;
    const MixSmem<TI, TO> at(tile_rows, k, k2, n, NT);
    u64* bars = reinterpret_cast<u64*>(smem) + MIX_STAGES * warp;
    float* bias_s = reinterpret_cast<float*>(smem + at.bias);
    unsigned char* stage0 = smem + at.stage0 + at.stage_bytes * stages * warp;
    const TI* x = static_cast<const TI*>(a.x);
    const TI* x2 = static_cast<const TI*>(a.x2);
    const TI* residual = static_cast<const TI*>(a.residual);
    const long long tiles = (a.rows + tile_rows - 1) / tile_rows, step = (long long)gridDim.x * warps;
    const long long first = (long long)blockIdx.x * warps + warp;
    if (lane == 0)
        for (int s = 0; s < stages; s++) mbar_init(&bars[s], 1);
    __syncwarp();
    const bool bulk_in = aligned16(x) && (!k2 || aligned16(x2)) && (!residual || aligned16(residual));
    const u32 tile_bytes = (u32)(tile_rows * (k + k2 + (residual ? n : 0)) * sizeof(TI));
    auto fetch = [&](long long tile, int s) {
        unsigned char* stage = stage0 + at.stage_bytes * s;
        const long long row0 = tile * tile_rows;
        if (bulk_in && row0 + tile_rows <= a.rows) {
            if (lane == 0) {
                mbar_expect_tx(&bars[s], tile_bytes);
                bulk_load(stage, x + row0 * k, (u32)(tile_rows * k * sizeof(TI)), &bars[s]);
                if (k2) bulk_load(stage + at.x2_at, x2 + row0 * k2, (u32)(tile_rows * k2 * sizeof(TI)), &bars[s]);
                if (residual) bulk_load(stage + at.r_at, residual + row0 * n, (u32)(tile_rows * n * sizeof(TI)), &bars[s]);
            }
        } else if (row0 < a.rows) {
            const int here = (int)min((long long)tile_rows, a.rows - row0);
            copy_in(stage, x + row0 * k, here * k);
            if (k2) copy_in(stage + at.x2_at, x2 + row0 * k2, here * k2);
            if (residual) copy_in(stage + at.r_at, residual + row0 * n, here * n);
            if (lane == 0) mbar_expect_tx(&bars[s], 0);
        }
    };
    for (int s = 0; s < stages; s++) fetch(first + s * step, s);

    // the weights, zeros behind the last channel of either side, while the first tiles arrive
    const int kp = up8(k);
    for (int i = threadIdx.x; i < (kp + up8(k2)) * 8 * NT; i += blockDim.x) {
        const int r = i / (8 * NT), c = i - r * (8 * NT);
        const bool second = r >= kp;
        const int j = second ? r - kp : r;
        float v = 0.f;
        if (c < n && j < (second ? k2 : k))
            v = load_weight(second ? a.weight2 : a.weight, a.transposed ? c * k + j : j * n + c, a.weight_dtype);
        unsigned char* to = smem + at.weights + mix_weight_at(NT, r, c);
        if constexpr (mix_both_terms(NT)) {
            u32 hi, lo;
            split(v, hi, lo);
            reinterpret_cast<u32*>(to)[0] = hi, reinterpret_cast<u32*>(to)[2] = lo;
        } else {
            *reinterpret_cast<float*>(to) = v;
        }
    }
    for (int i = threadIdx.x; i < 8 * NT; i += blockDim.x) bias_s[i] = a.bias && i < n ? load_weight(a.bias, i, a.weight_dtype) : 0.f;
    __syncthreads();

    const int g = lane >> 2, t = lane & 3;
    const u32 w_at = shared_address(smem + at.weights) + lane * (mix_block_bytes(NT) / 32);
    const bool split_w = a.weight_dtype == PL_F32, bulk_out = aligned16(a.out);
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
        TO* o_s = reinterpret_cast<TO*>(stage + at.r_at);
        const u32 stage_at = shared_address(stage);
#pragma unroll 1
        for (int r0 = 0; r0 < rows_here; r0 += BLOCK) {
            const int here = min(BLOCK, rows_here - r0);
            float acc[MT][NT][4];
#pragma unroll
            for (int j = 0; j < NT; j++) {
                const float2 b = *reinterpret_cast<const float2*>(bias_s + 8 * j + 2 * t);
#pragma unroll
                for (int m = 0; m < MT; m++) acc[m][j][0] = acc[m][j][2] = b.x, acc[m][j][1] = acc[m][j][3] = b.y;
            }
#pragma unroll 1
            for (int second = 0; second < (k2 ? 2 : 1); second++)
                mix_products<TI, NT, MT, PARTS>(acc, second ? stage_at + (u32)at.x2_at + r0 * k2 * sizeof(TI) : stage_at + r0 * k * sizeof(TI), second ? k2 : k,
                                                second ? w_at + kp / 8 * NT * mix_block_bytes(NT) : w_at, split_w);
#pragma unroll
            for (int m = 0; m < MT; m++)
#pragma unroll
                for (int h = 0; h < 2; h++) {   // rows g and g + 8 of the sixteen
                    // A channel that is not there, of the blocks that may have some: never the largest, nothing in a sum.
                    auto there = [&](int j) { return j / 2 < mix_full_blocks(NT) || 8 * (j / 2) + 2 * t + (j & 1) < n; };
                    const int row = (r0 + 16 * m + 8 * h + g) * n + 2 * t;
                    const u32 r_at = stage_at + (u32)at.r_at + row * sizeof(TI), to = stage_at + (u32)at.r_at + row * sizeof(TO);
                    float z[2 * NT];
#pragma unroll
                    for (int j = 0; j < 2 * NT; j++) z[j] = acc[m][j / 2][2 * h + (j & 1)];
                    if (residual) {
#pragma unroll
                        for (int j = 0; j < 2 * NT; j++)
                            if (there(j)) z[j] = fmaf(a.scale, lds_value<TI>(r_at + (8 * (j / 2) + (j & 1)) * sizeof(TI)), z[j]);
                    }
                    if (a.activation == PL_ACT_SOFTMAX) {
                        constexpr float LOG2_E = 1.4426950408889634f;
                        float top = -INFINITY, den = 0.f;
#pragma unroll
                        for (int j = 0; j < 2 * NT; j++) {
                            if (!there(j)) z[j] = -INFINITY;
                            top = fmaxf(top, z[j]);
                        }
                        top = fmaxf(top, __shfl_xor_sync(~0u, top, 1));
                        top = fmaxf(top, __shfl_xor_sync(~0u, top, 2));
                        if (top == -INFINITY) top = 0.f;   // nothing allowed: zeros (a NaN among them stays one)
#pragma unroll
                        for (int j = 0; j < 2 * NT; j++) {
                            z[j] = exp2_approx((z[j] - top) * LOG2_E);   // (in one step the type's least value would overflow)
                            den += z[j];
                        }
                        den += __shfl_xor_sync(~0u, den, 1);
                        den += __shfl_xor_sync(~0u, den, 2);
                        const float inv = den == 0.f ? 0.f : __fdividef(1.f, den);   // (1 to 128: the quick quotient is within a step)
#pragma unroll
                        for (int j = 0; j < 2 * NT; j++) z[j] *= inv;
                    } else if (a.activation == PL_ACT_RELU) {
#pragma unroll
                        for (int j = 0; j < 2 * NT; j++) z[j] = z[j] < 0.f ? 0.f : z[j];
                    }
                    if (!alive) {
#pragma unroll
                        for (int j = 0; j < 2 * NT; j++) z[j] = NAN;   // nothing that could pass for a result
                    }
                    // The output goes where the residual was.  Each lane has read the values at the places that it writes; with
                    // an output of fewer bytes than the input there is no residual.
#pragma unroll
                    for (int j = 0; j < 2 * NT; j++)
                        if (there(j)) sts_value<TO>(to + (8 * (j / 2) + (j & 1)) * sizeof(TO), z[j]);
                }
            if constexpr (MT == 2) {   // whole blocks: 32 rows of any number of channels
                const long long row0 = tile0 + r0;
                auto keep = [&](const auto* rows, int c, uint8_t* codes, int16_t* scales, bool nonzero) {
                    const long long from = row0 * c;
                    pack_by_warp(rows + r0 * c, here * c, codes + from, scales + from / PACK_BLOCK, nonzero,
                                 (reinterpret_cast<uintptr_t>(codes) & 3) == 0);
                };
                if (a.x_codes) keep(reinterpret_cast<const TI*>(stage), k, a.x_codes, a.x_scales, false);
                if (a.x2_codes) keep(reinterpret_cast<const TI*>(stage + at.x2_at), k2, a.x2_codes, a.x2_scales, false);
                if (a.out_codes) {
                    __syncwarp();
                    keep(o_s, n, a.out_codes, a.out_scales, a.activation == PL_ACT_RELU);
                }
            }
        }
        fence_async_proxy();
        __syncwarp();
        copy_out(static_cast<TO*>(a.out) + tile0 * n, o_s, rows_here * n, bulk_out && rows_here == tile_rows);
        if (lane == 0) {
            bulk_commit();
            bulk_wait_read();
        }
        __syncwarp();
        if (alive) fetch(tile + stages * step, s);
        if (++s == stages) s = 0, parity ^= 1;
    }
    if (!alive)   // gave up once: no copy may be in flight when the CTA ends
        for (int i = 0; i < stages; i++) mbar_wait(&bars[i], 0), mbar_wait(&bars[i], 1);
}

}  // namespace pl
