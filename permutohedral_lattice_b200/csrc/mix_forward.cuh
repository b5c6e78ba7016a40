// out = act(x W [+ x2 W2] [+ bias] [+ s residual]) of rows of up to 128 channels.
//
// One pass over memory: tiles of rows come and go by bulk copies (see mix_common.cuh), the weights stay in shared memory for
// all tiles of a CTA, a warp takes 16 MT rows at a time through the tensor cores and finishes them in registers (a row's logits lie in
// the registers of four lanes: the maximum and the sum of a softmax take two shuffles each); the output leaves from where the
// residual came in.
//
// 16 x 512x512 rows of 21 + 21 channels to 21, floats: 252 us, 5.6 TB/s of what has to be moved.  Half of them: 133 us; without the products
// 117, without the softmax too 113, and 101 for torch's addcmul, which reads three tensors and writes one.  Four CTAs of four warps an SM:
// three, five and six (which spill) took 148, 141 and 153 where four took 143.  What is left are issue slots: IPC 2 of 4.
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
    int blocks;                        // of 16 MT rows in a tile
    int x_apart, x2_apart, out_apart;  // rows may lie apart in shared memory (see RowsApart): x, x2, residual and out
    uint8_t *x_codes, *x2_codes, *out_codes;
    int16_t *x_scales, *x2_scales, *out_scales;
};

__host__ __device__ constexpr int up8(int v) { return (v + 7) & ~7; }
__host__ __device__ constexpr size_t up16(size_t v) { return (v + 15) & ~(size_t)15; }
// How the products are made.  Plain and parted: m16n8k8 on terms of floats, parted adds up eight channels' products before they
// join the sums (see mix_product8).  Pairs: m16n8k16, for 16-bit values times weights of the same type.
enum MixWay { MIX_PLAIN, MIX_PARTED, MIX_PAIRS };

// Weights in shared memory: blocks of 8 (16 in pairs) x 8 as the lanes take them, both terms of each with up to 32 output channels
// (see mix_common.cuh).
__host__ __device__ constexpr bool mix_both_terms(int nt, int way) { return nt <= 4 && way != MIX_PAIRS; }
__host__ __device__ constexpr int mix_block_bytes(int nt, int way) { return mix_both_terms(nt, way) ? 512 : 256; }
__host__ __device__ constexpr int mix_step(int way) { return way == MIX_PAIRS ? 16 : 8; }   // channels of one product
__host__ __device__ constexpr int up_to(int v, int m) { return (v + m - 1) / m * m; }
__host__ __device__ constexpr size_t mix_weight_bytes(int nt, int way, int rows) { return (size_t)rows / mix_step(way) * nt * mix_block_bytes(nt, way); }
// The first of the bytes of row r, column c.
__host__ __device__ constexpr int mix_weight_at(int nt, int way, int r, int c) {
    return way == MIX_PAIRS ? ((r >> 4) * nt + (c >> 3)) * 256 + (4 * (c & 7) + (r >> 1 & 3)) * 8 + 4 * (r >> 3 & 1) + 2 * (r & 1)
                            : ((r >> 3) * nt + (c >> 3)) * mix_block_bytes(nt, way) + (4 * (c & 7) + (r & 3)) * (mix_block_bytes(nt, way) / 32) + 4 * (r >> 2 & 1);
}
// CTAs of four warps that an SM's registers have to hold.
__host__ __device__ constexpr int mix_forward_ctas(int nt, int way) { return nt <= 4 ? 4 : way == MIX_PAIRS ? 3 : 2; }
// Column blocks all of whose channels are there, whatever n: those of up to 64 channels are compiled one by one.
__host__ __device__ constexpr int mix_full_blocks(int nt) { return nt <= 8 ? nt - 1 : nt / 2; }

template <typename TI, typename TO>
struct MixSmem {   // byte offsets; a stage holds the tile's rows of x, x2 and of the residual, in whose place the output leaves
    RowsApart x, x2, out;
    size_t weights, bias, stage0, x2_at, r_at, stage_bytes;
    __host__ __device__ MixSmem(const MixArgs& a, int rows, int nt, int way)
        : x(a.k, sizeof(TI), a.x_apart), x2(a.k2, sizeof(TI), a.x2_apart), out(a.n, sizeof(TO), a.out_apart) {
        weights = up16(sizeof(u64) * 2 * MIX_WARPS);   // barriers before
        bias = up16(weights + mix_weight_bytes(nt, way, up_to(a.k, mix_step(way)) + up_to(a.k2, mix_step(way))));
        stage0 = up16(bias + sizeof(float) * 8 * nt);
        x2_at = up16(sizeof(TI) * (size_t)rows * x.stride);
        r_at = x2_at + up16(sizeof(TI) * (size_t)rows * x2.stride);
        stage_bytes = up16(r_at + sizeof(TO) * (size_t)rows * out.stride);   // (a residual has the output's type)
    }
    __host__ __device__ size_t bytes(int warps) const { return stage0 + stage_bytes * warps; }
};

// The left side of a product of eight channels: those of the lane's 2 MT rows, which begin (at its channel) at rows[].  EDGE: fewer are left;
// behind them lies another row, which may hold NaN.
template <typename TI, int MT, bool EDGE>
__device__ __forceinline__ void mix_load_left(float (&v)[MT][4], const u32 (&rows)[2 * MT], int left) {
    const int t = threadIdx.x & 3;
#pragma unroll
    for (int m = 0; m < MT; m++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const u32 at = rows[2 * m + (i & 1)] + (i & 2 ? 4 : 0) * sizeof(TI);
            if constexpr (EDGE) v[m][i] = lds_value_if<TI>(t + (i & 2 ? 4 : 0) < left, at);
            else v[m][i] = lds_value<TI>(at);
        }
}
template <typename TI, int MT>
__device__ __forceinline__ void mix_split_left(u32 (&hi)[MT][4], u32 (&lo)[MT][4], const float (&v)[MT][4]) {
#pragma unroll
    for (int m = 0; m < MT; m++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if constexpr (sizeof(TI) == 4) split(v[m][i], hi[m][i], lo[m][i]);
            else hi[m][i] = __float_as_uint(v[m][i]);
        }
}
// acc += the left side times eight weight rows, which begin at w.
// PARTS: the products by themselves, then added to the sums as floats are.  The tensor cores cut what they add to: of
// sums of more than a hundred terms that cancel (128 labels: dz W^T) it cost 1.6 bits.
template <typename TI, int NT, int MT, bool PARTS>
__device__ __forceinline__ void mix_product8(float (&acc)[MT][NT][4], const u32 (&a_hi)[MT][4], const u32 (&a_lo)[MT][4], u32 w, bool split_w) {
    constexpr int JG = NT % 16 == 0 ? 8 : NT % 4 == 0 ? 4 : NT % 3 == 0 ? 3 : NT % 2 == 0 ? 2 : NT == 1 ? 1 : NT;
#pragma unroll
    for (int j0 = 0; j0 < NT; j0 += JG) {
        u32 b_hi[JG][2], b_lo[JG][2];
#pragma unroll
        for (int j = 0; j < JG; j++) {
            if constexpr (mix_both_terms(NT, MIX_PLAIN)) {
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
// All k channels of the rows that begin at x_at.  (The next eight loaded while eight are multiplied: 142 us where this takes 133.  Other warps
// hide the loads, and the loop has less to move about.)
template <typename TI, int NT, int MT, bool PARTS>
__device__ __forceinline__ void mix_products(float (&acc)[MT][NT][4], u32 x_at, int k, int stride, u32 w, bool split_w) {
    const int g = (threadIdx.x & 31) >> 2, t = threadIdx.x & 3;
    u32 rows[2 * MT];
#pragma unroll
    for (int m = 0; m < 2 * MT; m++) rows[m] = x_at + ((8 * m + g) * stride + t) * sizeof(TI);
    int left = k;
#pragma unroll 1
    for (; left >= 8; left -= 8, w += NT * mix_block_bytes(NT, MIX_PLAIN)) {
        float v[MT][4];
        u32 a_hi[MT][4], a_lo[MT][4];
        mix_load_left<TI, MT, false>(v, rows, left);
        mix_split_left<TI, MT>(a_hi, a_lo, v);
#pragma unroll
        for (int m = 0; m < 2 * MT; m++) rows[m] += 8 * sizeof(TI);
        mix_product8<TI, NT, MT, PARTS>(acc, a_hi, a_lo, w, split_w);
    }
    if (left > 0) {
        float v[MT][4];
        u32 a_hi[MT][4], a_lo[MT][4];
        mix_load_left<TI, MT, true>(v, rows, left);
        mix_split_left<TI, MT>(a_hi, a_lo, v);
        mix_product8<TI, NT, MT, PARTS>(acc, a_hi, a_lo, w, split_w);
    }
}
// The same in pairs.  A row of an odd number of 16-bit values begins between words: its pairs are put together.
template <typename TI, int MT>
__device__ __forceinline__ void mix_load_pairs(u32 (&v)[MT][4], const u32 (&rows)[2 * MT], int left, bool words) {
    const int t = threadIdx.x & 3;
#pragma unroll
    for (int m = 0; m < MT; m++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int c = 2 * t + (i & 2 ? 8 : 0);
            const u32 at = rows[2 * m + (i & 1)] + (i & 2 ? 16 : 0);
            if (words) v[m][i] = lds_u32_if(c < left, at);   // (behind the last channel lies another row, which may hold NaN)
            else v[m][i] = lds_u16_if(c < left, at) | lds_u16_if(c + 1 < left, at + 2) << 16;
        }
}
template <typename TI, int NT, int MT>
__device__ __forceinline__ void mix_products_of_pairs(float (&acc)[MT][NT][4], u32 x_at, int k, int stride, u32 w) {
    const int g = (threadIdx.x & 31) >> 2, t = threadIdx.x & 3;
    const bool words = k % 2 == 0;   // (then the stride is even, too)
    u32 rows[2 * MT];
#pragma unroll
    for (int m = 0; m < 2 * MT; m++) rows[m] = x_at + ((8 * m + g) * stride + 2 * t) * 2;
#pragma unroll 1
    for (int left = k; left > 0; left -= 16, w += NT * 256) {
        u32 v[MT][4];
        mix_load_pairs<TI, MT>(v, rows, left, words);
#pragma unroll
        for (int m = 0; m < 2 * MT; m++) rows[m] += 32;
#pragma unroll
        for (int j = 0; j < NT; j++) {
            const uint2 b = lds2(w + 256 * j);
            const u32 both[2] = {b.x, b.y};
#pragma unroll
            for (int m = 0; m < MT; m++) mma16<TI>(acc[m][j], v[m], both);
        }
    }
}

// Columns 8 (j / 2) + 2 t + j % 2 of R rows, four lanes a row.  A channel that is not there, of the blocks that may have some: never the
// largest, nothing in a sum.
template <int NT>
__device__ __forceinline__ bool mix_there(int j, int n) {
    return j / 2 < mix_full_blocks(NT) || 8 * (j / 2) + 2 * (int)(threadIdx.x & 3) + (j & 1) < n;
}
template <int R, int NT>
__device__ __forceinline__ void mix_activate(float (&z)[R][2 * NT], int activation, int n) {
    if (activation == PL_ACT_SOFTMAX) {
        constexpr float LOG2_E = 1.4426950408889634f;
        float top[R], den[R];
#pragma unroll
        for (int m = 0; m < R; m++) top[m] = -INFINITY, den[m] = 0.f;
#pragma unroll
        for (int j = 0; j < 2 * NT; j++)
#pragma unroll
            for (int m = 0; m < R; m++) {
                if (!mix_there<NT>(j, n)) z[m][j] = -INFINITY;
                top[m] = fmaxf(top[m], z[m][j]);
            }
#pragma unroll
        for (int o = 1; o < 4; o <<= 1)
#pragma unroll
            for (int m = 0; m < R; m++) top[m] = fmaxf(top[m], __shfl_xor_sync(~0u, top[m], o));
#pragma unroll
        for (int m = 0; m < R; m++)
            if (top[m] == -INFINITY) top[m] = 0.f;   // nothing allowed: zeros (a NaN among them stays one)
#pragma unroll
        for (int j = 0; j < 2 * NT; j++)
#pragma unroll
            for (int m = 0; m < R; m++) {
                z[m][j] = exp2_approx((z[m][j] - top[m]) * LOG2_E);   // (in one step the type's least value would overflow)
                den[m] += z[m][j];
            }
#pragma unroll
        for (int o = 1; o < 4; o <<= 1)
#pragma unroll
            for (int m = 0; m < R; m++) den[m] += __shfl_xor_sync(~0u, den[m], o);
#pragma unroll
        for (int m = 0; m < R; m++) {
            const float inv = den[m] == 0.f ? 0.f : __fdividef(1.f, den[m]);   // (1 to 128: the quick quotient is within a step)
#pragma unroll
            for (int j = 0; j < 2 * NT; j++) z[m][j] *= inv;
        }
    } else if (activation == PL_ACT_RELU) {
#pragma unroll
        for (int m = 0; m < R; m++)
#pragma unroll
            for (int j = 0; j < 2 * NT; j++) z[m][j] = z[m][j] < 0.f ? 0.f : z[m][j];
    }
}

// KEEP: the activations go to 8 bits, too (a kernel of its own: as a branch it cost the others a tenth of their time).
// A warp has one stage.  Its rows of x and x2 are fetched again as soon as they have been multiplied, while the rows of the tile are
// finished, those of the residual when the output has left.
template <typename TI, typename TO, int NT, int MT, int WAY, bool KEEP>
__global__ void __launch_bounds__(32 * MIX_WARPS, mix_forward_ctas(NT, WAY)) mix_forward(MixArgs a) {
    extern __shared__ __align__(128) unsigned char smem[];
    constexpr int BLOCK = 16 * MT;
    const int warps = (int)blockDim.x / 32, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int tile_rows = BLOCK * a.blocks, k = a.k, k2 = a.k2, n = a.n;
    const MixSmem<TI, TO> at(a, tile_rows, NT, WAY);
    u64* bars = reinterpret_cast<u64*>(smem) + 2 * warp;   // of x and x2, of the residual
    float* bias_s = reinterpret_cast<float*>(smem + at.bias);
    unsigned char* stage = smem + at.stage0 + at.stage_bytes * warp;
    const TI* x = static_cast<const TI*>(a.x);
    const TI* x2 = static_cast<const TI*>(a.x2);
    const TI* residual = static_cast<const TI*>(a.residual);
    const long long tiles = (a.rows + tile_rows - 1) / tile_rows, step = (long long)gridDim.x * warps;
    const long long first = (long long)blockIdx.x * warps + warp;
    if (lane == 0) mbar_init(&bars[0], 1), mbar_init(&bars[1], 1);
    __syncwarp();
    const bool bulk_x = (at.x.apart() || aligned16(x)) && (!k2 || at.x2.apart() || aligned16(x2)), bulk_r = at.out.apart() || aligned16(residual);
    const u32 x_bytes = (u32)(tile_rows * sizeof(TI)) * ((at.x.apart() ? 0 : k) + (at.x2.apart() ? 0 : k2));
    const u32 r_bytes = (u32)(tile_rows * sizeof(TI)) * (at.out.apart() ? 0 : n);
    auto rows_in = [&](size_t place, const TI* from, int c, const RowsApart& r, int here, bool bulk, u64* bar) {
        TI* to = reinterpret_cast<TI*>(stage + place);
        if (r.apart()) copy_rows_in(to, from, here, r);
        else if (!bulk) copy_in(to, from, here * c);
        else if (lane == 0) bulk_load(to, from, (u32)(tile_rows * c * sizeof(TI)), bar);
    };
    auto fetch_x = [&](long long tile) {
        const long long row0 = tile * tile_rows;
        const int here = (int)max(0ll, min((long long)tile_rows, a.rows - row0));
        const bool bulk = bulk_x && here == tile_rows;
        if (here) {
            if (lane == 0) mbar_expect_tx(&bars[0], bulk ? x_bytes : 0);
            rows_in(0, x + row0 * k, k, at.x, here, bulk, &bars[0]);
            if (k2) rows_in(at.x2_at, x2 + row0 * k2, k2, at.x2, here, bulk, &bars[0]);
        }
        cp_async_commit();
    };
    auto fetch_r = [&](long long tile) {
        const long long row0 = tile * tile_rows;
        const int here = residual ? (int)max(0ll, min((long long)tile_rows, a.rows - row0)) : 0;
        const bool bulk = bulk_r && here == tile_rows;
        if (here) {
            if (lane == 0) mbar_expect_tx(&bars[1], bulk ? r_bytes : 0);
            rows_in(at.r_at, residual + row0 * n, n, at.out, here, bulk, &bars[1]);
        }
        cp_async_commit();
    };
    fetch_x(first);
    fetch_r(first);

    // the weights, zeros behind the last channel of either side, while the first tiles arrive
    const int kp = up_to(k, mix_step(WAY));
    for_weights<8 * NT>(kp + up_to(k2, mix_step(WAY)), kp, k, k2, n, a.weight, a.weight2, a.transposed, a.weight_dtype, [&](int r, int c, float v) {
        unsigned char* to = smem + at.weights + mix_weight_at(NT, WAY, r, c);
        if constexpr (WAY == MIX_PAIRS) {
            *reinterpret_cast<TI*>(to) = from_float<TI>(v);
        } else if constexpr (mix_both_terms(NT, WAY)) {
            u32 hi, lo;
            split(v, hi, lo);
            reinterpret_cast<u32*>(to)[0] = hi, reinterpret_cast<u32*>(to)[2] = lo;
        } else {
            *reinterpret_cast<float*>(to) = v;
        }
    });
    for (int i = threadIdx.x; i < 8 * NT; i += blockDim.x) bias_s[i] = a.bias && i < n ? load_weight(a.bias, i, a.weight_dtype) : 0.f;
    __syncthreads();

    const int g = lane >> 2, t = lane & 3;
    const u32 w_at = shared_address(smem + at.weights) + lane * (mix_block_bytes(NT, WAY) / 32);
    const bool split_w = a.weight_dtype == PL_F32, bulk_out = aligned16(a.out);
    TO* o_s = reinterpret_cast<TO*>(stage + at.r_at);
    const u32 stage_at = shared_address(stage);
    // What has been asked for is there for all lanes; false once it did not come.  (One group of copies has to be committed behind the one
    // that is waited for: a tile's residual behind its x and x2, the next x and x2 behind a residual.)
    auto arrived = [&](u64* bar, int parity, bool before) {
        cp_async_wait_one();
        const bool there = before && mbar_wait(bar, parity);
        const bool all = __all_sync(~0u, there);
        __syncwarp();
        return all;
    };
    bool alive = true;
    int parity = 0;
    for (long long tile = first; tile < tiles; tile += step, parity ^= 1) {
        alive = arrived(&bars[0], parity, alive);
        const long long tile0 = tile * tile_rows;
        const int rows_here = (int)min((long long)tile_rows, a.rows - tile0);
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
            for (int second = 0; second < (k2 ? 2 : 1); second++) {
                const int width = second ? k2 : k;
                const int stride = second ? at.x2.stride : at.x.stride;
                const u32 x_at = stage_at + (second ? (u32)at.x2_at : 0) + r0 * stride * sizeof(TI);
                const u32 w = w_at + (second ? kp / mix_step(WAY) * NT * mix_block_bytes(NT, WAY) : 0);
                if constexpr (WAY == MIX_PAIRS) mix_products_of_pairs<TI, NT, MT>(acc, x_at, width, stride, w);
                else mix_products<TI, NT, MT, WAY == MIX_PARTED>(acc, x_at, width, stride, w, split_w);
            }
            const long long row0 = tile0 + r0;
            auto keep = [&](const auto* rows, int c, const RowsApart& r, uint8_t* codes, int16_t* scales, bool nonzero) {
                const long long from = row0 * c;
                const bool wide = (reinterpret_cast<uintptr_t>(codes) & 3) == 0;
                if (!r.apart()) pack_by_warp(rows + r0 * c, here * c, codes + from, scales + from / PACK_BLOCK, nonzero, wide);
                else   // (see launch_forward: rows lie apart only where the codes are aligned and blocks whole)
                    pack_blocks_of(rows + r0 * r.stride, here * c, codes + from, scales + from / PACK_BLOCK, nonzero, [&](int i) { return r.at(i); });
            };
            if constexpr (KEEP) {   // whole blocks: 32 rows of any number of channels
                static_assert(MT == 2);
                if (a.x_codes) keep(reinterpret_cast<const TI*>(stage), k, at.x, a.x_codes, a.x_scales, false);
                if (a.x2_codes) keep(reinterpret_cast<const TI*>(stage + at.x2_at), k2, at.x2, a.x2_codes, a.x2_scales, false);
            }
            const bool last = r0 + BLOCK >= rows_here;
            if (last) {
                __syncwarp();
                if (alive) fetch_x(tile + step);
            }
            if (r0 == 0 && residual) {
                if (!last) cp_async_commit();   // in a tile of several blocks the next x is not on its way yet: an empty group in its place
                alive = arrived(&bars[1], parity, alive);
            }
            // The lane's 2 MT rows, 8 m + g of the block: z[m].
            constexpr int R = 2 * MT;
            const int ns = at.out.stride, row = (r0 + g) * ns + 2 * t;
            const u32 r_at = stage_at + (u32)at.r_at + row * sizeof(TI), to = stage_at + (u32)at.r_at + row * sizeof(TO);
            float z[R][2 * NT];
#pragma unroll
            for (int m = 0; m < R; m++)
#pragma unroll
                for (int j = 0; j < 2 * NT; j++) z[m][j] = acc[m / 2][j / 2][2 * (m & 1) + (j & 1)];
            if (residual) {
#pragma unroll
                for (int j = 0; j < 2 * NT; j++)
#pragma unroll
                    for (int m = 0; m < R; m++)
                    {
                        const u32 at = r_at + (8 * m * ns + 8 * (j / 2) + (j & 1)) * sizeof(TI);
                        z[m][j] = fmaf(a.scale, j / 2 < mix_full_blocks(NT) ? lds_value<TI>(at) : lds_value_if<TI>(mix_there<NT>(j, n), at), z[m][j]);
                    }
            }
            mix_activate<R, NT>(z, a.activation, n);
            if (!alive) {
#pragma unroll
                for (int m = 0; m < R; m++)
#pragma unroll
                    for (int j = 0; j < 2 * NT; j++) z[m][j] = NAN;   // gave up: nothing that could pass for a result
            }
            // The output goes where the residual was: each lane has read the values at the places that it writes.  With an output of
            // fewer bytes than the input there is no residual.
#pragma unroll
            for (int j = 0; j < 2 * NT; j++)
#pragma unroll
                for (int m = 0; m < R; m++) {
                    const u32 at = to + (8 * m * ns + 8 * (j / 2) + (j & 1)) * sizeof(TO);
                    if (j / 2 < mix_full_blocks(NT)) sts_value<TO>(at, z[m][j]);
                    else sts_value_if<TO>(mix_there<NT>(j, n), at, z[m][j]);
                }
            if constexpr (KEEP) {
                if (a.out_codes) {
                    __syncwarp();
                    keep(o_s, n, at.out, a.out_codes, a.out_scales, a.activation == PL_ACT_RELU);
                }
            }
        }
        fence_async_proxy();
        __syncwarp();
        if (at.out.apart()) copy_rows_out(static_cast<TO*>(a.out) + tile0 * n, o_s, rows_here, at.out);
        else copy_out(static_cast<TO*>(a.out) + tile0 * n, o_s, rows_here * n, bulk_out && rows_here == tile_rows);
        if (lane == 0) {
            bulk_commit();
            bulk_wait_read();
        }
        __syncwarp();
        if (alive) fetch_r(tile + step);
    }
    if (!alive)   // gave up once: no copy may be in flight when the CTA ends
        for (int i = 0; i < 2; i++) mbar_wait(&bars[i], 0), mbar_wait(&bars[i], 1);
}

// ---------------------------------------------------------------------------------------------
// Many channels out (65 and more) of float rows, what mix_forward_tensor does not take (see tensor_pays).  The weights of both inputs take up to 128 KB of shared memory, which leaves too
// little for whole rows: a warp takes 16 rows, 32 channels at a time, by way of its registers (the next ones are on their way while
// these are multiplied), reads the residual and writes its rows from registers.  154 401 rows with a softmax: 101 + 101 channels to 101 210 us,
// 67 + 67 to 67 150, 32 to 96 59, 16 to 68 41.  All columns are computed, up to 128 of them.  Its shape was chosen on 128 + 128 channels to 128,
// which mix_forward_tensor has taken since: 269 us (558 with whole rows in shared memory and four warps an SM; 8, 12 and 14 warps 289, 269
// and 306; four blocks of columns at once in place of eight 285), the tensor cores busy 43 % of the time (110 us, three products of 11-bit terms
// for one of floats at 276 TFLOP/s), warps waiting for products that they depend on.
// ---------------------------------------------------------------------------------------------
constexpr int WIDE_WARPS = 12, WIDE_CHUNK = 32, WIDE_STRIDE = WIDE_CHUNK + 4;   // (rows of 36 floats: 8 rows by 4 channels in 32 banks)
constexpr int WIDE_NT = 16;
__host__ __device__ constexpr size_t wide_smem(int k, int k2) {
    return mix_weight_bytes(WIDE_NT, MIX_PARTED, up8(k) + up8(k2)) + sizeof(float) * (8 * WIDE_NT + WIDE_WARPS * 16 * WIDE_STRIDE);
}
template <typename TO>
__global__ void __launch_bounds__(32 * WIDE_WARPS, 1) mix_forward_wide(MixArgs a) {
    extern __shared__ __align__(128) unsigned char smem[];
    constexpr int NT = WIDE_NT;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int k = a.k, k2 = a.k2, n = a.n, kp = up8(k), all_p = kp + up8(k2);
    float* bias_s = reinterpret_cast<float*>(smem + mix_weight_bytes(NT, MIX_PARTED, all_p));
    float* rows_s = bias_s + 8 * NT + warp * 16 * WIDE_STRIDE;
    for_weights<8 * NT>(all_p, kp, k, k2, n, a.weight, a.weight2, a.transposed, a.weight_dtype,
                        [&](int r, int c, float v) { *reinterpret_cast<float*>(smem + mix_weight_at(NT, MIX_PARTED, r, c)) = v; });
    for (int i = threadIdx.x; i < 8 * NT; i += blockDim.x) bias_s[i] = a.bias && i < n ? load_weight(a.bias, i, a.weight_dtype) : 0.f;
    __syncthreads();
    const float* x = static_cast<const float*>(a.x);
    const float* x2 = static_cast<const float*>(a.x2);
    const float* residual = static_cast<const float*>(a.residual);
    TO* out = static_cast<TO*>(a.out);
    const u32 w_at = shared_address(smem) + lane * 8, rows_at = shared_address(rows_s);
    const bool split_w = a.weight_dtype == PL_F32;
    const int chunks = (k + WIDE_CHUNK - 1) / WIDE_CHUNK, all = chunks + (k2 + WIDE_CHUNK - 1) / WIDE_CHUNK;
    const long long tiles = (a.rows + 15) / 16, step = (long long)gridDim.x * WIDE_WARPS;
    float next[16];
    auto fetch = [&](long long tile, int chunk) {   // a channel a lane, 16 rows
        const bool second = chunk >= chunks;
        const int width = second ? k2 : k, c = (second ? chunk - chunks : chunk) * WIDE_CHUNK + lane;
        const float* from = (second ? x2 : x) + tile * 16 * width + c;
        const int here = tile < tiles && c < width ? (int)min(16ll, a.rows - tile * 16) : 0;
#pragma unroll
        for (int r = 0; r < 16; r++) next[r] = r < here ? from[(long long)r * width] : 0.f;
    };
    long long tile = (long long)blockIdx.x * WIDE_WARPS + warp;
    fetch(tile, 0);
    for (; tile < tiles; tile += step) {
        float acc[1][NT][4];
#pragma unroll
        for (int j = 0; j < NT; j++) {
            const float2 b = *reinterpret_cast<const float2*>(bias_s + 8 * j + 2 * t);
            acc[0][j][0] = acc[0][j][2] = b.x, acc[0][j][1] = acc[0][j][3] = b.y;
        }
#pragma unroll 1
        for (int chunk = 0; chunk < all; chunk++) {
            __syncwarp();
#pragma unroll
            for (int r = 0; r < 16; r++) rows_s[r * WIDE_STRIDE + lane] = next[r];
            __syncwarp();
            if (chunk + 1 < all) fetch(tile, chunk + 1);
            else fetch(tile + step, 0);
            const bool second = chunk >= chunks;
            const int c0 = (second ? chunk - chunks : chunk) * WIDE_CHUNK, left = (second ? k2 : k) - c0;
            u32 w = w_at + ((second ? kp : 0) + c0) / 8 * NT * 256;
            u32 rows[2] = {rows_at + (g * WIDE_STRIDE + t) * 4, rows_at + ((8 + g) * WIDE_STRIDE + t) * 4};
#pragma unroll 1
            for (int c = 0; c < min(left, WIDE_CHUNK); c += 8, w += NT * 256) {
                float v[1][4];
                u32 a_hi[1][4], a_lo[1][4];
                mix_load_left<float, 1, false>(v, rows, 8);   // (zeros behind the last channel)
                mix_split_left<float, 1>(a_hi, a_lo, v);
                rows[0] += 32, rows[1] += 32;
                mix_product8<float, NT, 1, true>(acc, a_hi, a_lo, w, split_w);
            }
        }
        float z[2][2 * NT];
        const long long row0 = tile * 16 + g;
#pragma unroll
        for (int m = 0; m < 2; m++) {
            const long long at = (row0 + 8 * m) * n + 2 * t;
            const bool row_there = row0 + 8 * m < a.rows;
#pragma unroll
            for (int j = 0; j < 2 * NT; j++) {
                z[m][j] = acc[0][j / 2][2 * m + (j & 1)];
                if (residual && row_there && mix_there<NT>(j, n)) z[m][j] = fmaf(a.scale, residual[at + 8 * (j / 2) + (j & 1)], z[m][j]);
            }
        }
        mix_activate<2, NT>(z, a.activation, n);
#pragma unroll
        for (int m = 0; m < 2; m++) {
            const long long at = (row0 + 8 * m) * n + 2 * t;
            if (row0 + 8 * m >= a.rows) continue;
#pragma unroll
            for (int j = 0; j < 2 * NT; j++)
                if (mix_there<NT>(j, n)) out[at + 8 * (j / 2) + (j & 1)] = from_float<TO>(z[m][j]);
        }
    }
}

}  // namespace pl
