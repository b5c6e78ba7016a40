// Many channels out (68 and more, see tensor_pays) of float rows, on the fifth-generation tensor cores: tiles of 128 rows by 128 columns,
// sums in tensor memory.  x and the weights go through 32 channels at a time: all threads fetch them into registers while the products of the
// 32 before run, take each value as two terms of 11 bits (see mix_common.cuh) and write these to shared memory as the products read them;
// one thread then asks for the products.  Of three: hi hi, lo hi, hi lo.
//
// Sums.  The tensor cores cut what they add to; sums of 128 labels that cancel (dz W^T) lost 1.6 bits by it.  So hi hi of every third 32
// channels goes to a sum of its own, and all products with a low term, 2^-11 of the others, to a fourth; the four of a row are added up as
// floats are.  Each takes 128 columns of tensor memory, all of it: a CTA an SM.
//
// 154 401 rows of 128 + 128 channels to 128: 175 us, 269 by mix_forward_wide.  The bytes take 48 us and the products 0.4 of some 2 us that
// 32 channels take (without two of the three 196 us where it took 201).  It is bound by the way of the next 32 through registers (201 with
// their loads asked for after the barrier, 141 without loads), by their terms' way to shared memory (263 where eight threads write to the
// same banks) and by the output, a row in four threads (321 with an access a channel; 256 threads 205).
#pragma once
#include "mix_forward.cuh"

namespace pl {

constexpr int TC_THREADS = 512, TC_ROWS = 128, TC_COLUMNS = 128, TC_CHUNK = 32, TC_SUMS = 3;
constexpr int TC_PARTS = TC_THREADS / 128, TC_OWN = TC_COLUMNS / TC_PARTS, TC_U = 1024 / TC_THREADS;   // threads of a row, columns of each; pieces that it fetches
// Operands in shared memory: blocks of 8 rows by 4 channels, 16 bytes a row, blocks of the same channels one after another.  16 bytes more
// between channels, so that eight threads with the channels of one row write to different banks.
constexpr int TC_ROW_BLOCKS = 128, TC_CHANNEL_BLOCKS = 128 * 16 + 16;   // bytes from a block of rows, of channels to the next
constexpr int TC_OPERAND = TC_CHUNK / 4 * TC_CHANNEL_BLOCKS;              // bytes of 128 rows by 32 channels
constexpr size_t TC_SMEM = 128 + 2 * sizeof(float) * TC_PARTS * TC_ROWS + sizeof(float) * TC_COLUMNS + 2 * 4 * (size_t)TC_OPERAND;

__device__ __forceinline__ u64 tc_operand(u32 address) {   // no swizzle, channels leading
    return (u64)((address >> 4) & 0x3FFF) | (u64)(TC_CHANNEL_BLOCKS >> 4) << 16 | (u64)(TC_ROW_BLOCKS >> 4) << 32 | 1ull << 46;
}
// d (+)= a b^T: 128 x 128 x 8, 11-bit numbers, sums in float
__device__ __forceinline__ void tc_product(u32 d, u64 a, u64 b, bool add) {
    constexpr u32 SHAPE = 1u << 4 | 2u << 7 | 2u << 10 | (TC_COLUMNS / 8) << 17 | (TC_ROWS / 16) << 24;
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::tf32 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b),
                 "r"(SHAPE), "r"((u32)add)
                 : "memory");
}
__device__ __forceinline__ void tc_commit(u64* bar) {   // the barrier's phase ends when all products asked for so far are done
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(shared_address(bar)) : "memory");
}
__device__ __forceinline__ void tc_load16(float (&v)[16], u32 at) {   // a row of the lane's own, 16 columns
    u32 r[16];
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
                   "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(at));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < 16; i++) v[i] = __uint_as_float(r[i]);
}

// Faster from 64 channels in, in rows of whole float4 out.  us at 10 000 / 100 000 / 400 000 rows, mix_forward_wide and this: 64 to 128
// channels 22 / 75 / 241 and 13 / 67 / 232, 67 + 67 to 68 34 / 109 / 362 and 16 / 82 / 298; 16 to 68 11 / 30 / 103 and 9 / 36 / 137.  Rows
// that leave as single channels take 101 to 101 channels 92 us at 100 000, 119 here.  (Sizes alone decide: an address changes no bit of a result.)
__host__ inline bool tensor_pays(const MixArgs& a) { return a.k + a.k2 >= 64 && a.n % 4 == 0; }

template <typename TO, typename W>
__global__ void __launch_bounds__(TC_THREADS, 1) mix_forward_tensor(MixArgs a) {
    extern __shared__ __align__(128) unsigned char smem[];
    u64* bars = reinterpret_cast<u64*>(smem);                       // of the two buffers
    u32* tensor_s = reinterpret_cast<u32*>(smem + 64);
    float* top_s = reinterpret_cast<float*>(smem + 128);            // [parts][128]: of a row's parts
    float* den_s = top_s + TC_PARTS * TC_ROWS;
    float* bias_s = den_s + TC_PARTS * TC_ROWS;
    unsigned char* buffers = reinterpret_cast<unsigned char*>(bias_s + TC_COLUMNS);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, k = a.k, k2 = a.k2, n = a.n;
    const float* x = static_cast<const float*>(a.x);
    const float* x2 = static_cast<const float*>(a.x2);
    const float* residual = static_cast<const float*>(a.residual);
    TO* out = static_cast<TO*>(a.out);
    if (threadIdx.x == 0) mbar_init(&bars[0], 1), mbar_init(&bars[1], 1);
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(shared_address(tensor_s)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    for (int i = threadIdx.x; i < TC_COLUMNS; i += TC_THREADS) bias_s[i] = a.bias && i < n ? load_weight(a.bias, i, a.weight_dtype) : 0.f;
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const u32 tensor = *tensor_s;

    const int chunks = (k + TC_CHUNK - 1) / TC_CHUNK, all = chunks + (k2 + TC_CHUNK - 1) / TC_CHUNK;
    const long long tiles = (a.rows + TC_ROWS - 1) / TC_ROWS;
    const bool quads = k % 4 == 0 && aligned16(x), quads2 = k2 % 4 == 0 && aligned16(x2), quads_out = aligned16(residual) && aligned16(out);
    // What a thread fetches of 32 channels: four channels of rows i / 8 (i = its number, and so on), and of the weights.
    // (What is not there is read elsewhere and made zero when it is stored: nothing waits for a load before then, and no branch parts them.)
    float4 next_x[TC_U];
    W next_w[TC_U][4];
    const int my_c = 4 * (threadIdx.x & 7), my_row = threadIdx.x >> 3;
    // (A row of the weights is one of columns, or of channels where they are transposed: threads side by side read along it.  dz and
    // two dz W^T of 154 401 rows and 128 + 128 labels: 228 us, 337 where they read across.)
    const int my_cw = a.transposed ? my_c : 4 * (threadIdx.x >> 7), my_col = a.transposed ? my_row : threadIdx.x & 127;
    const int next_cw = a.transposed ? 0 : 4 * TC_PARTS, next_col = a.transposed ? TC_THREADS / 8 : 0;   // from one piece to the next
    auto fetch = [&](long long tile, int chunk) {
        const bool second = chunk >= chunks;
        const int width = second ? k2 : k, c0 = (second ? chunk - chunks : chunk) * TC_CHUNK;
        const W* w = static_cast<const W*>(second ? a.weight2 : a.weight);
        const int of_channel = a.transposed ? 1 : n, of_column = a.transposed ? k : 1;
#pragma unroll
        for (int u = 0; u < TC_U; u++)
#pragma unroll
            for (int e = 0; e < 4; e++) next_w[u][e] = w[min(c0 + my_cw + next_cw * u + e, width - 1) * of_channel + min(my_col + next_col * u, n - 1) * of_column];
        const float* rows = second ? x2 : x;
        const int c = c0 + my_c;
#pragma unroll
        for (int u = 0; u < TC_U; u++) {
            const float* from = rows + min(tile * TC_ROWS + my_row + TC_THREADS / 8 * u, a.rows - 1) * width;
            if (second ? quads2 : quads) next_x[u] = *reinterpret_cast<const float4*>(from + min(c, width - 4));
            else next_x[u] = make_float4(from[min(c, width - 1)], from[min(c + 1, width - 1)], from[min(c + 2, width - 1)], from[min(c + 3, width - 1)]);
        }
    };
    auto store_terms = [&](unsigned char* hi_at, int at, float v0, float v1, float v2, float v3) {   // and the low ones behind the high ones
        uint4 hi, lo;
        split(v0, hi.x, lo.x);
        split(v1, hi.y, lo.y);
        split(v2, hi.z, lo.z);
        split(v3, hi.w, lo.w);
        *reinterpret_cast<uint4*>(hi_at + at) = hi;
        *reinterpret_cast<uint4*>(hi_at + TC_OPERAND + at) = lo;
    };
    auto store = [&](unsigned char* buffer, long long tile, int chunk) {
        const bool second = chunk >= chunks;
        const int width = second ? k2 : k, c0 = (second ? chunk - chunks : chunk) * TC_CHUNK, left = width - c0 - my_c;
#pragma unroll
        for (int u = 0; u < TC_U; u++) {
            const int row = my_row + TC_THREADS / 8 * u, have = tile * TC_ROWS + row < a.rows ? left : 0;
            const float4 q = next_x[u];
            store_terms(buffer, my_c / 4 * TC_CHANNEL_BLOCKS + (row >> 3) * TC_ROW_BLOCKS + (row & 7) * 16, have > 0 ? q.x : 0.f, have > 1 ? q.y : 0.f,
                        have > 2 ? q.z : 0.f, have > 3 ? q.w : 0.f);
            const int cw = my_cw + next_cw * u, col = my_col + next_col * u, have_w = col < n ? width - c0 - cw : 0;
            store_terms(buffer + 2 * TC_OPERAND, cw / 4 * TC_CHANNEL_BLOCKS + (col >> 3) * TC_ROW_BLOCKS + (col & 7) * 16,
                        have_w > 0 ? to_float(next_w[u][0]) : 0.f, have_w > 1 ? to_float(next_w[u][1]) : 0.f, have_w > 2 ? to_float(next_w[u][2]) : 0.f,
                        have_w > 3 ? to_float(next_w[u][3]) : 0.f);
        }
    };
    const int part = warp >> 2, row_in_tile = 32 * (warp & 3) + lane;
    const u32 my_sums = tensor + ((u32)(32 * (warp & 3)) << 16) + TC_OWN * part;   // this lane's row, this warp's part of the columns
    bool alive = true;
    u32 count = 0;   // chunks so far: buffer count % 2, for the (count / 2)-th time
    fetch(blockIdx.x, 0);
    for (long long tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
#pragma unroll 1
        for (int chunk = 0; chunk < all; chunk++, count++) {
            unsigned char* buffer = buffers + (count & 1) * 4 * TC_OPERAND;
            u64* bar = &bars[count & 1];
            if (count >= 2) alive = alive && mbar_wait(bar, ((count >> 1) - 1) & 1);   // the products that read it last
            store(buffer, tile, chunk);
            if (chunk + 1 < all) fetch(tile, chunk + 1);
            else fetch(tile + gridDim.x, 0);
            fence_async_proxy();
            alive = __syncthreads_and(alive ? 1 : 0) != 0;
            if (threadIdx.x == 0 && alive) {
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const u32 at = shared_address(buffer);
                const int left = chunk >= chunks ? k2 - (chunk - chunks) * TC_CHUNK : k - chunk * TC_CHUNK;
                const u32 sum = tensor + TC_COLUMNS * (chunk % TC_SUMS), lows = tensor + TC_COLUMNS * TC_SUMS;
                for (int c = 0; c < min(left, TC_CHUNK); c += 8) {
                    const u32 step = c / 4 * TC_CHANNEL_BLOCKS;
                    const u64 x_hi = tc_operand(at + step), x_lo = tc_operand(at + TC_OPERAND + step);
                    const u64 w_hi = tc_operand(at + 2 * TC_OPERAND + step), w_lo = tc_operand(at + 3 * TC_OPERAND + step);
                    tc_product(sum, x_hi, w_hi, chunk >= TC_SUMS || c > 0);
                    tc_product(lows, x_lo, w_hi, chunk > 0 || c > 0);
                    tc_product(lows, x_hi, w_lo, true);
                }
                tc_commit(bar);
            }
        }
        alive = alive && mbar_wait(&bars[(count - 1) & 1], ((count - 1) >> 1) & 1);   // all products of the tile
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        alive = __all_sync(~0u, alive);
        const long long row = tile * TC_ROWS + row_in_tile;
        const bool there = row < a.rows;
        const int c0 = TC_OWN * part;
        float z[TC_OWN];
#pragma unroll
        for (int j = 0; j < TC_OWN; j += 16) {
            float v[16];
            tc_load16(v, my_sums + TC_COLUMNS * TC_SUMS + j);
#pragma unroll
            for (int i = 0; i < 16; i++) z[j + i] = v[i];
            for (int s = 0; s < min(all, TC_SUMS); s++) {
                tc_load16(v, my_sums + TC_COLUMNS * s + j);
#pragma unroll
                for (int i = 0; i < 16; i++) z[j + i] += v[i];
            }
        }
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");   // (the next products come after the next barrier of all)
        if (residual) {   // (what is not there is read elsewhere, and nobody keeps what becomes of it)
            const float* from = residual + min(row, a.rows - 1) * n;
            if (quads_out) {
#pragma unroll
                for (int j = 0; j < TC_OWN; j += 4) {
                    const float4 q = *reinterpret_cast<const float4*>(from + min(c0 + j, n - 4));
                    z[j] = fmaf(a.scale, q.x, z[j]), z[j + 1] = fmaf(a.scale, q.y, z[j + 1]);
                    z[j + 2] = fmaf(a.scale, q.z, z[j + 2]), z[j + 3] = fmaf(a.scale, q.w, z[j + 3]);
                }
            } else {
#pragma unroll
                for (int j = 0; j < TC_OWN; j++) z[j] = fmaf(a.scale, from[min(c0 + j, n - 1)], z[j]);
            }
        }
#pragma unroll
        for (int j = 0; j < TC_OWN; j++) z[j] += bias_s[c0 + j];
        if (!alive) {
#pragma unroll
            for (int j = 0; j < TC_OWN; j++) z[j] = NAN;   // gave up: nothing that could pass for a result
        }
        if (a.activation == PL_ACT_SOFTMAX) {   // (see mix_activate; a row lies in four threads here)
            float top = -INFINITY, den = 0.f;
#pragma unroll
            for (int j = 0; j < TC_OWN; j++) {
                if (c0 + j >= n) z[j] = -INFINITY;
                top = fmaxf(top, z[j]);
            }
            top_s[part * TC_ROWS + row_in_tile] = top;
            __syncthreads();
#pragma unroll
            for (int q = 0; q < TC_PARTS; q++) top = fmaxf(top, top_s[q * TC_ROWS + row_in_tile]);
            if (top == -INFINITY) top = 0.f;
#pragma unroll
            for (int j = 0; j < TC_OWN; j++) {
                z[j] = exp2_approx((z[j] - top) * 1.4426950408889634f);
                den += z[j];
            }
            den_s[part * TC_ROWS + row_in_tile] = den;
            __syncthreads();
            den = 0.f;
#pragma unroll
            for (int q = 0; q < TC_PARTS; q++) den += den_s[q * TC_ROWS + row_in_tile];   // (the same order for all)
            const float inv = den == 0.f ? 0.f : __fdividef(1.f, den);
#pragma unroll
            for (int j = 0; j < TC_OWN; j++) z[j] *= inv;
        } else if (a.activation == PL_ACT_RELU) {
#pragma unroll
            for (int j = 0; j < TC_OWN; j++) z[j] = z[j] < 0.f ? 0.f : z[j];
        }
        if (!there) continue;
        TO* to = out + row * n + c0;
        if (quads_out) {
#pragma unroll
            for (int j = 0; j < TC_OWN; j += 4)
                if (c0 + j < n) {
                    const float v[4] = {z[j], z[j + 1], z[j + 2], z[j + 3]};
                    store4(to + j, v);
                }
        } else {
#pragma unroll
            for (int j = 0; j < TC_OWN; j++)
                if (c0 + j < n) to[j] = from_float<TO>(z[j]);
        }
    }
    if (!alive) mbar_wait(&bars[0], 0), mbar_wait(&bars[0], 1), mbar_wait(&bars[1], 0), mbar_wait(&bars[1], 1);   // nothing in flight
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tensor) : "memory");
}

}  // namespace pl
