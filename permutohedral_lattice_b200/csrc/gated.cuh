// The gated feed-forward block of rows of points, and its gradients:
//
//   g = x Wg + bg,  u = x Wu + bu,  a = act(g) u,  out = a Wd + bd + s residual
//   da = dout Wd^T,  dg = da u act'(g),  du = da act(g),  dx = dg Wg^T + du Wu^T
//   dWg = x^T dg,  dWu = x^T du,  dWd = a^T dout,  dbg, dbu, dbd: sums over rows of dg, du, dout
//
// The hidden values (g, u, a and their gradients) never leave the SM: a CTA takes a tile of rows through the hidden channels a chunk
// at a time.  A chunk's g and u (and da) are products in tensor memory, its a (dg, du) go to shared memory as the next products' operand.
// The biases are a row more of the weights beside a one in every row of x.  The backward pass makes g and u again, in two kernels: gated_kernel<DX>
// sums dx over the chunks of a tile as the forward pass does out, gated_kernel<DW> sums the weights' gradients over the tiles of a
// chunk, a chunk a CTA, and adds them to a share of its own in the workspace now and then (`drain`, see gated_launch.cuh); gated_sums adds up the
// shares in order.
//
// Warps: eight turn the first products into the second's operand, and take out the sums; one asks for products; four fetch rows and
// weights.  They meet at barriers in shared memory; every wait is bounded.  If one runs out, all give up and the results are NaN.
#pragma once
#include "gated_tensor.cuh"

namespace pl {

constexpr int GATED_HIDDEN = 512;   // channels in between, at most
constexpr int GATED_WORKERS = 8, GATED_LOADERS = 4, GATED_THREADS = 32 * (GATED_WORKERS + 1 + GATED_LOADERS);
enum GatedPass { GATED_OUT, GATED_DX, GATED_DW };

struct GatedArgs {
    long long rows;
    int k, h, n, activation;
    int kp, np;                      // columns of a tile of x (with the ones, if there are biases of g or u) and of out
    int chunks, splits;              // of the hidden channels; CTAs of a chunk (DW)
    int x_buffers, w_buffers, a_buffers, s_buffers, d_buffers, drain;
    float scale;
    const void *x, *gate_weight, *up_weight, *down_weight, *gate_bias, *up_bias, *down_bias, *residual, *grad;
    int biased, wide_x, wide_grad, wide_hidden, wide_down, wide_out;   // wide: rows of whole 16 bytes on 16-byte boundaries
    int wide_dresidual, down_bias_wanted;   // (DX, DW)
    void *out, *dresidual;           // out: or dx
    float* shares;                   // [chunks][splits][columns of sums][128]
};

template <typename T>
__host__ __device__ constexpr int gated_chunk() { return sizeof(T) == 4 ? 32 : 64; }   // hidden channels

// Where things lie in shared memory: offsets, bytes of a buffer, in all.
template <typename T, GatedPass PASS, int ROWS>
struct GatedSmem {
    static constexpr int C = gated_chunk<T>(), TERMS = Tensor<T>::TERMS;
    static constexpr int A = TERMS * tile_bytes(ROWS, PASS == GATED_OUT ? C : 2 * C), ACT = PASS == GATED_DW ? TERMS * tile_bytes(ROWS, C) : 0;
    static constexpr int BARRIERS = 1024;
    int grad, x, down, w;            // bytes: a tile of dout, of x with it, of Wd, of all weights of a chunk
    int at_x, at_w, at_a, at_ones, total;
    __host__ __device__ GatedSmem(const GatedArgs& p) {
        grad = PASS == GATED_OUT ? 0 : TERMS * tile_bytes(ROWS, p.np);
        x = grad + TERMS * tile_bytes(ROWS, p.kp);
        down = TERMS * tile_bytes(C, p.np);
        w = down + TERMS * tile_bytes(p.kp, 2 * C);
        at_x = BARRIERS;
        at_w = at_x + p.x_buffers * x;
        at_a = at_w + p.w_buffers * w;
        at_ones = at_a + p.a_buffers * (A + ACT);
        // (products of 128 rows read on behind a tile of 64, and of 128 columns behind one of fewer: what they make of it nobody takes)
        total = at_ones + (PASS == GATED_DW ? tile_bytes(ROWS, 16) : 0) + 2048;
    }
};
// Columns of tensor memory.  DW: of the sums of dWg and dWu, dWd, and dbd.
template <typename T, GatedPass PASS>
struct GatedColumns {
    static constexpr int C = gated_chunk<T>(), WIDE = PASS == GATED_OUT ? 2 * C : 3 * C, SUMS = Tensor<T>::TERMS == 3 ? 2 : 1;
    int d, d_one, low, down, bias, total;
    __host__ __device__ GatedColumns(const GatedArgs& p) {
        d = p.s_buffers * WIDE;
        if (PASS == GATED_DW) {
            down = p.kp;
            bias = down + C;
            d_one = bias + (p.down_bias_wanted ? 16 : 0);
        } else {
            down = bias = 0;
            d_one = PASS == GATED_OUT ? p.np : (p.k + 15) / 16 * 16;
        }
        low = SUMS == 2 ? d_one : 0;         // from a sum to that of its small products
        total = d + p.d_buffers * SUMS * d_one;
    }
};

__device__ __forceinline__ float gated_sigmoid(float g) { return __fdividef(1.f, 1.f + exp2_approx(-1.4426950408889634f * g)); }
// act(g); slope: act'(g)
template <int ACT, bool SLOPE>
__device__ __forceinline__ float gated_act(float g, float& slope) {
    if constexpr (ACT == PL_GATE_SILU) {
        const float s = gated_sigmoid(g);
        if (SLOPE) slope = s * fmaf(g, 1.f - s, 1.f);
        return g * s;
    } else if constexpr (ACT == PL_GATE_SIGMOID) {
        const float s = gated_sigmoid(g);
        if (SLOPE) slope = s * (1.f - s);
        return s;
    } else if constexpr (ACT == PL_GATE_GELU) {
        const float cdf = fmaf(0.5f, erff(0.70710678118654752f * g), 0.5f);
        if (SLOPE) slope = fmaf(g, 0.3989422804014327f * exp2_approx(-0.72134752044448170f * g * g), cdf);
        return g * cdf;
    } else {
        if (SLOPE) slope = g > 0.f ? 1.f : g <= 0.f ? 0.f : g;   // (NaN: itself)
        return g < 0.f ? 0.f : g;
    }
}

// rows x columns values to those of a tile of so many rows by the loaders: row r of `valid` from src + r stride, `valid_columns` of them;
// zeros elsewhere, but for `last`, the row after the valid ones if it is given, and ones in column `ones` of the valid rows.  wide: by 16
// bytes.  plane: bytes from a term to the next.
template <typename T>
__device__ __forceinline__ void stage(unsigned char* to, int rows, int columns, int plane, const T* src, long long stride, int valid, int valid_columns,
                                      const T* last, int ones, bool wide, int thread) {
    constexpr int U = 4, STEP = 32 * GATED_LOADERS;
    const int blocks = columns / 8, cb = column_blocks(rows), items = rows * blocks;
    for (int i0 = thread; i0 < items; i0 += U * STEP) {
        float v[U][8];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int i = i0 + u * STEP, r = i / blocks, c = 8 * (i - r * blocks);
            const T* from = r < valid ? src + r * stride + c : last && r == valid ? last + c : nullptr;
            if (i >= items || c >= valid_columns) from = nullptr;
            if (sizeof(T) == 2 && wide && from && r < valid) {
                cp_async16(to + c / 8 * cb + r * 16, from);
                continue;
            }
#pragma unroll
            for (int e = 0; e < 8; e++) v[u][e] = 0.f;
            if (from) {
                if (wide && r < valid) {
                    float q[4];
                    load4(q, from);
#pragma unroll
                    for (int e = 0; e < 4; e++) v[u][e] = q[e];
                    load4(q, from + 4);
#pragma unroll
                    for (int e = 0; e < 4; e++) v[u][4 + e] = q[e];
                } else {
#pragma unroll
                    for (int e = 0; e < 8; e++)
                        if (c + e < valid_columns) v[u][e] = to_float(from[e]);
                }
            }
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int i = i0 + u * STEP, r = i / blocks, c = 8 * (i - r * blocks);
            if (i >= items || (sizeof(T) == 2 && wide && r < valid && c < valid_columns)) continue;
            if (ones >= c && ones < c + 8 && r < valid) {
#pragma unroll
                for (int e = 0; e < 8; e++)
                    if (c + e == ones) v[u][e] = 1.f;
            }
            store_terms8<T>(to + c / 8 * cb + r * 16, plane, v[u]);
        }
    }
}

struct GatedBarriers {
    u64 x_full[2], x_free[2], w_full[16], w_free[16], s_full[2], s_free[2], a_full[2], a_free[2], d_full[2], d_free[2], end;
    u32 tensor, dead;
};
static_assert(sizeof(GatedBarriers) <= 512);

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
    // Gives up half a second after it began, or (unless it is `last`) when others have.
    __device__ __forceinline__ bool on(u64* bar, int parity, bool last = false) {
        if (!alive || mbar_done(bar, parity & 1)) return alive;
        const u64 began = global_timer();
        for (int i = 1; !mbar_done(bar, parity & 1); i++)
            if ((*dead && !last) || i >= 1 << 26 || ((i & 63) == 0 && global_timer() - began > 500000000ull)) {
                *dead = 1;
                return alive = false;
            }
        return true;
    }
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

// 16 hidden channels of a row: from g, u (and da) to what the second products take.
template <typename T, GatedPass PASS, int ACT, int ROWS>
__device__ __forceinline__ void gated_work(const float (&g)[16], const float (&u)[16], const float (&da)[16], unsigned char* a, int row, int column) {
    constexpr int C = gated_chunk<T>(), CB = column_blocks(ROWS), PLANE = tile_bytes(ROWS, PASS == GATED_OUT ? C : 2 * C);
#pragma unroll
    for (int j = 0; j < 16; j += 8) {
        float v[8], w[8], z[8];
#pragma unroll
        for (int e = 0; e < 8; e++) {
            float slope;
            const float act = gated_act<ACT, PASS != GATED_OUT>(g[j + e], slope);
            if constexpr (PASS == GATED_OUT) {
                v[e] = act * u[j + e];
            } else {
                v[e] = da[j + e] * u[j + e] * slope;
                w[e] = da[j + e] * act;
                z[e] = act * u[j + e];
            }
        }
        unsigned char* to = a + (column + j) / 8 * CB + row * 16;
        store_terms8<T>(to, PLANE, v);
        if constexpr (PASS != GATED_OUT) store_terms8<T>(to + C / 8 * CB, PLANE, w);
        if constexpr (PASS == GATED_DW) store_terms8<T>(to + Tensor<T>::TERMS * PLANE, tile_bytes(ROWS, C), z);
    }
}

template <typename T, GatedPass PASS, int ROWS>
__global__ void __launch_bounds__(GATED_THREADS, 1) gated_kernel(const __grid_constant__ GatedArgs p) {
    extern __shared__ __align__(128) unsigned char smem[];
    using Smem = GatedSmem<T, PASS, ROWS>;
    using Columns = GatedColumns<T, PASS>;
    constexpr int C = gated_chunk<T>(), TERMS = Tensor<T>::TERMS;
    const Smem at(p);
    const Columns col(p);
    GatedBarriers& b = *reinterpret_cast<GatedBarriers*>(smem);
    float* bias_s = reinterpret_cast<float*>(smem + 512);   // of out
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; i++) {
            mbar_init(&b.x_full[i], 32 * GATED_LOADERS), mbar_init(&b.x_free[i], 1);
            mbar_init(&b.s_full[i], 1), mbar_init(&b.s_free[i], GATED_WORKERS);
            mbar_init(&b.a_full[i], GATED_WORKERS), mbar_init(&b.a_free[i], 1);
            mbar_init(&b.d_full[i], 1), mbar_init(&b.d_free[i], GATED_WORKERS);
        }
        for (int i = 0; i < p.w_buffers; i++) mbar_init(&b.w_full[i], 32 * GATED_LOADERS), mbar_init(&b.w_free[i], 1);
        mbar_init(&b.end, 1);
        b.dead = 0;
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(shared_address(&b.tensor)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    if constexpr (PASS == GATED_OUT)
        for (int i = threadIdx.x; i < p.np; i += GATED_THREADS) bias_s[i] = p.down_bias && i < p.n ? to_float(static_cast<const T*>(p.down_bias)[i]) : 0.f;
    if constexpr (PASS == GATED_DW) {   // a column of ones
        for (int i = threadIdx.x; i < tile_bytes(ROWS, 16) / 4; i += GATED_THREADS) reinterpret_cast<u32*>(smem + at.at_ones)[i] = 0;
        __syncthreads();
        for (int i = threadIdx.x; i < ROWS; i += GATED_THREADS)
            *reinterpret_cast<typename Tensor<T>::Term*>(smem + at.at_ones + 16 * i) = from_float<typename Tensor<T>::Term>(1.f);
        fence_async_proxy();
    }
    tensor_before_sync();
    __syncthreads();
    tensor_after_sync();
    const u32 tensor = b.tensor;
    Waits wait{&b.dead};

    // What this CTA does: tiles from `first` on, every `step`-th, each through `chunks` chunks from `chunk0` on.
    const long long tiles = (p.rows + ROWS - 1) / ROWS;
    const int split = PASS == GATED_DW ? blockIdx.x / p.chunks : blockIdx.x, step = PASS == GATED_DW ? p.splits : gridDim.x;
    const int chunk0 = PASS == GATED_DW ? blockIdx.x % p.chunks : 0, chunks = PASS == GATED_DW ? 1 : p.chunks;
    const long long mine = split < tiles ? (tiles - split + step - 1) / step : 0;
    const long long all = mine * chunks;                                  // steps: chunks of tiles
    const int group = PASS == GATED_DW ? p.drain : chunks;                // steps whose sums are one
    const bool resident = p.w_buffers >= chunks;

    if (warp > GATED_WORKERS) {   // loaders
        const int thread = threadIdx.x - 32 * (GATED_WORKERS + 1);
        Turn xt, wt;
        for (long long t = 0; t < mine && wait.alive; t++) {
            const long long row0 = (split + t * step) * ROWS;
            const int valid = (int)min((long long)ROWS, p.rows - row0);
            if (!wait.free(b.x_free, xt)) break;
            unsigned char* x = smem + at.at_x + xt.at * at.x;
            if constexpr (PASS != GATED_OUT)
                stage<T>(x, ROWS, p.np, tile_bytes(ROWS, p.np), static_cast<const T*>(p.grad) + row0 * p.n, p.n, valid, p.n, nullptr, -1, p.wide_grad, thread);
            stage<T>(x + at.grad, ROWS, p.kp, tile_bytes(ROWS, p.kp), static_cast<const T*>(p.x) + row0 * p.k, p.k, valid, p.k, nullptr,
                     p.biased ? p.k : -1, p.wide_x, thread);
            if (sizeof(T) == 2) cp_async_wait_all();
            fence_async_proxy();
            mbar_arrive(&b.x_full[xt.at]);
            xt.next(p.x_buffers);
            if (t > 0 && resident) continue;
            for (int c = 0; c < chunks; c++) {
                if (!wait.free(b.w_free, wt)) break;
                unsigned char* w = smem + at.at_w + wt.at * at.w;
                const int h0 = (chunk0 + c) * C, have = min(C, p.h - h0);
                const T *wg = static_cast<const T*>(p.gate_weight) + h0, *wu = static_cast<const T*>(p.up_weight) + h0;
                const T *bg = static_cast<const T*>(p.gate_bias), *bu = static_cast<const T*>(p.up_bias);
                stage<T>(w, C, p.np, tile_bytes(C, p.np), static_cast<const T*>(p.down_weight) + (long long)h0 * p.n, p.n, have, p.n, nullptr, -1, p.wide_down,
                         thread);
                // gate and up side by side in one tile
                const int plane = tile_bytes(p.kp, 2 * C);
                stage<T>(w + at.down, p.kp, C, plane, wg, p.h, p.k, have, bg ? bg + h0 : nullptr, -1, p.wide_hidden, thread);
                stage<T>(w + at.down + tile_bytes(p.kp, C), p.kp, C, plane, wu, p.h, p.k, have, bu ? bu + h0 : nullptr, -1, p.wide_hidden, thread);
                if (sizeof(T) == 2) cp_async_wait_all();
                fence_async_proxy();
                mbar_arrive(&b.w_full[wt.at]);
                wt.next(p.w_buffers);
            }
        }
    } else if (warp == GATED_WORKERS) {   // products
        if (lane == 0) {
            Turn x1, w1, s1, w2, x2, a2, d2;   // of the first and the second products
            int c1 = 0, in_group = 0;
            long long q1 = 0;
            const int k_steps = p.kp / 16, n_steps = p.np / 16;
            auto first = [&]() {   // g, u (, da) of the next step
                if (q1 >= all) return;
                if (c1 == 0 && !wait.full(b.x_full, x1)) return;
                if (!(resident && q1 >= chunks) && !wait.full(b.w_full, w1)) return;
                if (!wait.free(b.s_free, s1)) return;
                tensor_after_sync();
                const u32 x = shared_address(smem + at.at_x + x1.at * at.x), w = shared_address(smem + at.at_w + w1.at * at.w);
                const u32 s = tensor + s1.at * Columns::WIDE;
                products<T>(s, s, over_columns(x + at.grad, ROWS, p.kp), over_rows(w + at.down, p.kp, 2 * C), 2 * C, k_steps, false, false);
                if constexpr (PASS != GATED_OUT) products<T>(s + 2 * C, s + 2 * C, over_columns(x, ROWS, p.np), over_columns(w, C, p.np), C, n_steps, false, false);
                tensor_commit(&b.s_full[s1.at]);
                s1.next(p.s_buffers), w1.next(p.w_buffers);
                q1++;
                if (++c1 == chunks) {
                    c1 = 0;
                    if (PASS != GATED_DW) tensor_commit(&b.x_free[x1.at]);
                    x1.next(p.x_buffers);
                }
            };
            // One step ahead, where there is room for it: its weights', and in DW (where the second products read x too) its rows'.
            const bool ahead = (resident || p.w_buffers >= 2) && (PASS != GATED_DW || p.x_buffers == 2);
            if (ahead) first();
            for (long long q = 0; q < all && wait.alive; q++) {
                first();
                if (!wait.alive || !wait.full(b.a_full, a2)) break;
                if (in_group == 0 && !wait.free(b.d_free, d2)) break;
                tensor_after_sync();
                const u32 x = shared_address(smem + at.at_x + x2.at * at.x), w = shared_address(smem + at.at_w + w2.at * at.w);
                const u32 a = shared_address(smem + at.at_a + a2.at * (Smem::A + Smem::ACT));
                const u32 d = tensor + col.d + d2.at * Columns::SUMS * col.d_one;
                const bool add = in_group > 0;
                if constexpr (PASS == GATED_OUT) {
                    products<T>(d, d + col.low, over_columns(a, ROWS, C), over_rows(w, C, p.np), p.np, C / 16, add, add);
                } else if constexpr (PASS == GATED_DX) {
                    products<T>(d, d + col.low, over_columns(a, ROWS, 2 * C), over_columns(w + at.down, p.kp, 2 * C), col.d_one, 2 * C / 16, add, add);
                } else {
                    products<T>(d, d + col.low, over_rows(a, ROWS, 2 * C), over_rows(x + at.grad, ROWS, p.kp), p.kp, ROWS / 16, add, add);
                    products<T>(d + col.down, d + col.down + col.low, over_rows(x, ROWS, p.np), over_rows(a + Smem::A, ROWS, C), C, ROWS / 16, add, add);
                    if (p.down_bias_wanted) {   // (a one has one term)
                        const u32 shape = 1u << 4 | Tensor<T>::FORMAT << 7 | Tensor<T>::FORMAT << 10 | 1u << 15 | 1u << 16 | 2u << 17 | 8u << 24;
                        const Operand rows_of = over_rows(x, ROWS, p.np), one = over_rows(shared_address(smem + at.at_ones), ROWS, 16);
                        for (int t = TERMS - 1; t >= 0; t--)
                            for (int s = 0; s < ROWS / 16; s++)
                                tensor_product(d + col.bias + (t ? col.low : 0), rows_of.descriptor(s, t), one.descriptor(s, 0), shape,
                                               add || s > 0 || (TERMS == 3 && t == 1));
                    }
                    tensor_commit(&b.x_free[x2.at]);
                    x2.next(p.x_buffers);
                }
                tensor_commit(&b.a_free[a2.at]);
                if (!resident) tensor_commit(&b.w_free[w2.at]);
                a2.next(p.a_buffers), w2.next(p.w_buffers);
                if (++in_group == group || q + 1 == all) {
                    in_group = 0;
                    tensor_commit(&b.d_full[d2.at]);
                    d2.next(p.d_buffers);
                }
            }
            tensor_commit(&b.end);
        }
    } else {   // workers
        const int quarter = warp & 3, half = warp >> 2, row = 32 * quarter + lane;
        const bool works = 32 * quarter < ROWS;
        const u32 lanes = tensor + ((u32)(32 * quarter) << 16);
        Turn st, act, dt;
        int in_group = 0;
        long long group_index = 0;
        // The finished sums: of tile group_index, or of as many groups of tiles.
        auto take_out = [&](long long index) {
            if (!wait.full(b.d_full, dt)) return;
            tensor_after_sync();
            const u32 d = lanes + col.d + dt.at * Columns::SUMS * col.d_one;
            const long long at_row = PASS == GATED_DW ? 0 : (split + index * step) * ROWS + row;
            const bool there = works && at_row < p.rows;
            float* share = PASS == GATED_DW ? p.shares + ((long long)chunk0 * p.splits + split) * col.d_one * 128 + row : nullptr;
            for (int c = 16 * half; c < col.d_one; c += 32) {
                float v[16], low[16];
                __syncwarp();
                tensor_load16(v, d + c);
                if (Columns::SUMS == 2) tensor_load16(low, d + col.low + c);
                tensor_loaded();
                if (Columns::SUMS == 2) {
#pragma unroll
                    for (int j = 0; j < 16; j++) v[j] += low[j];
                }
                if constexpr (PASS == GATED_DW) {
                    float* to = share + (long long)c * 128;
#pragma unroll
                    for (int j = 0; j < 16; j++) low[j] = index ? to[j * 128] : 0.f;
#pragma unroll
                    for (int j = 0; j < 16; j++) to[j * 128] = low[j] + v[j];
                } else if (there) {
                    const int width = PASS == GATED_OUT ? p.n : p.k;
                    if constexpr (PASS == GATED_OUT) {
#pragma unroll
                        for (int j = 0; j < 16; j++) v[j] += bias_s[c + j];
                        if (p.residual) {
                            float r[16];
                            load16(r, static_cast<const T*>(p.residual) + at_row * width + c, width - c, p.wide_out);
#pragma unroll
                            for (int j = 0; j < 16; j++) v[j] = fmaf(p.scale, r[j], v[j]);
                        }
                    }
                    store16(static_cast<T*>(p.out) + at_row * width + c, v, width - c, p.wide_out);
                }
            }
            if constexpr (PASS == GATED_DX) {   // s dout, which has just been read
                if (p.dresidual && there)
                    for (int c = 16 * half; c < p.np; c += 32) {
                        float v[16];
                        load16(v, static_cast<const T*>(p.grad) + at_row * p.n + c, p.n - c, p.wide_dresidual);
#pragma unroll
                        for (int j = 0; j < 16; j++) v[j] *= p.scale;
                        store16(static_cast<T*>(p.dresidual) + at_row * p.n + c, v, p.n - c, p.wide_dresidual);
                    }
                __syncwarp();
            }
            tensor_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(&b.d_free[dt.at]);
            dt.next(p.d_buffers);
        };
        for (long long q = 0; q < all && wait.alive; q++) {
            if (!wait.full(b.s_full, st)) break;
            if (!wait.free(b.a_free, act)) break;
            tensor_after_sync();
            const u32 s = lanes + st.at * Columns::WIDE;
            unsigned char* a = smem + at.at_a + act.at * (Smem::A + Smem::ACT);
            if (works) {
#pragma unroll 1
                for (int j = 0; j < C / 2; j += 16) {
                    const int c = half * (C / 2) + j;
                    float g[16], u[16], da[16];
                    tensor_load16(g, s + c);
                    tensor_load16(u, s + C + c);
                    if (PASS != GATED_OUT) tensor_load16(da, s + 2 * C + c);
                    tensor_loaded();
                    if (p.activation == PL_GATE_SILU) gated_work<T, PASS, PL_GATE_SILU, ROWS>(g, u, da, a, row, c);
                    else if (p.activation == PL_GATE_GELU) gated_work<T, PASS, PL_GATE_GELU, ROWS>(g, u, da, a, row, c);
                    else if (p.activation == PL_GATE_SIGMOID) gated_work<T, PASS, PL_GATE_SIGMOID, ROWS>(g, u, da, a, row, c);
                    else gated_work<T, PASS, PL_GATE_RELU, ROWS>(g, u, da, a, row, c);
                }
            }
            fence_async_proxy();
            tensor_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(&b.s_free[st.at]), mbar_arrive(&b.a_full[act.at]);
            st.next(p.s_buffers), act.next(p.a_buffers);
            if (in_group == 0 && q > 0) take_out(group_index++);   // of the group before: its last products had this step's time
            if (++in_group == group) in_group = 0;
        }
        if (wait.alive && all > 0) take_out(group_index);
    }
    // All products are done, or a wait has run out: then nothing that could pass for a result.
    __syncwarp();
    if (warp == GATED_WORKERS) Waits{&b.dead}.on(&b.end, 0, true);
    __syncthreads();
    if (b.dead) {
        if constexpr (PASS == GATED_DW) {
            float* share = p.shares + ((long long)chunk0 * p.splits + split) * col.d_one * 128;
            for (int i = threadIdx.x; i < col.d_one * 128; i += GATED_THREADS) share[i] = NAN;
        } else {
            const int width = PASS == GATED_OUT ? p.n : p.k;
            for (long long t = 0; t < mine; t++) {
                const long long row0 = (split + t * step) * ROWS, count = min((long long)ROWS, p.rows - row0) * width;
                for (long long i = threadIdx.x; i < count; i += GATED_THREADS) static_cast<T*>(p.out)[row0 * width + i] = from_float<T>(NAN);
                if (PASS == GATED_DX && p.dresidual)
                    for (long long i = threadIdx.x; i < min((long long)ROWS, p.rows - row0) * p.n; i += GATED_THREADS)
                        static_cast<T*>(p.dresidual)[row0 * p.n + i] = from_float<T>(NAN);
            }
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
    int k, h, n, kp, chunk, chunks, splits, columns, down, bias;
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
        chunk = i / p.chunk, column = r, line = i % p.chunk + (up ? p.chunk : 0);
    } else {
        r -= 2 * (p.k + 1);
        if (i >= p.n) return;
        if (r == p.h ? !p.down_bias : !p.down_weight) return;
        to = r == p.h ? static_cast<T*>(p.down_bias) + i : static_cast<T*>(p.down_weight) + (long long)r * p.n + i;
        chunk = r == p.h ? 0 : r / p.chunk, column = r == p.h ? p.bias : p.down + r % p.chunk, line = i;
    }
    const float* from = p.shares + ((long long)chunk * p.splits * p.columns + column) * 128 + line;
    float sum = 0.f;
#pragma unroll 8
    for (int s = 0; s < p.splits; s++) sum += from[(long long)s * p.columns * 128];
    *to = from_float<T>(sum);
}

}  // namespace pl
