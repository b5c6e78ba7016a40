// Norms after and before a block of a network, with dropout, gate and scaled residual between them; rows are points.
//
//   u = (x - m) r wa + ba      m, r: mean and reciprocal deviation of the row (layer), or m = 0 and the root of the mean square (rms); or x
//   v = u keep / (1 - p),  h = s residual + gate v,  y = (h - m') r' wb + bb
//
// and their gradients, with h made again from what came in:
//
//   dh += r' (t - mean(t) - h^ mean(t h^)),  t = dy wb, h^ = (h - m') r'   (rms: without mean(t))
//   dresidual = s dh,  dgate = dh v,  du = dh gate keep / (1 - p),  dx as dh, of t = du wa;  dwa = sum over rows du x^ and so on
//
// One pass over memory each way: a row lies in the registers of 1 to 32 lanes, its sums take shuffles, the parameters' vectors lie in
// shared memory.  The sums over rows stay in a thread's registers for all its rows, then go by way of the CTA to a share of its own in the
// workspace, and a second kernel adds the shares up in order.  Statistics and sums are floats; each result is rounded once.
//
// 617 604 rows of 256 float16 channels, residual and norm: 199 us, 6.35 TB/s of what has to be moved.  4 194 304 of 32 bfloat16 between two blocks, with
// dropout: 242 us, 4.4 TB/s, and the gradients 535, 3.0 TB/s; 174 and 388 without the generator.  3 409 920 of 21 floats with a gate of every value: 205 and 393,
// 5.6 and 4.4 TB/s.  Issue slots bound the narrow ones (60 % busy): shuffles, conversions, and of the generator a product for each of ten rounds and value pair.
// The gradients through two norms of 8 values a lane take more than the 128 registers of a thread: 36 to 204 bytes of them go by way of local memory.  Rows that are not whole pieces,
// of more than 256 channels: 150 000 x 511 floats, residual and two norms 241 us forward, 1480 backward, where 512 channels take 200 and 380.
#pragma once
#include "mix_common.cuh"
#include "philox.cuh"

namespace pl {

constexpr int NORM_MOST = 512;         // channels
constexpr int NORM_THREADS = 256, NORM_WARPS = NORM_THREADS / 32;
constexpr int NORM_VECTORS = 5;        // of parameters, and of their gradients
enum NormVector { NORM_WA, NORM_BA, NORM_WB, NORM_BB, NORM_GATE };

struct NormArgs {
    long long rows;
    int c;                             // channels
    int after, before;                 // pl_norm_kind
    float eps_after, eps_before, scale;
    const void *x, *residual, *gate;   // gate: of every value
    const void* vectors[NORM_VECTORS]; // of the channels, NULL where there are none
    int vector_dtype;
    Dropout drop;
    void *h, *y;
    const void *dh, *dy;
    void *dx, *dresidual, *dgate;
    float* shares;                     // [CTAs][NORM_VECTORS][c]; NULL: no vector's gradient is wanted
    int wanted;                        // bits of them
    int ctas;                          // (host) how many ran
};

// Pieces of a row: V values that follow one another in memory, 16 bytes where rows are whole pieces on 16-byte boundaries, else one value (21
// channels of floats, side by side in their lanes, take as many sectors either way).
template <typename T, bool WIDE>
struct Piece {
    static constexpr int V = WIDE ? 16 / (int)sizeof(T) : 1;
    using Raw = typename std::conditional<WIDE, uint4, T>::type;   // as it comes
    __device__ __forceinline__ static Raw nothing() {
        if constexpr (WIDE) return make_uint4(0, 0, 0, 0);
        else return from_float<T>(0.f);
    }
    __device__ __forceinline__ static void values(float* v, const Raw& q) {
        if constexpr (!WIDE) {
            v[0] = to_float(q);
        } else if constexpr (sizeof(T) == 4) {
            v[0] = __uint_as_float(q.x), v[1] = __uint_as_float(q.y), v[2] = __uint_as_float(q.z), v[3] = __uint_as_float(q.w);
        } else {
            const T* e = reinterpret_cast<const T*>(&q);
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = to_float(e[j]);
        }
    }
    __device__ __forceinline__ static void load(float* v, const T* p) { values(v, *reinterpret_cast<const Raw*>(p)); }
    __device__ __forceinline__ static void store(T* p, const float* v) {
        if constexpr (!WIDE) {
            *p = from_float<T>(v[0]);
        } else if constexpr (sizeof(T) == 4) {
            *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
        } else {
            uint4 q;
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                if constexpr (std::is_same<T, __half>::value) reinterpret_cast<__half2*>(&q)[j / 2] = __floats2half2_rn(v[j], v[j + 1]);
                else reinterpret_cast<__nv_bfloat162*>(&q)[j / 2] = __floats2bfloat162_rn(v[j], v[j + 1]);
            }
            *reinterpret_cast<uint4*>(p) = q;
        }
    }
    __device__ __forceinline__ static void shared(float* v, const float* p) {
        if constexpr (!WIDE) {
            v[0] = *p;
        } else {
#pragma unroll
            for (int j = 0; j < V; j += 4) {
                const float4 q = *reinterpret_cast<const float4*>(p + j);
                v[j] = q.x, v[j + 1] = q.y, v[j + 2] = q.z, v[j + 3] = q.w;
            }
        }
    }
};

// Rows in registers: E values a lane at most, piece i of lane l of a row the (l + i LANES)-th.
// PACKED: two elements an instruction (the gradients of 3.4 million rows of 21 floats 450 us without, 392 with; but 16 million rows' worth of 16-bit pieces
// forward 178 without, 212 with, for what it takes to pair registers).
template <typename T, bool WIDE, int E, int LANES, bool PACKED>
struct RowLanes {
    using P = Piece<T, WIDE>;
    using Raw = typename P::Raw;
    static constexpr int V = P::V, N = E / V;
    static_assert(E % V == 0 && E % 2 == 0);
    __device__ __forceinline__ static float2 mul(float2 a, float2 b) { return PACKED ? mul2(a, b) : make_float2(a.x * b.x, a.y * b.y); }
    __device__ __forceinline__ static float2 add(float2 a, float2 b) { return PACKED ? add2(a, b) : make_float2(a.x + b.x, a.y + b.y); }
    __device__ __forceinline__ static float2 fma(float2 a, float2 b, float2 c) { return PACKED ? fma2(a, b, c) : make_float2(fmaf(a.x, b.x, c.x), fmaf(a.y, b.y, c.y)); }
    __device__ __forceinline__ static float2 two(const float (&v)[E], int e) { return make_float2(v[e], v[e + 1]); }
    __device__ __forceinline__ static void set(float (&v)[E], int e, float2 q) { v[e] = q.x, v[e + 1] = q.y; }
    template <typename F>
    __device__ __forceinline__ static void each(F f) {
#pragma unroll
        for (int e = 0; e < E; e += 2) f(e);
    }
    int l, c, whole;                   // pieces that all lanes of a row have
    float per;                         // 1 / c
    bool tail, there;                  // whether this lane has the piece behind the whole ones; whether its row is
    long long first;                   // the row's first value
    __device__ __forceinline__ RowLanes(const NormArgs& a) {
        l = (threadIdx.x & 31) & (LANES - 1), c = a.c, whole = c / V / LANES;
        per = 1.f / (float)c;
        tail = l + whole * LANES < c / V;
    }
    __device__ __forceinline__ void at(long long row, long long rows) { there = row < rows, first = row * c; }
    __device__ __forceinline__ int channel(int i) const { return (l + i * LANES) * V; }
    __device__ __forceinline__ bool has(int i) const { return i < whole || (i == whole && tail); }
    __device__ __forceinline__ void fetch(Raw (&q)[N], const void* from) const {
        const T* p = static_cast<const T*>(from) + first + l * V;
#pragma unroll
        for (int i = 0; i < N; i++) {
            q[i] = P::nothing();
            if (there && has(i)) q[i] = *reinterpret_cast<const Raw*>(p + i * LANES * V);
        }
    }
    __device__ __forceinline__ void values(float (&v)[E], const Raw (&q)[N]) const {
#pragma unroll
        for (int i = 0; i < N; i++) {
            P::values(v + i * V, q[i]);
        }
    }
    __device__ __forceinline__ void store(void* to, const float (&v)[E]) const {
        T* p = static_cast<T*>(to) + first + l * V;
#pragma unroll
        for (int i = 0; i < N; i++) {
            if (there && has(i)) P::store(p + i * LANES * V, v + i * V);
        }
    }
    // f(element, the vector's value for it) of pairs; a lane without a channel gets another channel's
    template <typename F>
    __device__ __forceinline__ void with(const float* vector, F f) const {
        float w[E];
#pragma unroll
        for (int i = 0; i < N; i++) P::shared(w + i * V, vector + min(channel(i), c - V));
#pragma unroll
        for (int e = 0; e < E; e += 2) f(e, make_float2(w[e], w[e + 1]));
    }
    __device__ __forceinline__ void times(float (&v)[E], const float* vector) const {
        with(vector, [&](int e, float2 w) { set(v, e, mul(two(v, e), w)); });
    }
    __device__ __forceinline__ void plus(float (&v)[E], const float* vector) const {
        with(vector, [&](int e, float2 w) { set(v, e, add(two(v, e), w)); });
    }
    __device__ __forceinline__ float sum(float v) const {   // of the row's lanes, the same in all of them
#pragma unroll
        for (int o = 16; o; o >>= 1)
            if (o < LANES) v += __shfl_xor_sync(~0u, v, o);
        return v;
    }
    // a[e] b[e] (or a[e]) summed over the row's channels.  (What lanes without a channel hold is never summed nor stored.)
    template <bool PRODUCT>
    __device__ __forceinline__ float sum_of(const float (&a)[E], const float (&b)[E]) const {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < N; i++) {
            if constexpr (V == 1) {
                s = has(i) ? (PRODUCT ? fmaf(a[i], b[i], s) : s + a[i]) : s;
            } else {
                float2 p = make_float2(0.f, 0.f);
#pragma unroll
                for (int e = i * V; e < i * V + V; e += 2) p = PRODUCT ? fma(two(a, e), two(b, e), p) : add(p, two(a, e));
                s += has(i) ? p.x + p.y : 0.f;
            }
        }
        return sum(s);
    }
    // v to its normed form without weight and bias; returns the reciprocal deviation.
    __device__ __forceinline__ float normalise(float (&v)[E], int kind, float eps) const {
        if (kind == PL_NORM_LAYER) {
            const float mean = sum_of<false>(v, v) * per;
            each([&](int e) { set(v, e, add(two(v, e), make_float2(-mean, -mean))); });
        }
        const float rstd = rsqrtf(fmaf(sum_of<true>(v, v), per, eps));
        each([&](int e) { set(v, e, mul(two(v, e), make_float2(rstd, rstd))); });
        return rstd;
    }
    // d, the gradient of the normed form, to that of what went in: rstd (d - mean(d) - hat mean(d hat))
    __device__ __forceinline__ void back(float (&d)[E], const float (&hat)[E], float rstd, int kind) const {
        const float q = -sum_of<true>(d, hat) * per;
        if (kind == PL_NORM_LAYER) {
            const float s = -sum_of<false>(d, d) * per;
            each([&](int e) { set(d, e, add(two(d, e), make_float2(s, s))); });
        }
        each([&](int e) { set(d, e, mul(fma(two(hat, e), make_float2(q, q), two(d, e)), make_float2(rstd, rstd))); });
    }
    // mask[e]: all ones where element e stays, else zero.  Values are counted through the whole tensor.  Single values: the words of the warp's
    // rows, which follow one another, by way of shared memory (a word for every value by its own lane would make each four times).
    __device__ __forceinline__ void kept(u32 (&mask)[E], const Philox& random, u32 threshold, long long warp_first, uint4* words_s) const {
        if constexpr (WIDE) {
#pragma unroll
            for (int i = 0; i < N; i++)
#pragma unroll
                for (int j = 0; j < V; j += 4) {
                    const uint4 w = random.words((u64)(first + channel(i) + j) >> 2);
                    mask[i * V + j] = w.x >= threshold ? ~0u : 0u, mask[i * V + j + 1] = w.y >= threshold ? ~0u : 0u;
                    mask[i * V + j + 2] = w.z >= threshold ? ~0u : 0u, mask[i * V + j + 3] = w.w >= threshold ? ~0u : 0u;
                }
        } else {
            const u64 quad = (u64)warp_first >> 2;
            const int count = (int)(((u64)warp_first + (32 / LANES) * c + 3) / 4 - quad), lane = threadIdx.x & 31;
            __syncwarp();   // the last rows' words have been read
            for (int q = lane; q < count; q += 32) words_s[q] = random.words(quad + q);
            __syncwarp();
            const u32* word = reinterpret_cast<const u32*>(words_s) + (int)(first - (long long)(quad << 2)) + l;
#pragma unroll
            for (int i = 0; i < N; i++) {
                mask[i] = there && has(i) && word[i * LANES] >= threshold ? ~0u : 0u;
            }
        }
    }
    __device__ __forceinline__ void drop(float (&v)[E], const u32 (&mask)[E], float scale) const {   // what is dropped is zero, whatever it was
        each([&](int e) {
            const float2 q = mul(two(v, e), make_float2(scale, scale));
            v[e] = __uint_as_float(__float_as_uint(q.x) & mask[e]), v[e + 1] = __uint_as_float(__float_as_uint(q.y) & mask[e + 1]);
        });
    }
};
// Quads of words that the rows of a warp may need: 32 E values at most, not begun at a quad's first one.
__host__ __device__ constexpr int norm_words(int e) { return 8 * e + 2; }

__device__ __forceinline__ void norm_vectors_to(float* vectors_s, const NormArgs& a) {
    for (int w = 0; w < NORM_VECTORS; w++)
        if (a.vectors[w])
            for (int i = threadIdx.x; i < a.c; i += NORM_THREADS) vectors_s[w * NORM_MOST + i] = load_weight(a.vectors[w], i, a.vector_dtype);
    __syncthreads();
}

// CTAs of an SM: where nothing is dropped four of 16-bit rows (2 470 000 x 256: 227 us with three, 202), with the generator's keys three.  Single values of more than 256
// channels: one, whose threads have registers for a row (150 000 x 511 floats, residual and two norms: 241 us; with two, which spilled some 300 bytes a thread, 837).
template <typename T, bool WIDE, int E, int LANES, bool DROPS>
__global__ void __launch_bounds__(NORM_THREADS, E > 8 ? (WIDE ? 2 : 1) : WIDE && sizeof(T) == 2 && !DROPS ? 4 : 1) norm_forward(const __grid_constant__ NormArgs a) {
    __shared__ __align__(16) float vectors_s[NORM_VECTORS * NORM_MOST];
    __shared__ uint4 words_s[WIDE || !DROPS ? 1 : NORM_WARPS * norm_words(E)];
    norm_vectors_to(vectors_s, a);
    using Row = RowLanes<T, WIDE, E, LANES, !(WIDE && sizeof(T) == 2)>;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const Philox random(a.drop);
    Row r(a);
    const int per_warp = 32 / LANES, own = lane / LANES;
    const long long step = (long long)gridDim.x * NORM_WARPS * per_warp;
    // A warp's next rows are on their way while these are worked on.
    typename Row::Raw next_x[Row::N], next_residual[Row::N], next_gate[Row::N];
    auto fetch = [&](long long r0) {
        r.at(r0 + own, a.rows);
        r.fetch(next_x, a.x);
        if (a.residual) r.fetch(next_residual, a.residual);
        if (a.gate) r.fetch(next_gate, a.gate);
    };
    long long r0 = ((long long)blockIdx.x * NORM_WARPS + warp) * per_warp;
    if (r0 < a.rows) fetch(r0);
    for (; r0 < a.rows; r0 += step) {
        float v[E], residual[E], gate[E];
        r.values(v, next_x);
        if (a.residual) r.values(residual, next_residual);
        if (a.gate) r.values(gate, next_gate);
        fetch(r0 + step);
        r.at(r0 + own, a.rows);
        if (a.after) {
            r.normalise(v, a.after, a.eps_after);
            if (a.vectors[NORM_WA]) r.times(v, vectors_s + NORM_WA * NORM_MOST);
            if (a.vectors[NORM_BA]) r.plus(v, vectors_s + NORM_BA * NORM_MOST);
        }
        if constexpr (DROPS) {
            u32 mask[E];
            r.kept(mask, random, a.drop.threshold, r0 * a.c, words_s + (WIDE ? 0 : warp * norm_words(E)));
            r.drop(v, mask, a.drop.scale);
        }
        if (a.gate) r.each([&](int e) { r.set(v, e, r.mul(r.two(v, e), r.two(gate, e))); });
        else if (a.vectors[NORM_GATE]) r.times(v, vectors_s + NORM_GATE * NORM_MOST);
        if (a.residual) r.each([&](int e) { r.set(v, e, r.fma(make_float2(a.scale, a.scale), r.two(residual, e), r.two(v, e))); });
        if (a.h) r.store(a.h, v);
        if (a.before) {
            r.normalise(v, a.before, a.eps_before);
            if (a.vectors[NORM_WB]) r.times(v, vectors_s + NORM_WB * NORM_MOST);
            if (a.vectors[NORM_BB]) r.plus(v, vectors_s + NORM_BB * NORM_MOST);
            r.store(a.y, v);
        }
    }
}

template <typename T, bool WIDE, int E, int LANES, bool AFTER, bool BEFORE>
__global__ void __launch_bounds__(NORM_THREADS, E <= 8 ? 2 : 1) norm_backward(const __grid_constant__ NormArgs a) {
    __shared__ __align__(16) float vectors_s[NORM_VECTORS * NORM_MOST];
    __shared__ uint4 words_s[WIDE ? 1 : NORM_WARPS * norm_words(E)];
    norm_vectors_to(vectors_s, a);
    using Row = RowLanes<T, WIDE, E, LANES, true>;
    constexpr bool AHEAD = WIDE && sizeof(T) == 2 && E <= 8;   // room for the next rows as they come
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const bool drops = a.drop.threshold != 0;
    const Philox random(a.drop);
    Row r(a);
    const int per_warp = 32 / LANES, own = lane / LANES;
    const long long step = (long long)gridDim.x * NORM_WARPS * per_warp;
    float sum_wa[E], sum_ba[E], sum_wb[E], sum_bb[E], sum_gate[E];   // (of a norm that is there both, a bias or not; with two norms a part of all this spills, see above)
#pragma unroll
    for (int e = 0; e < E; e++) sum_wa[e] = sum_ba[e] = sum_wb[e] = sum_bb[e] = sum_gate[e] = 0.f;
    typename Row::Raw raw_x[Row::N], raw_residual[Row::N], raw_gate[Row::N], raw_dh[Row::N], raw_dy[Row::N];
    auto fetch = [&](long long r0) {
        r.at(r0 + own, a.rows);
        if (a.x) r.fetch(raw_x, a.x);
        if (a.gate) r.fetch(raw_gate, a.gate);
        if (a.dh) r.fetch(raw_dh, a.dh);
        if constexpr (BEFORE) {
            if (a.residual) r.fetch(raw_residual, a.residual);
            r.fetch(raw_dy, a.dy);
        }
    };
    long long r0 = ((long long)blockIdx.x * NORM_WARPS + warp) * per_warp;
    if (AHEAD && r0 < a.rows) fetch(r0);
    for (; r0 < a.rows; r0 += step) {
        if (!AHEAD) fetch(r0);
        float x[E], h[E], gate[E], d[E], dy[E], rstd = 0.f;
        if (a.x) r.values(x, raw_x);
        else r.each([&](int e) { x[e] = x[e + 1] = 0.f; });
        if (a.dh) r.values(d, raw_dh);
        else r.each([&](int e) { d[e] = d[e + 1] = 0.f; });
        if constexpr (BEFORE) {
            if (a.residual) r.values(h, raw_residual);
            else r.each([&](int e) { h[e] = h[e + 1] = 0.f; });
            r.values(dy, raw_dy);
        }
        if (a.gate) r.values(gate, raw_gate);
        else if (a.vectors[NORM_GATE]) r.with(vectors_s + NORM_GATE * NORM_MOST, [&](int e, float2 w) { r.set(gate, e, w); });
        else r.each([&](int e) { gate[e] = gate[e + 1] = 1.f; });
        if (AHEAD) {
            fetch(r0 + step);
            r.at(r0 + own, a.rows);
        }
        u32 mask[E];
        if (drops) r.kept(mask, random, a.drop.threshold, r0 * a.c, words_s + (WIDE ? 0 : warp * norm_words(E)));
        if constexpr (AFTER) rstd = r.normalise(x, a.after, a.eps_after);   // x is x^ from here on
        float v[E];
        r.each([&](int e) { r.set(v, e, r.two(x, e)); });
        if constexpr (AFTER) {
            if (a.vectors[NORM_WA]) r.times(v, vectors_s + NORM_WA * NORM_MOST);
            if (a.vectors[NORM_BA]) r.plus(v, vectors_s + NORM_BA * NORM_MOST);
        }
        if (drops) r.drop(v, mask, a.drop.scale);
        if constexpr (BEFORE) {
            r.each([&](int e) { r.set(h, e, r.fma(make_float2(a.scale, a.scale), r.two(h, e), r.mul(r.two(v, e), r.two(gate, e)))); });
            const float rstd_h = r.normalise(h, a.before, a.eps_before);
            if (a.wanted >> NORM_WB & 1) r.each([&](int e) { r.set(sum_wb, e, r.fma(r.two(dy, e), r.two(h, e), r.two(sum_wb, e))); });
            if (a.wanted >> NORM_BB & 1) r.each([&](int e) { r.set(sum_bb, e, r.add(r.two(sum_bb, e), r.two(dy, e))); });
            if (a.vectors[NORM_WB]) r.times(dy, vectors_s + NORM_WB * NORM_MOST);
            r.back(dy, h, rstd_h, a.before);
            r.each([&](int e) { r.set(d, e, r.add(r.two(d, e), r.two(dy, e))); });
        }
        if (a.dresidual) {
            float t[E];
            r.each([&](int e) { r.set(t, e, r.mul(make_float2(a.scale, a.scale), r.two(d, e))); });
            r.store(a.dresidual, t);
        }
        if (a.dgate) {
            float t[E];
            r.each([&](int e) { r.set(t, e, r.mul(r.two(d, e), r.two(v, e))); });
            r.store(a.dgate, t);
        } else if (a.wanted >> NORM_GATE & 1) {
            r.each([&](int e) { r.set(sum_gate, e, r.fma(r.two(d, e), r.two(v, e), r.two(sum_gate, e))); });
        }
        if (a.gate || a.vectors[NORM_GATE]) r.each([&](int e) { r.set(d, e, r.mul(r.two(d, e), r.two(gate, e))); });
        if (drops) r.drop(d, mask, a.drop.scale);
        if constexpr (AFTER) {
            if (a.wanted >> NORM_WA & 1) r.each([&](int e) { r.set(sum_wa, e, r.fma(r.two(d, e), r.two(x, e), r.two(sum_wa, e))); });
            if (a.wanted >> NORM_BA & 1) r.each([&](int e) { r.set(sum_ba, e, r.add(r.two(sum_ba, e), r.two(d, e))); });
            if (a.vectors[NORM_WA]) r.times(d, vectors_s + NORM_WA * NORM_MOST);
            r.back(d, x, rstd, a.after);
        }
        if (a.dx) r.store(a.dx, d);
    }
    if (!a.shares) return;
    // The CTA's sums: of the rows of a warp by shuffles, of the warps by way of shared memory, a vector at a time.
    __shared__ float warps_s[NORM_WARPS][NORM_MOST];
    float* share = a.shares + (long long)blockIdx.x * NORM_VECTORS * a.c;
    auto gather = [&](const float (&s)[E], int which) {
        if (!(a.wanted >> which & 1)) return;
        __syncthreads();
#pragma unroll
        for (int e = 0; e < E; e++) {
            float t = s[e];
#pragma unroll
            for (int o = 1; o < 32; o <<= 1)
                if (o >= LANES) t += __shfl_xor_sync(~0u, t, o);
            if (lane < LANES && r.has(e / Row::V)) warps_s[warp][r.channel(e / Row::V) + e % Row::V] = t;
        }
        __syncthreads();
        for (int i = threadIdx.x; i < a.c; i += NORM_THREADS) {
            float t = 0.f;
#pragma unroll
            for (int w = 0; w < NORM_WARPS; w++) t += warps_s[w][i];
            share[which * a.c + i] = t;
        }
    };
    if constexpr (AFTER) gather(sum_wa, NORM_WA), gather(sum_ba, NORM_BA);
    if constexpr (BEFORE) gather(sum_wb, NORM_WB), gather(sum_bb, NORM_BB);
    gather(sum_gate, NORM_GATE);
}

// The vectors' gradients from the CTAs' shares: 32 values a CTA, 8 warps with an eighth of the shares each.  In doubles: floats' chain of 74 was as much off
// as all that went before (a million rows of 32 channels: 2e-7, 1.3e-7 in doubles).
struct NormSums {
    const float* shares;
    int ctas, c, dtype;
    void* to[NORM_VECTORS];   // NULL: not wanted
};
__device__ __forceinline__ void store_weight(void* w, int i, int dtype, float v) {
    if (dtype == PL_F32) static_cast<float*>(w)[i] = v;
    else if (dtype == PL_F16) static_cast<__half*>(w)[i] = __float2half_rn(v);
    else static_cast<__nv_bfloat16*>(w)[i] = __float2bfloat16_rn(v);
}
static __global__ void __launch_bounds__(NORM_THREADS) norm_sums(const __grid_constant__ NormSums a) {
    __shared__ double part_s[NORM_WARPS][33];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, which = blockIdx.y, i = blockIdx.x * 32 + lane;
    if (!a.to[which]) return;
    double t = 0.0;
    if (i < a.c)
        for (int s = warp; s < a.ctas; s += NORM_WARPS) t += (double)a.shares[((long long)s * NORM_VECTORS + which) * a.c + i];
    part_s[warp][lane] = t;
    __syncthreads();
    if (warp || i >= a.c) return;
#pragma unroll
    for (int w = 1; w < NORM_WARPS; w++) t += part_s[w][lane];
    store_weight(a.to[which], i, a.dtype, (float)t);
}

// out = s residual + x keep / (1 - p), value by value; scaled: s x besides (the residual's gradient, where x is that of out).  Either may be NULL.
struct DropArgs {
    long long n;
    const void *x, *residual;
    void *out, *scaled;
    float scale;
    Dropout drop;
};
// Two pieces a thread at a time, both on their way before the first is worked on (88 million floats and a residual: 164 us, one 186, four 170; bfloat16 values take 118, issue slots 62 % busy: the generator's some 40 products and exclusive ors for four).
constexpr int DROP_PIECES = 2;
template <typename T, bool WIDE>
__global__ void __launch_bounds__(256) drop_values(const __grid_constant__ DropArgs a) {
    using P = Piece<T, true>;
    constexpr int V = P::V, U = DROP_PIECES;
    const Philox random(a.drop);
    const T *x = static_cast<const T*>(a.x), *residual = static_cast<const T*>(a.residual);
    T *out = static_cast<T*>(a.out), *scaled = static_cast<T*>(a.scaled);
    const long long step = (long long)gridDim.x * 256 * V * U;
    for (long long i0 = (long long)blockIdx.x * 256 * V * U + threadIdx.x * V; i0 < a.n; i0 += step) {
        uint4 raw[U], raw_residual[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const long long i = i0 + u * 256 * V;
            if (WIDE && i + V <= a.n) {
                raw[u] = *reinterpret_cast<const uint4*>(x + i);
                if (residual) raw_residual[u] = *reinterpret_cast<const uint4*>(residual + i);
            }
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            const long long i = i0 + u * 256 * V;
            if (i >= a.n) break;
            const int count = (int)min((long long)V, a.n - i);
            const bool whole = WIDE && count == V;
            float v[V], q[V];
            if (whole) {
                P::values(v, raw[u]);
                if (residual) P::values(q, raw_residual[u]);
            } else {
#pragma unroll
                for (int j = 0; j < V; j++) {
                    v[j] = j < count ? to_float(x[i + j]) : 0.f;
                    if (residual) q[j] = j < count ? to_float(residual[i + j]) : 0.f;
                }
            }
            if (scaled) {
                float t[V];
#pragma unroll
                for (int j = 0; j < V; j++) t[j] = a.scale * v[j];
                if (whole) P::store(scaled + i, t);
                else
                    for (int j = 0; j < V; j++)
                        if (j < count) scaled[i + j] = from_float<T>(t[j]);
            }
            if (!out) continue;
#pragma unroll
            for (int j = 0; j < V; j += 4) {
                const uint4 w = random.words((u64)(i + j) >> 2);
                v[j] = w.x >= a.drop.threshold ? v[j] * a.drop.scale : 0.f;
                v[j + 1] = w.y >= a.drop.threshold ? v[j + 1] * a.drop.scale : 0.f;
                v[j + 2] = w.z >= a.drop.threshold ? v[j + 2] * a.drop.scale : 0.f;
                v[j + 3] = w.w >= a.drop.threshold ? v[j + 3] * a.drop.scale : 0.f;
            }
            if (residual) {
#pragma unroll
                for (int j = 0; j < V; j++) v[j] = fmaf(a.scale, q[j], v[j]);
            }
            if (whole) P::store(out + i, v);
            else
                for (int j = 0; j < V; j++)
                    if (j < count) out[i + j] = from_float<T>(v[j]);
        }
    }
}

}  // namespace pl
