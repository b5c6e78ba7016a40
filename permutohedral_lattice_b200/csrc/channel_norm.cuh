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
    int c, lanes;                      // channels; lanes of a row, a power of two
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

// A row in registers: E values a lane, in pieces of V that follow one another in memory, piece i of lane l the (l + i lanes)-th.
// V is 16 bytes where rows are whole pieces on 16-byte boundaries, else one value: 21 channels of floats, side by side, take as
// many sectors either way.
template <typename T, bool WIDE>
struct Piece {
    static constexpr int V = WIDE ? 16 / (int)sizeof(T) : 1;
    __device__ __forceinline__ static void load(float* v, const T* p) {
        if constexpr (!WIDE) {
            v[0] = to_float(*p);
        } else if constexpr (sizeof(T) == 4) {
            const float4 q = *reinterpret_cast<const float4*>(p);
            v[0] = q.x, v[1] = q.y, v[2] = q.z, v[3] = q.w;
        } else {
            const uint4 q = *reinterpret_cast<const uint4*>(p);
            const T* e = reinterpret_cast<const T*>(&q);
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = to_float(e[j]);
        }
    }
    __device__ __forceinline__ static void store(T* p, const float* v) {
        if constexpr (!WIDE) {
            *p = from_float<T>(v[0]);
        } else if constexpr (sizeof(T) == 4) {
            *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
        } else {
            uint4 q;
            T* e = reinterpret_cast<T*>(&q);
#pragma unroll
            for (int j = 0; j < 8; j++) e[j] = from_float<T>(v[j]);
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

template <typename T, bool WIDE, int E>
struct RowLanes {
    using P = Piece<T, WIDE>;
    static constexpr int V = P::V, N = E / V;
    static_assert(E % V == 0);
    int lanes, l, c;
    bool there;
    long long first;   // the row's first value
    __device__ __forceinline__ int channel(int i) const { return (l + i * lanes) * V; }
    __device__ __forceinline__ bool live(int i) const { return there && channel(i) < c; }
    __device__ __forceinline__ void load(float (&v)[E], const void* from) const {
        const T* p = static_cast<const T*>(from) + first;
#pragma unroll
        for (int i = 0; i < N; i++) {
#pragma unroll
            for (int j = 0; j < V; j++) v[i * V + j] = 0.f;
            if (live(i)) P::load(v + i * V, p + channel(i));
        }
    }
    __device__ __forceinline__ void store(void* to, const float (&v)[E]) const {
        T* p = static_cast<T*>(to) + first;
#pragma unroll
        for (int i = 0; i < N; i++)
            if (live(i)) P::store(p + channel(i), v + i * V);
    }
    // f(element, the vector's value for it); a lane without a channel gets another channel's
    template <typename F>
    __device__ __forceinline__ void with(const float* vector, F f) const {
#pragma unroll
        for (int i = 0; i < N; i++) {
            float w[V];
            P::shared(w, vector + min(channel(i), c - V));
#pragma unroll
            for (int j = 0; j < V; j++) f(i * V + j, w[j]);
        }
    }
    __device__ __forceinline__ float sum(float v) const {   // of the row's lanes, the same in all of them
        for (int o = lanes >> 1; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
        return v;
    }
    // v to its normed form without weight and bias, zero where there is no channel; returns the reciprocal deviation
    __device__ __forceinline__ float normalise(float (&v)[E], int kind, float eps) const {
        const float per = 1.f / (float)c;
        if (kind == PL_NORM_LAYER) {
            float s = 0.f;
#pragma unroll
            for (int e = 0; e < E; e++) s += v[e];
            const float mean = sum(s) * per;
#pragma unroll
            for (int e = 0; e < E; e++) v[e] = live(e / V) ? v[e] - mean : 0.f;
        }
        float q = 0.f;
#pragma unroll
        for (int e = 0; e < E; e++) q = fmaf(v[e], v[e], q);
        const float rstd = rsqrtf(fmaf(sum(q), per, eps));
#pragma unroll
        for (int e = 0; e < E; e++) v[e] *= rstd;
        return rstd;
    }
    // d, the gradient of the normed form (zero where there is no channel), to that of what went in
    __device__ __forceinline__ void back(float (&d)[E], const float (&hat)[E], float rstd, int kind) const {
        const float per = 1.f / (float)c;
        float s = 0.f, q = 0.f;
#pragma unroll
        for (int e = 0; e < E; e++) s += d[e], q = fmaf(d[e], hat[e], q);
        q = sum(q) * per;
        s = kind == PL_NORM_LAYER ? sum(s) * per : 0.f;
#pragma unroll
        for (int e = 0; e < E; e++) d[e] = rstd * (d[e] - s - hat[e] * q);
    }
    // Bit e: element e stays.  Values are counted through the whole tensor.  Single values: the words of the warp's rows, which follow one
    // another, by way of shared memory (a word for every value by its own lane would make each four times).
    __device__ __forceinline__ u32 kept(const Philox& random, u32 threshold, long long warp_first, uint4* words_s) const {
        u32 bits = 0;
        if constexpr (WIDE) {
#pragma unroll
            for (int i = 0; i < N; i++)
#pragma unroll
                for (int j = 0; j < V; j += 4) {
                    const uint4 w = random.words((u64)(first + channel(i) + j) >> 2);
                    bits |= ((u32)(w.x >= threshold) | (u32)(w.y >= threshold) << 1 | (u32)(w.z >= threshold) << 2 | (u32)(w.w >= threshold) << 3) << (i * V + j);
                }
        } else {
            const u64 quad = (u64)warp_first >> 2;
            const int count = (int)(((u64)warp_first + (32 / lanes) * c + 3) / 4 - quad), lane = threadIdx.x & 31;
            __syncwarp();   // the last rows' words have been read
            for (int q = lane; q < count; q += 32) words_s[q] = random.words(quad + q);
            __syncwarp();
            const u32* word = reinterpret_cast<const u32*>(words_s) + (first - (long long)(quad << 2));
#pragma unroll
            for (int i = 0; i < N; i++)
                if (live(i)) bits |= (u32)(word[channel(i)] >= threshold) << i;
        }
        return bits;
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

template <typename T, bool WIDE, int E>
__global__ void __launch_bounds__(NORM_THREADS) norm_forward(const __grid_constant__ NormArgs a) {
    __shared__ __align__(16) float vectors_s[NORM_VECTORS * NORM_MOST];
    __shared__ uint4 words_s[WIDE ? 1 : NORM_WARPS * norm_words(E)];
    norm_vectors_to(vectors_s, a);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, per_warp = 32 / a.lanes;
    const bool drops = a.drop.threshold != 0;
    const Philox random(a.drop);
    for (long long r0 = ((long long)blockIdx.x * NORM_WARPS + warp) * per_warp; r0 < a.rows; r0 += (long long)gridDim.x * NORM_WARPS * per_warp) {
        const long long row = r0 + lane / a.lanes;
        const RowLanes<T, WIDE, E> r{a.lanes, lane & (a.lanes - 1), a.c, row < a.rows, row * a.c};
        float v[E], residual[E], gate[E];
        r.load(v, a.x);
        if (a.residual) r.load(residual, a.residual);
        if (a.gate) r.load(gate, a.gate);
        if (a.after) {
            r.normalise(v, a.after, a.eps_after);
            if (a.vectors[NORM_WA]) r.with(vectors_s + NORM_WA * NORM_MOST, [&](int e, float w) { v[e] *= w; });
            if (a.vectors[NORM_BA]) r.with(vectors_s + NORM_BA * NORM_MOST, [&](int e, float w) { v[e] += w; });
        }
        if (drops) {
            const u32 kept = r.kept(random, a.drop.threshold, r0 * a.c, words_s + (WIDE ? 0 : warp * norm_words(E)));
#pragma unroll
            for (int e = 0; e < E; e++) v[e] = kept >> e & 1 ? v[e] * a.drop.scale : 0.f;
        }
        if (a.gate) {
#pragma unroll
            for (int e = 0; e < E; e++) v[e] *= gate[e];
        } else if (a.vectors[NORM_GATE]) {
            r.with(vectors_s + NORM_GATE * NORM_MOST, [&](int e, float w) { v[e] *= w; });
        }
        if (a.residual) {
#pragma unroll
            for (int e = 0; e < E; e++) v[e] = fmaf(a.scale, residual[e], v[e]);
        }
        if (a.h) r.store(a.h, v);
        if (a.before) {
#pragma unroll
            for (int e = 0; e < E; e++) v[e] = r.live(e / r.V) ? v[e] : 0.f;   // (a bias is no channel's there)
            r.normalise(v, a.before, a.eps_before);
            if (a.vectors[NORM_WB]) r.with(vectors_s + NORM_WB * NORM_MOST, [&](int e, float w) { v[e] *= w; });
            if (a.vectors[NORM_BB]) r.with(vectors_s + NORM_BB * NORM_MOST, [&](int e, float w) { v[e] += w; });
            r.store(a.y, v);
        }
    }
}

template <typename T, bool WIDE, int E, bool AFTER, bool BEFORE>
__global__ void __launch_bounds__(NORM_THREADS) norm_backward(const __grid_constant__ NormArgs a) {
    __shared__ __align__(16) float vectors_s[NORM_VECTORS * NORM_MOST];
    __shared__ uint4 words_s[WIDE ? 1 : NORM_WARPS * norm_words(E)];
    norm_vectors_to(vectors_s, a);
    using Row = RowLanes<T, WIDE, E>;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, per_warp = 32 / a.lanes;
    const bool drops = a.drop.threshold != 0;
    const Philox random(a.drop);
    float sum_wa[E], sum_ba[E], sum_wb[E], sum_bb[E], sum_gate[E];   // (those without a use take no registers)
#pragma unroll
    for (int e = 0; e < E; e++) sum_wa[e] = sum_ba[e] = sum_wb[e] = sum_bb[e] = sum_gate[e] = 0.f;
    for (long long r0 = ((long long)blockIdx.x * NORM_WARPS + warp) * per_warp; r0 < a.rows; r0 += (long long)gridDim.x * NORM_WARPS * per_warp) {
        const long long row = r0 + lane / a.lanes;
        const Row r{a.lanes, lane & (a.lanes - 1), a.c, row < a.rows, row * a.c};
        float x[E], h[E], gate[E], d[E], dy[E], rstd = 0.f;
        if (a.x) r.load(x, a.x);
        else {
#pragma unroll
            for (int e = 0; e < E; e++) x[e] = 0.f;
        }
        if (a.gate) r.load(gate, a.gate);
        if (a.dh) r.load(d, a.dh);
        else {
#pragma unroll
            for (int e = 0; e < E; e++) d[e] = 0.f;
        }
        if constexpr (BEFORE) {
            if (a.residual) r.load(h, a.residual);
            else {
#pragma unroll
                for (int e = 0; e < E; e++) h[e] = 0.f;
            }
            r.load(dy, a.dy);
        }
        u32 kept = ~0u;
        if (drops) kept = r.kept(random, a.drop.threshold, r0 * a.c, words_s + (WIDE ? 0 : warp * norm_words(E)));
        if (!a.gate) {
#pragma unroll
            for (int e = 0; e < E; e++) gate[e] = 1.f;
            if (a.vectors[NORM_GATE]) r.with(vectors_s + NORM_GATE * NORM_MOST, [&](int e, float w) { gate[e] = w; });
        }
        if constexpr (AFTER) rstd = r.normalise(x, a.after, a.eps_after);   // x is x^ from here on
        float v[E];
#pragma unroll
        for (int e = 0; e < E; e++) v[e] = x[e];
        if constexpr (AFTER) {
            if (a.vectors[NORM_WA]) r.with(vectors_s + NORM_WA * NORM_MOST, [&](int e, float w) { v[e] *= w; });
            if (a.vectors[NORM_BA]) r.with(vectors_s + NORM_BA * NORM_MOST, [&](int e, float w) { v[e] += w; });
        }
        if (drops) {
#pragma unroll
            for (int e = 0; e < E; e++) v[e] = kept >> e & 1 ? v[e] * a.drop.scale : 0.f;
        }
        if constexpr (BEFORE) {
#pragma unroll
            for (int e = 0; e < E; e++) h[e] = r.live(e / Row::V) ? fmaf(a.scale, h[e], v[e] * gate[e]) : 0.f;
            const float rstd_h = r.normalise(h, a.before, a.eps_before);
            if (a.shares) {
#pragma unroll
                for (int e = 0; e < E; e++) {
                    sum_wb[e] = fmaf(dy[e], h[e], sum_wb[e]);
                    sum_bb[e] += dy[e];
                }
            }
            if (a.vectors[NORM_WB]) r.with(vectors_s + NORM_WB * NORM_MOST, [&](int e, float w) { dy[e] *= w; });
            r.back(dy, h, rstd_h, a.before);
#pragma unroll
            for (int e = 0; e < E; e++) d[e] += r.live(e / Row::V) ? dy[e] : 0.f;   // (the mean is no channel's there)
        }
        if (a.dresidual) {
            float t[E];
#pragma unroll
            for (int e = 0; e < E; e++) t[e] = a.scale * d[e];
            r.store(a.dresidual, t);
        }
        if (a.dgate) {
            float t[E];
#pragma unroll
            for (int e = 0; e < E; e++) t[e] = d[e] * v[e];
            r.store(a.dgate, t);
        } else if (a.shares) {
#pragma unroll
            for (int e = 0; e < E; e++) sum_gate[e] = fmaf(d[e], v[e], sum_gate[e]);
        }
#pragma unroll
        for (int e = 0; e < E; e++) d[e] *= gate[e];
        if (drops) {
#pragma unroll
            for (int e = 0; e < E; e++) d[e] = kept >> e & 1 ? d[e] * a.drop.scale : 0.f;
        }
        if constexpr (AFTER) {
            if (a.shares) {
#pragma unroll
                for (int e = 0; e < E; e++) {
                    sum_wa[e] = fmaf(d[e], x[e], sum_wa[e]);
                    sum_ba[e] += d[e];
                }
            }
            if (a.vectors[NORM_WA]) r.with(vectors_s + NORM_WA * NORM_MOST, [&](int e, float w) { d[e] *= w; });
            r.back(d, x, rstd, a.after);
        }
        if (a.dx) r.store(a.dx, d);
    }
    if (!a.shares) return;
    // The CTA's sums: of the rows of a warp by shuffles, of the warps by way of shared memory, a vector at a time.
    __shared__ float warps_s[NORM_WARPS][NORM_MOST];
    float* share = a.shares + (long long)blockIdx.x * NORM_VECTORS * a.c;
    const Row r{a.lanes, lane & (a.lanes - 1), a.c, true, 0};
    auto gather = [&](const float (&s)[E], int which) {
        if (!(a.wanted >> which & 1)) return;
        __syncthreads();
#pragma unroll
        for (int e = 0; e < E; e++) {
            float t = s[e];
            for (int o = a.lanes; o < 32; o <<= 1) t += __shfl_xor_sync(~0u, t, o);
            if (lane < a.lanes && r.live(e / Row::V)) warps_s[warp][r.channel(e / Row::V) + e % Row::V] = t;
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

// The vectors' gradients from the CTAs' shares: 32 values a CTA, 8 warps with an eighth of the shares each.
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
    __shared__ float part_s[NORM_WARPS][33];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, which = blockIdx.y, i = blockIdx.x * 32 + lane;
    if (!a.to[which]) return;
    float t = 0.f;
    if (i < a.c)
        for (int s = warp; s < a.ctas; s += NORM_WARPS) t += a.shares[((long long)s * NORM_VECTORS + which) * a.c + i];
    part_s[warp][lane] = t;
    __syncthreads();
    if (warp || i >= a.c) return;
#pragma unroll
    for (int w = 1; w < NORM_WARPS; w++) t += part_s[w][lane];
    store_weight(a.to[which], i, a.dtype, t);
}

// out = s residual + x keep / (1 - p), value by value; scaled: s x besides (the residual's gradient, where x is that of out).  Either may be NULL.
struct DropArgs {
    long long n;
    const void *x, *residual;
    void *out, *scaled;
    float scale;
    Dropout drop;
};
template <typename T, bool WIDE>
__global__ void __launch_bounds__(256) drop_values(const __grid_constant__ DropArgs a) {
    using P = Piece<T, true>;
    constexpr int V = P::V;
    const Philox random(a.drop);
    const T *x = static_cast<const T*>(a.x), *residual = static_cast<const T*>(a.residual);
    T *out = static_cast<T*>(a.out), *scaled = static_cast<T*>(a.scaled);
    const long long step = (long long)gridDim.x * 256 * V;
    for (long long i = ((long long)blockIdx.x * 256 + threadIdx.x) * V; i < a.n; i += step) {
        const int count = (int)min((long long)V, a.n - i);
        const bool whole = WIDE && count == V;
        float v[V], q[V];
        if (whole) {
            P::load(v, x + i);
            if (residual) P::load(q, residual + i);
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

}  // namespace pl
