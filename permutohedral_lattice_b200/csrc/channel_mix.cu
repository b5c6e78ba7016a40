// Products of channels with bias, residual and activation, their gradients, and activations in 8 bits: the training side of
// the operators around the lattice filter (the C entry points at the end of include/pl_lattice.h).
//
//   z = x W [+ x2 W2] [+ bias] [+ s residual],   out = act(z)
//   dz = g (no activation), g [out > 0] (relu), out (g - sum_k g_k out_k) (softmax)
//   dresidual = s dz,  dx = dz W^T,  dx2 = dz W2^T,  dW = x^T dz,  dW2 = x2^T dz,  dbias = sum over rows of dz
//
// A translation unit of its own: nothing here has to round like the reference's geometry.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <algorithm>
#include <stdint.h>

#include "host_calls.h"

namespace pl {

typedef unsigned int u32;

constexpr int MIX_MOST = 128;   // channels of an input, and of the output
constexpr int PACK_BLOCK = 32;  // values that share an exponent

template <typename T>
__device__ __forceinline__ float to_float(T v) { return (float)v; }
template <typename T>
__device__ __forceinline__ T from_float(float v) { return (T)v; }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// ---------------------------------------------------------------------------------------------
// 8-bit blocks
// ---------------------------------------------------------------------------------------------
// Header of a block: e + 127 in the low byte (255: the block held an infinity or a NaN), bit 8: signed codes.  e is the least
// exponent >= -126 at which `most`, the largest magnitude's bits, is at most 255 (127) steps of 2^e: with most = 1.f 2^(E - 127)
// that is E - 134 (E - 133) if 1.f <= 255/128 (127/64), and one more if not; at most 120 (121), so that no code stands for
// more than float32 holds: codes saturate there.
__device__ __forceinline__ u32 block_header(u32 most, bool is_signed) {
    const int E = (int)(most >> 23);
    if (E == 255) return 255u;
    const u32 fraction = most & 0x7FFFFFu;
    int e = is_signed ? E - 133 + (fraction > 0x7E0000u ? 1 : 0) : E - 134 + (fraction > 0x7F0000u ? 1 : 0);
    e = min(max(e, -126), is_signed ? 121 : 120);
    return (u32)(e + 127) | (is_signed ? 256u : 0u);
}
__device__ __forceinline__ float power_of_two(int e) { return __int_as_float((e + 127) << 23); }   // -126 <= e <= 127
__device__ __forceinline__ int encode_value(float v, u32 header, bool keep_nonzero) {
    if ((header & 255u) == 255u) return 0;
    const int e = (int)(header & 255u) - 127;
    int code = __float2int_rn(v * power_of_two(-e));   // exact but for values far below half a step
    if (e >= 120) code = (header & 256u) ? min(max(code, -127), 127) : min(code, 255);
    if (keep_nonzero && code == 0 && v != 0.f) code = v < 0.f ? -1 : 1;
    return code & 255;
}
__device__ __forceinline__ float decode_value(u32 code, u32 header) {
    const u32 low = header & 255u;
    if (low == 255u) return __int_as_float(0x7FC00000);
    const int c = (header & 256u) ? (int)(signed char)code : (int)code;
    return (float)c * power_of_two((int)low - 127);
}

// A warp a block of 32 values.
template <typename T>
__global__ void __launch_bounds__(256) pack_blocks(uint8_t* __restrict__ codes, int16_t* __restrict__ scales,
                                                   const T* __restrict__ x, long long n, int keep_nonzero) {
    const int lane = threadIdx.x & 31;
    const long long blocks = (n + PACK_BLOCK - 1) / PACK_BLOCK;
    for (long long b = ((long long)blockIdx.x * 256 + threadIdx.x) >> 5; b < blocks; b += (long long)gridDim.x * 8) {
        const long long i = b * PACK_BLOCK + lane;
        const float v = i < n ? to_float(x[i]) : 0.f;
        const u32 most = __reduce_max_sync(~0u, __float_as_uint(v) & 0x7FFFFFFFu);
        const bool is_signed = __any_sync(~0u, v < 0.f);
        const u32 header = block_header(most, is_signed);
        if (i < n) codes[i] = (uint8_t)encode_value(v, header, keep_nonzero != 0);
        if (lane == 0) scales[b] = (int16_t)header;
    }
}

template <typename T>
__global__ void __launch_bounds__(256) unpack_blocks(T* __restrict__ x, const uint8_t* __restrict__ codes,
                                                     const int16_t* __restrict__ scales, long long n) {
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256)
        x[i] = from_float<T>(decode_value(codes[i], (u32)(uint16_t)scales[i / PACK_BLOCK]));
}

// ---------------------------------------------------------------------------------------------
// The products, a warp a row
// ---------------------------------------------------------------------------------------------
struct MixShape {
    long long rows;
    int k, k2, n, activation;
    float residual_scale;
};
struct Kept {   // an input as it is, or in 8 bits
    const void* full;
    const uint8_t* codes;
    const int16_t* scales;
};
template <typename T>
__device__ __forceinline__ float kept_value(const Kept& a, long long i) {
    return a.codes ? decode_value(a.codes[i], (u32)(uint16_t)a.scales[i / PACK_BLOCK])
                   : to_float(static_cast<const T*>(a.full)[i]);
}
__device__ __forceinline__ float warp_sum(float v) {
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
    return v;
}
__device__ __forceinline__ float warp_max(float v) {
    for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(~0u, v, o));
    return v;
}

template <typename T, typename W>
__global__ void __launch_bounds__(256)
mix_rows(MixShape m, T* __restrict__ out, const T* __restrict__ x, const T* __restrict__ x2, const W* __restrict__ weight,
         const W* __restrict__ weight2, const W* __restrict__ bias, const T* __restrict__ residual) {
    const int lane = threadIdx.x & 31;
    for (long long row = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); row < m.rows; row += (long long)gridDim.x * 8) {
        float z[4];
        bool nan = false;
        float top = -INFINITY;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int c = lane + 32 * j;
            float acc = 0.f;
            if (c < m.n) {
                for (int k = 0; k < m.k; k++) acc = fmaf(to_float(x[row * m.k + k]), to_float(weight[k * m.n + c]), acc);
                for (int k = 0; k < m.k2; k++) acc = fmaf(to_float(x2[row * m.k2 + k]), to_float(weight2[k * m.n + c]), acc);
                if (bias) acc += to_float(bias[c]);
                if (residual) acc = fmaf(m.residual_scale, to_float(residual[row * m.n + c]), acc);
                top = fmaxf(top, acc);
                nan |= acc != acc;
            }
            z[j] = acc;
        }
        if (m.activation == PL_ACT_SOFTMAX) {
            top = warp_max(top);
            nan = __any_sync(~0u, nan);
            float den = 0.f;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                z[j] = lane + 32 * j >= m.n ? 0.f : top == -INFINITY && !nan ? 0.f : expf(z[j] - top);
                den += z[j];
            }
            den = warp_sum(den);
            const float inv = den == 0.f ? 0.f : 1.f / den;
#pragma unroll
            for (int j = 0; j < 4; j++) z[j] *= inv;
        } else if (m.activation == PL_ACT_RELU) {
#pragma unroll
            for (int j = 0; j < 4; j++) z[j] = z[j] < 0.f ? 0.f : z[j];
        }
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (lane + 32 * j < m.n) out[row * m.n + lane + 32 * j] = from_float<T>(z[j]);
    }
}

// dz of every row (float, to the workspace), and what follows from a row alone.
template <typename T, typename W>
__global__ void __launch_bounds__(256)
mix_back_rows(MixShape m, float* __restrict__ dz_out, const T* __restrict__ grad, Kept out, const W* __restrict__ weight,
              const W* __restrict__ weight2, T* __restrict__ dx, T* __restrict__ dx2, T* __restrict__ dresidual) {
    __shared__ float dz_s[8][MIX_MOST];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (long long row = (long long)blockIdx.x * 8 + warp; row < m.rows; row += (long long)gridDim.x * 8) {
        float y[4], g[4], s = 0.f;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int c = lane + 32 * j;
            g[j] = c < m.n ? to_float(grad[row * m.n + c]) : 0.f;
            y[j] = c < m.n && m.activation != PL_ACT_NONE ? kept_value<T>(out, row * m.n + c) : 0.f;
            s = fmaf(y[j], g[j], s);
        }
        s = warp_sum(s);
        __syncwarp();
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int c = lane + 32 * j;
            if (c >= m.n) continue;
            const float dz = m.activation == PL_ACT_SOFTMAX ? y[j] * (g[j] - s)
                             : m.activation == PL_ACT_RELU  ? (y[j] > 0.f ? g[j] : 0.f)
                                                            : g[j];
            dz_s[warp][c] = dz;
            dz_out[row * m.n + c] = dz;
            if (dresidual) dresidual[row * m.n + c] = from_float<T>(m.residual_scale * dz);
        }
        __syncwarp();
        for (int k = lane; k < m.k + m.k2; k += 32) {
            const bool second = k >= m.k;
            if (second ? !dx2 : !dx) continue;
            const W* w = second ? weight2 + (k - m.k) * m.n : weight + k * m.n;
            float acc = 0.f;
            for (int c = 0; c < m.n; c++) acc = fmaf(dz_s[warp][c], to_float(w[c]), acc);
            if (second) dx2[row * m.k2 + k - m.k] = from_float<T>(acc);
            else dx[row * m.k + k] = from_float<T>(acc);
        }
        __syncwarp();
    }
}

// Element (k, c) of dW, dW2 and dbias: a CTA an element, sums in double in a fixed order.
template <typename T, typename W>
__global__ void __launch_bounds__(256)
mix_back_weights(MixShape m, const float* __restrict__ dz, Kept x, Kept x2, W* __restrict__ dweight, W* __restrict__ dweight2,
                 W* __restrict__ dbias) {
    __shared__ double part[256];
    const int k = blockIdx.x / m.n, c = blockIdx.x - k * m.n;
    W* to = k < m.k ? dweight + (size_t)k * m.n : k < m.k + m.k2 ? dweight2 + (size_t)(k - m.k) * m.n : dbias;
    if (k < m.k ? !dweight : k < m.k + m.k2 ? !dweight2 : !dbias) return;
    double sum = 0.0;
    for (long long r = threadIdx.x; r < m.rows; r += 256) {
        const float a = k < m.k ? kept_value<T>(x, r * m.k + k) : k < m.k + m.k2 ? kept_value<T>(x2, r * m.k2 + k - m.k) : 1.f;
        sum += (double)a * (double)dz[r * m.n + c];
    }
    part[threadIdx.x] = sum;
    __syncthreads();
    for (int o = 128; o; o >>= 1) {
        if (threadIdx.x < o) part[threadIdx.x] += part[threadIdx.x + o];
        __syncthreads();
    }
    if (threadIdx.x == 0) to[c] = from_float<W>((float)part[0]);
}

// ---------------------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------------------
static int check_shape(const pl_mix* m) {
    if (!m || m->rows < 0 || m->k < 1 || m->k2 < 0 || m->n < 1) return PL_INVALID_ARGUMENT;
    if (m->activation < PL_ACT_NONE || m->activation > PL_ACT_SOFTMAX) return PL_INVALID_ARGUMENT;
    if (m->dtype < PL_F32 || m->dtype > PL_BF16) return PL_INVALID_ARGUMENT;
    if (m->weight_dtype != PL_F32 && m->weight_dtype != m->dtype) return PL_INVALID_ARGUMENT;
    if (m->k > MIX_MOST || m->k2 > MIX_MOST || m->n > MIX_MOST) return PL_UNSUPPORTED_DIMS;
    if (m->rows > ((long long)1 << 40)) return PL_INVALID_ARGUMENT;
    return PL_OK;
}
static MixShape shape_of(const pl_mix* m) { return {m->rows, m->k, m->k2, m->n, m->activation, m->residual_scale}; }
static unsigned grid_for(long long items, long long per_cta, int ctas_per_sm) {
    return (unsigned)std::max(1ll, std::min((items + per_cta - 1) / per_cta, (long long)num_sms() * ctas_per_sm));
}

// CALL(T, W) for the types of values and weights
#define PL_MIX_TYPES(dtype, weight_dtype, CALL)                                                       \
    ((dtype) == PL_F32   ? CALL(float, float)                                                         \
     : (dtype) == PL_F16 ? ((weight_dtype) == PL_F32 ? CALL(__half, float) : CALL(__half, __half))    \
                         : ((weight_dtype) == PL_F32 ? CALL(__nv_bfloat16, float) : CALL(__nv_bfloat16, __nv_bfloat16)))

template <typename T>
static int launch_pack(pl_packed to, const void* x, int64_t n, bool keep_nonzero, cudaStream_t st) {
    pack_blocks<T><<<grid_for(n, 256, 8), 256, 0, st>>>(to.codes, to.scales, static_cast<const T*>(x), n, keep_nonzero);
    PL_COUNT_LAUNCHES(1);
    PL_CUDA(cudaGetLastError());
    return PL_OK;
}
static int pack_any(pl_packed to, const void* x, int64_t n, int dtype, bool keep_nonzero, cudaStream_t st) {
    return dtype == PL_F32   ? launch_pack<float>(to, x, n, keep_nonzero, st)
           : dtype == PL_F16 ? launch_pack<__half>(to, x, n, keep_nonzero, st)
                             : launch_pack<__nv_bfloat16>(to, x, n, keep_nonzero, st);
}
template <typename T>
static int launch_unpack(void* x, const pl_packed& from, int64_t n, cudaStream_t st) {
    unpack_blocks<T><<<grid_for(n, 256, 8), 256, 0, st>>>(static_cast<T*>(x), from.codes, from.scales, n);
    PL_COUNT_LAUNCHES(1);
    PL_CUDA(cudaGetLastError());
    return PL_OK;
}

template <typename T, typename W>
static int launch_mix(const pl_mix* m, void* out, const void* x, const void* x2, const void* weight, const void* weight2,
                      const void* bias, const void* residual, cudaStream_t st) {
    mix_rows<T, W><<<grid_for(m->rows, 8, 8), 256, 0, st>>>(
        shape_of(m), static_cast<T*>(out), static_cast<const T*>(x), static_cast<const T*>(x2), static_cast<const W*>(weight),
        static_cast<const W*>(weight2), static_cast<const W*>(bias), static_cast<const T*>(residual));
    PL_COUNT_LAUNCHES(1);
    PL_CUDA(cudaGetLastError());
    return PL_OK;
}
template <typename T, typename W>
static int launch_back(const pl_mix* m, const void* grad, Kept out, Kept x, Kept x2, const void* weight, const void* weight2,
                       const pl_mix_gradients& d, float* dz, cudaStream_t st) {
    mix_back_rows<T, W><<<grid_for(m->rows, 8, 8), 256, 0, st>>>(
        shape_of(m), dz, static_cast<const T*>(grad), out, static_cast<const W*>(weight), static_cast<const W*>(weight2),
        static_cast<T*>(d.x), static_cast<T*>(d.x2), static_cast<T*>(d.residual));
    PL_COUNT_LAUNCHES(1);
    if (d.weight || d.weight2 || d.bias) {
        mix_back_weights<T, W><<<(unsigned)((m->k + m->k2 + 1) * m->n), 256, 0, st>>>(
            shape_of(m), dz, x, x2, static_cast<W*>(d.weight), static_cast<W*>(d.weight2), static_cast<W*>(d.bias));
        PL_COUNT_LAUNCHES(1);
    }
    PL_CUDA(cudaGetLastError());
    return PL_OK;
}

static bool whole(const pl_packed& p) { return p.codes && p.scales; }

}  // namespace pl

using namespace pl;

extern "C" {

int pl_pack_activations(pl_packed packed, const void* x, int64_t n, int dtype, int keep_nonzero, void* stream) {
    if (n < 0 || dtype < PL_F32 || dtype > PL_BF16) return PL_INVALID_ARGUMENT;
    if (n == 0) return PL_OK;
    if (!whole(packed) || !x) return PL_INVALID_ARGUMENT;
    return pack_any(packed, x, n, dtype, keep_nonzero != 0, (cudaStream_t)stream);
}

int pl_unpack_activations(void* x, pl_packed packed, int64_t n, int dtype, void* stream) {
    if (n < 0 || dtype < PL_F32 || dtype > PL_BF16) return PL_INVALID_ARGUMENT;
    if (n == 0) return PL_OK;
    if (!whole(packed) || !x) return PL_INVALID_ARGUMENT;
    const cudaStream_t st = (cudaStream_t)stream;
    return dtype == PL_F32   ? launch_unpack<float>(x, packed, n, st)
           : dtype == PL_F16 ? launch_unpack<__half>(x, packed, n, st)
                             : launch_unpack<__nv_bfloat16>(x, packed, n, st);
}

int pl_channel_mix(const pl_mix* m, void* out, const void* x, const void* x2, const void* weight, const void* weight2,
                   const void* bias, const void* residual, pl_packed keep_x, pl_packed keep_x2, pl_packed keep_out, void* stream) {
    PL_TRY(check_shape(m));
    if (m->rows == 0) return PL_OK;
    if (!out || !x || !weight || (m->k2 && (!x2 || !weight2))) return PL_INVALID_ARGUMENT;
    for (const pl_packed* p : {&keep_x, &keep_x2, &keep_out})
        if ((p->codes != nullptr) != (p->scales != nullptr)) return PL_INVALID_ARGUMENT;
    if (keep_x2.codes && !m->k2) return PL_INVALID_ARGUMENT;
    const cudaStream_t st = (cudaStream_t)stream;
#define PL_MIX_CALL(T, W) launch_mix<T, W>(m, out, x, x2, weight, weight2, bias, residual, st)
    PL_TRY(PL_MIX_TYPES(m->dtype, m->weight_dtype, PL_MIX_CALL));
#undef PL_MIX_CALL
    if (keep_x.codes) PL_TRY(pack_any(keep_x, x, m->rows * m->k, m->dtype, false, st));
    if (keep_x2.codes) PL_TRY(pack_any(keep_x2, x2, m->rows * m->k2, m->dtype, false, st));
    if (keep_out.codes) PL_TRY(pack_any(keep_out, out, m->rows * m->n, m->dtype, m->activation == PL_ACT_RELU, st));
    return PL_OK;
}

int pl_channel_mix_workspace_bytes(const pl_mix* m, size_t* bytes) {
    PL_TRY(check_shape(m));
    if (!bytes) return PL_INVALID_ARGUMENT;
    *bytes = sizeof(float) * (size_t)m->rows * m->n;
    return PL_OK;
}

int pl_channel_mix_backward(const pl_mix* m, const void* grad_out, pl_kept out, pl_kept x, pl_kept x2, const void* weight,
                            const void* weight2, pl_mix_gradients d, void* workspace, size_t workspace_bytes, void* stream) {
    size_t need = 0;
    PL_TRY(pl_channel_mix_workspace_bytes(m, &need));
    const size_t weight_size = m->weight_dtype == PL_F32 ? 4 : 2;
    if (m->rows == 0) {   // sums of nothing
        const cudaStream_t st = (cudaStream_t)stream;
        if (d.weight) PL_CUDA(cudaMemsetAsync(d.weight, 0, weight_size * m->k * m->n, st));
        if (d.weight2) PL_CUDA(cudaMemsetAsync(d.weight2, 0, weight_size * m->k2 * m->n, st));
        if (d.bias) PL_CUDA(cudaMemsetAsync(d.bias, 0, weight_size * m->n, st));
        return PL_OK;
    }
    auto given = [](const pl_kept& a) { return a.packed.codes ? a.packed.scales != nullptr : a.full != nullptr; };
    if (!grad_out || (m->activation != PL_ACT_NONE && !given(out))) return PL_INVALID_ARGUMENT;
    if ((d.weight && !given(x)) || (d.x && !weight)) return PL_INVALID_ARGUMENT;
    if ((d.weight2 && (!m->k2 || !given(x2))) || (d.x2 && (!m->k2 || !weight2))) return PL_INVALID_ARGUMENT;
    if (!workspace || workspace_bytes < need) return PL_WORKSPACE_TOO_SMALL;
    auto kept = [](const pl_kept& a) { return Kept{a.full, a.packed.codes, a.packed.scales}; };
#define PL_MIX_CALL(T, W)                                                                                            \
    launch_back<T, W>(m, grad_out, kept(out), kept(x), kept(x2), weight, weight2, d, static_cast<float*>(workspace), \
                      (cudaStream_t)stream)
    return PL_MIX_TYPES(m->dtype, m->weight_dtype, PL_MIX_CALL);
#undef PL_MIX_CALL
}

}  // extern "C"
