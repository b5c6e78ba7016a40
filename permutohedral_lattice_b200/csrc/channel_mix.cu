// Products of channels with bias, residual and activation, their gradients, and activations in 8 bits: the training side of
// the operators around the lattice filter (the C entry points at the end of include/pl_lattice.h).
//
//   z = x W [+ x2 W2] [+ bias] [+ s residual],   out = act(z)
//   dz = g (no activation), g [out > 0] (relu), out (g - sum_k g_k out_k) (softmax)
//   dresidual = s dz,  dx = dz W^T,  dx2 = dz W2^T,  dW = x^T dz,  dW2 = x2^T dz,  dbias = sum over rows of dz
//
// A translation unit of its own: nothing here has to round like the reference's geometry.
#include <cuda_runtime.h>
#include <algorithm>
#include <stdint.h>

#include "mix_host.h"

namespace pl {

// Values to codes and back: bound by memory, 88 million floats to 8 bits in 81 us (5.5 TB/s), 44 million back to bfloat16 in 28 (4.9).
// wide: every address is a multiple of what its accesses take (16 bytes of float, 8 of 16-bit values,
// 4 of codes).
template <typename T>
__global__ void __launch_bounds__(256) pack_blocks(uint8_t* __restrict__ codes, int16_t* __restrict__ scales,
                                                   const T* __restrict__ x, long long n, int keep_nonzero, int wide) {
    const int lane = threadIdx.x & 31;
    int first, second;
    runs_of_lane(first, second);
    const long long step = (long long)gridDim.x * 2048;
    for (long long i0 = (long long)blockIdx.x * 2048 + (threadIdx.x >> 5) * 256; i0 < n; i0 += step) {   // (the same for a warp)
        if (!wide || i0 + 256 > n) {
            pack_rest(x + i0, (int)min(256ll, n - i0), codes + i0, scales + i0 / PACK_BLOCK, keep_nonzero != 0);
            continue;
        }
        float v[8], q[4];
        load4(q, x + i0 + first);
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = q[i];
        load4(q, x + i0 + second);
#pragma unroll
        for (int i = 0; i < 4; i++) v[4 + i] = q[i];
        u32 header;
        const uint2 c = encode8(v, header, keep_nonzero != 0);
        *reinterpret_cast<u32*>(codes + i0 + first) = c.x;
        *reinterpret_cast<u32*>(codes + i0 + second) = c.y;
        if ((lane & 3) == 0) scales[i0 / PACK_BLOCK + (lane >> 2)] = (int16_t)header;
    }
}

// 16 bytes of values a thread, four times on the way at once.
constexpr int UNPACK_AT_ONCE = 4;
template <typename T>
__host__ __device__ constexpr int unpack_values() { return 256 * UNPACK_AT_ONCE * 16 / (int)sizeof(T); }   // of a CTA at a time
template <typename T>
__global__ void __launch_bounds__(256) unpack_blocks(T* __restrict__ x, const uint8_t* __restrict__ codes,
                                                     const int16_t* __restrict__ scales, long long n, int wide) {
    constexpr int PER = 16 / sizeof(T), U = UNPACK_AT_ONCE;
    const long long step = (long long)gridDim.x * unpack_values<T>();
    for (long long i0 = (long long)blockIdx.x * unpack_values<T>() + threadIdx.x * PER; i0 < n; i0 += step) {
        u32 c[U][PER / 4], header[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const long long i = i0 + u * 256 * PER;
            header[u] = i < n ? (u32)(u16)scales[i / PACK_BLOCK] : 0;
#pragma unroll
            for (int w = 0; w < PER / 4; w++) {
                c[u][w] = 0;
                if (wide && i + PER <= n) c[u][w] = reinterpret_cast<const u32*>(codes + i)[w];
                else
                    for (int j = 0; j < 4; j++)
                        if (i + 4 * w + j < n) c[u][w] |= (u32)codes[i + 4 * w + j] << (8 * j);
            }
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            const long long i = i0 + u * 256 * PER;
            if (i >= n) break;
            float v[PER / 4][4];
#pragma unroll
            for (int w = 0; w < PER / 4; w++) decode4(v[w], c[u][w], header[u]);
            if (wide && i + PER <= n) {
                if constexpr (PER == 4) {
                    store4(x + i, v[0]);
                } else {
                    uint4 q;
                    T* h = reinterpret_cast<T*>(&q);
#pragma unroll
                    for (int j = 0; j < PER; j++) h[j] = from_float<T>(v[j / 4][j & 3]);
                    *reinterpret_cast<uint4*>(x + i) = q;
                }
            } else {
                for (int j = 0; j < PER; j++)
                    if (i + j < n) x[i + j] = from_float<T>(v[j / 4][j & 3]);
            }
        }
    }
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
template <typename T>
static int launch_pack(pl_packed to, const void* x, int64_t n, bool keep_nonzero, cudaStream_t st) {
    const bool wide = aligned(x, 4 * sizeof(T)) && aligned(to.codes, 4);
    pack_blocks<T><<<grid_for(n, 2048, 8), 256, 0, st>>>(to.codes, to.scales, static_cast<const T*>(x), n, keep_nonzero, wide);
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
    const bool wide = aligned(x, 16) && aligned(from.codes, 4);
    unpack_blocks<T><<<grid_for(n, unpack_values<T>(), 8), 256, 0, st>>>(static_cast<T*>(x), from.codes, from.scales, n, wide);
    PL_COUNT_LAUNCHES(1);
    PL_CUDA(cudaGetLastError());
    return PL_OK;
}

static size_t shares_bytes(const pl_mix* m) {
    return up16(sizeof(float) * (size_t)(m->k + m->k2 + 1) * m->n * num_sms() * BACK_CTAS);
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
    MixArgs a = {};
    a.rows = m->rows;
    a.k = m->k, a.k2 = m->k2, a.n = m->n, a.activation = m->activation, a.scale = m->residual_scale;
    a.x = x, a.x2 = m->k2 ? x2 : nullptr, a.weight = weight, a.weight2 = weight2, a.bias = bias, a.residual = residual, a.out = out;
    a.weight_dtype = m->weight_dtype;
    const bool fused = mix_keeps_in_forward(m->n);
    if (fused) {
        a.x_codes = keep_x.codes, a.x_scales = keep_x.scales;
        a.x2_codes = keep_x2.codes, a.x2_scales = keep_x2.scales;
        a.out_codes = keep_out.codes, a.out_scales = keep_out.scales;
    }
    PL_TRY(m->dtype == PL_F32 ? mix_forward_floats(a, PL_F32, st) : mix_forward_halves(a, m->dtype, st));
    if (fused) return PL_OK;
    if (keep_x.codes) PL_TRY(pack_any(keep_x, x, m->rows * m->k, m->dtype, false, st));
    if (keep_x2.codes) PL_TRY(pack_any(keep_x2, x2, m->rows * m->k2, m->dtype, false, st));
    if (keep_out.codes) PL_TRY(pack_any(keep_out, out, m->rows * m->n, m->dtype, m->activation == PL_ACT_RELU, st));
    return PL_OK;
}

int pl_channel_mix_workspace_bytes(const pl_mix* m, size_t* bytes) {
    PL_TRY(check_shape(m));
    if (!bytes) return PL_INVALID_ARGUMENT;
    *bytes = shares_bytes(m) + (mix_narrow(m->k, m->k2, m->n) ? 0 : sizeof(float) * (size_t)m->rows * m->n);
    return PL_OK;
}

int pl_channel_mix_backward(const pl_mix* m, const void* grad_out, pl_kept out, pl_kept x, pl_kept x2, const void* weight,
                            const void* weight2, pl_mix_gradients d, void* workspace, size_t workspace_bytes, void* stream) {
    size_t need = 0;
    PL_TRY(pl_channel_mix_workspace_bytes(m, &need));
    const size_t weight_size = size_of(m->weight_dtype);
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
    if (!aligned(workspace, 16)) return PL_INVALID_ARGUMENT;
    auto kept = [](const pl_kept& k) { return Kept{k.full, k.packed.codes, k.packed.scales}; };
    MixBackArgs a = {};
    a.rows = m->rows;
    a.k = m->k, a.k2 = m->k2, a.n = m->n, a.activation = m->activation, a.scale = m->residual_scale;
    a.grad = grad_out;
    if (m->activation != PL_ACT_NONE) a.out = kept(out);
    a.want_x = d.weight != nullptr, a.want_x2 = d.weight2 != nullptr;
    if (a.want_x) a.x = kept(x);
    if (a.want_x2) a.x2 = kept(x2);
    a.weight = weight, a.weight2 = weight2, a.weight_dtype = m->weight_dtype;
    a.dx = d.x, a.dx2 = d.x2, a.dresidual = d.residual;
    a.bias = d.bias != nullptr;
    if (d.weight || d.weight2 || d.bias) a.shares = static_cast<float*>(workspace);
    a.dz = reinterpret_cast<float*>(static_cast<unsigned char*>(workspace) + shares_bytes(m));
    const cudaStream_t st = (cudaStream_t)stream;
    return m->dtype == PL_F32 ? mix_backward_floats(a, d, st) : mix_backward_halves(a, m->dtype, d, st);
}

}  // extern "C"
