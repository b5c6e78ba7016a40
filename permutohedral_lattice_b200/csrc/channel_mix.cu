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
#include <stdlib.h>
#include <stdio.h>
#ifndef MIXF_MT
#define MIXF_MT 2
#endif
#include <stdint.h>

#include "host_calls.h"
#include "mix_common.cuh"
#include "mix_forward.cuh"
#include "mix_backward.cuh"
#include "mix_tiny.cuh"

namespace pl {

// Values to codes and back.  wide: every address is a multiple of what its accesses take (16 bytes of float, 8 of 16-bit values,
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

template <typename T>
__global__ void __launch_bounds__(256) unpack_blocks(T* __restrict__ x, const uint8_t* __restrict__ codes,
                                                     const int16_t* __restrict__ scales, long long n, int wide) {
    const long long step = (long long)gridDim.x * 1024;
    for (long long i = (long long)blockIdx.x * 1024 + threadIdx.x * 4; i < n; i += step) {
        const u32 header = (u32)(u16)scales[i / PACK_BLOCK];
        u32 c = 0;
        float v[4];
        if (wide && i + 3 < n) c = *reinterpret_cast<const u32*>(codes + i);
        else
            for (int j = 0; j < 4; j++)
                if (i + j < n) c |= (u32)codes[i + j] << (8 * j);
        decode4(v, c, header);
        if (wide && i + 3 < n) store4(x + i, v);
        else
            for (int j = 0; j < 4; j++)
                if (i + j < n) x[i + j] = from_float<T>(v[j]);
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
static unsigned grid_for(long long items, long long per_cta, int ctas_per_sm) {
    return (unsigned)std::max(1ll, std::min((items + per_cta - 1) / per_cta, (long long)num_sms() * ctas_per_sm));
}
static size_t size_of(int dtype) { return dtype == PL_F32 ? 4 : 2; }
static bool aligned(const void* p, size_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

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
    const bool wide = aligned(x, 4 * sizeof(T)) && aligned(from.codes, 4);
    unpack_blocks<T><<<grid_for(n, 1024, 8), 256, 0, st>>>(static_cast<T*>(x), from.codes, from.scales, n, wide);
    PL_COUNT_LAUNCHES(1);
    PL_CUDA(cudaGetLastError());
    return PL_OK;
}

constexpr size_t SMEM_SM = 228 * 1024, SMEM_CTA = 227 * 1024;   // shared memory of an SM, and the most that a CTA may have
// How a kernel runs whose warps have tiles of their own, smem(warps, stages, blocks) bytes a CTA: blocks of rows in a tile, stages of
// a warp, warps of a CTA, CTAs.
struct MixLaunch {
    int warps, stages, blocks, ctas;
    size_t smem;
};
template <typename Smem>
static MixLaunch mix_launch(long long rows, int block_rows, size_t block_bytes, int most_ctas, int most_stages, int most_blocks, Smem smem) {
    static const char* e = getenv("PLX");   // warps stages blocks ctas
    int ew = 0, es = 0, eb = 0, ec = 0;
    if (e) sscanf(e, "%d %d %d %d", &ew, &es, &eb, &ec);
    MixLaunch l;
    const long long all = (rows + block_rows - 1) / block_rows;
    // A tile of some 4 KB, as long as there are tiles for four warps of every SM; a CTA of four warps, as long as there are tiles for
    // every SM.
    l.blocks = (int)std::max<size_t>(1, std::min<size_t>(most_blocks, 4096 / block_bytes));
    if (eb) l.blocks = std::min(eb, most_blocks);
    while (l.blocks > 1 && all < (long long)l.blocks * 4 * num_sms()) l.blocks--;
    const long long tiles = (all + l.blocks - 1) / l.blocks;
    l.warps = (int)std::max(1ll, std::min((long long)(ew ? ew : 4), tiles / num_sms()));
    // Two stages where three CTAs of an SM have room for them: what a warp waits for a tile is otherwise better hidden by other warps
    // (the gradients of 21 labels: 700 us with two stages and eight warps an SM, 602 with one and twelve).
    l.stages = tiles > (long long)l.warps * num_sms() ? std::min(es ? es : 2, most_stages) : 1;
    if (!es && l.stages == 2 && 3 * (smem(l.warps, 2, l.blocks) + 1024) > SMEM_SM) l.stages = 1;
    while (l.stages > 1 && smem(l.warps, l.stages, l.blocks) > SMEM_CTA) l.stages--;
    while (l.blocks > 1 && smem(l.warps, l.stages, l.blocks) > SMEM_CTA) l.blocks--;
    while (l.warps > 1 && smem(l.warps, l.stages, l.blocks) > SMEM_CTA) l.warps--;
    l.smem = smem(l.warps, l.stages, l.blocks);
    const int fit = (int)std::max<size_t>(1, SMEM_SM / (l.smem + 1024));
    const long long per_cta = (long long)block_rows * l.blocks * l.warps;
    l.ctas = (int)std::min<long long>((rows + per_cta - 1) / per_cta, (long long)num_sms() * std::min(ec ? ec : most_ctas, fit));
    return l;
}

template <typename TI, typename TO, int NT, int MT, int WAY>
static int launch_forward(MixArgs a, cudaStream_t st) {
    const MixLaunch l = mix_launch(a.rows, 16 * MT, 16 * MT * (sizeof(TI) * (a.k + a.k2 + (a.residual ? a.n : 0)) + sizeof(TO) * a.n), mix_forward_ctas(NT, WAY), MIX_STAGES, 8,
                                   [&](int warps, int stages, int blocks) {
                                       return MixSmem<TI, TO>(16 * MT * blocks, a.k, a.k2, a.n, NT, WAY).bytes(warps, stages);
                                   });
    a.stages = l.stages, a.blocks = l.blocks;
    PL_TRY((ensure_dynamic_smem<mix_forward<TI, TO, NT, MT, WAY>>(l.smem)));
    mix_forward<TI, TO, NT, MT, WAY><<<l.ctas, 32 * l.warps, l.smem, st>>>(a);
    PL_COUNT_LAUNCHES(1);
    PL_CUDA(cudaGetLastError());
    return PL_OK;
}
// Output channels in steps of 8: the accumulators of a warp's rows are in registers.  From 65 channels on a warp takes
// 16 rows in place of 32.
static bool keeps_in_forward(int n) { return n <= 64; }
template <typename TI, typename TO, int WAY>
static int forward_of(const MixArgs& a, cudaStream_t st) {
    if (a.n <= 8) return launch_forward<TI, TO, 1, 2, WAY>(a, st);
    if (a.n <= 16) return launch_forward<TI, TO, 2, 2, WAY>(a, st);
    if (a.n <= 24) return launch_forward<TI, TO, 3, 2, WAY>(a, st);
    if (a.n <= 32) return launch_forward<TI, TO, 4, 2, WAY>(a, st);
    if constexpr (WAY != MIX_PLAIN) {
        return a.n <= 40   ? launch_forward<TI, TO, 5, 2, WAY>(a, st)
               : a.n <= 48 ? launch_forward<TI, TO, 6, 2, WAY>(a, st)
               : a.n <= 56 ? launch_forward<TI, TO, 7, 2, WAY>(a, st)
               : a.n <= 64 ? launch_forward<TI, TO, 8, 2, WAY>(a, st)
                           : launch_forward<TI, TO, 16, 1, WAY>(a, st);
    }
    return PL_INTERNAL_ERROR;
}
template <typename TO>
static int launch_forward_wide(const MixArgs& a, cudaStream_t st) {
    const size_t smem = wide_smem(a.k, a.k2);
    PL_TRY((ensure_dynamic_smem<mix_forward_wide<TO>>(smem)));
    const long long tiles = (a.rows + 15) / 16;
    const unsigned ctas = (unsigned)std::min<long long>((tiles + WIDE_WARPS - 1) / WIDE_WARPS, num_sms());
    mix_forward_wide<TO><<<ctas, 32 * WIDE_WARPS, smem, st>>>(a);
    PL_COUNT_LAUNCHES(1);
    PL_CUDA(cudaGetLastError());
    return PL_OK;
}
// Channels of every operand where they are the same, 2 or 4, and all rows begin at multiples of their size; else 0.
static int tiny_channels(int k, int k2, int n, size_t size, const void* const* rows, int count) {
    if (k != n || (k2 && k2 != n) || (n != 2 && n != 4)) return 0;
    for (int i = 0; i < count; i++)
        if (!aligned(rows[i], n * size)) return 0;
    return n;
}
static bool tiny(int k, int k2, int n) { return k <= TINY && k2 <= TINY && n <= TINY; }
template <typename TI, typename TO>
static int forward_any(const MixArgs& a, cudaStream_t st) {
    if constexpr (std::is_same<TI, TO>::value) {
        if (tiny(a.k, a.k2, a.n)) {
            const unsigned grid = grid_for(a.rows, 256 * TINY_ROWS, 4);
            const void* rows[] = {a.x, a.x2, a.residual, a.out};
            const int v = tiny_channels(a.k, a.k2, a.n, sizeof(TI), rows, 4);
            if (v == 4) mix_tiny<TI, 4><<<grid, 256, 0, st>>>(a);
            else if (v == 2) mix_tiny<TI, 2><<<grid, 256, 0, st>>>(a);
            else mix_tiny<TI, 0><<<grid, 256, 0, st>>>(a);
            PL_COUNT_LAUNCHES(1);
            PL_CUDA(cudaGetLastError());
            return PL_OK;
        }
    }
    if constexpr (sizeof(TI) == 4) {
        if (a.n > 64) return launch_forward_wide<TO>(a, st);
    }
    if constexpr (sizeof(TI) == 2) {
        if (a.weight_dtype != PL_F32) return forward_of<TI, TO, MIX_PAIRS>(a, st);
    }
    // few products to a sum: what the tensor cores cut stays below 2^-21 of it
    if (a.k + a.k2 <= 96 && a.n <= 32) return forward_of<TI, TO, MIX_PLAIN>(a, st);
    return forward_of<TI, TO, MIX_PARTED>(a, st);
}

constexpr int BACK_CTAS = 3;   // of an SM, at most: as many shares of dW there may be
static bool narrow(const pl_mix* m) { return up8(m->k) + up8(m->k2) <= 80 && m->n <= 32; }
static size_t shares_bytes(const pl_mix* m) {
    return up16(sizeof(float) * (size_t)(m->k + m->k2 + 1) * m->n * num_sms() * BACK_CTAS);
}

static int add_shares(const MixBackArgs& a, const pl_mix_gradients& d, int ctas, cudaStream_t st) {
    const unsigned grid = (unsigned)(((a.k + a.k2 + 1) * a.n + 31) / 32);
#define PL_ADD(W) \
    mix_add_shares<W><<<grid, 256, 0, st>>>(a.shares, ctas, a.k, a.k2, a.n, static_cast<W*>(d.weight), static_cast<W*>(d.weight2), static_cast<W*>(d.bias))
    if (a.weight_dtype == PL_F32) PL_ADD(float);
    else if (a.weight_dtype == PL_F16) PL_ADD(__half);
    else PL_ADD(__nv_bfloat16);
#undef PL_ADD
    PL_COUNT_LAUNCHES(1);
    PL_CUDA(cudaGetLastError());
    return PL_OK;
}

template <typename T, bool PACKED, int MB, int NB>
static int launch_narrow(MixBackArgs a, const pl_mix_gradients& d, cudaStream_t st) {
    // in 8 bits: one stage, and as many blocks of rows as give 32 headers of each array (see mix_backward)
    const int widest = std::max(a.n, std::max(a.k, a.k2));
    const MixLaunch l = mix_launch(a.rows, 32, 32 * sizeof(T) * (2 * a.n + 2 * (a.k + a.k2)), MB * NB > 12 ? 2 : BACK_CTAS, PACKED ? 1 : MIX_STAGES,
                                   PACKED ? std::max(1, 32 / widest) : 8, [&](int warps, int stages, int blocks) {
                                       MixBackArgs b = a;
                                       b.blocks = blocks, b.stages = stages;
                                       return std::max(MixBackSmem(b, warps, NB, sizeof(T), PACKED).bytes(warps), mix_share_bytes(warps, MB, NB));
                                   });
    a.stages = l.stages, a.blocks = l.blocks;
    PL_TRY((ensure_dynamic_smem<mix_backward<T, PACKED, MB, NB>>(l.smem)));
    mix_backward<T, PACKED, MB, NB><<<l.ctas, 32 * l.warps, l.smem, st>>>(a);
    PL_COUNT_LAUNCHES(1);
    PL_CUDA(cudaGetLastError());
    return a.shares ? add_shares(a, d, l.ctas, st) : PL_OK;
}
// dW in blocks of eight channels, a multiple of 16 in all: what narrow() allows is at most 80.
template <typename T, bool PACKED>
static int narrow_any(const MixBackArgs& a, const pl_mix_gradients& d, cudaStream_t st) {
    const int rows = up8(a.k) + up8(a.k2);
    return rows <= 16 && a.n <= 8    ? launch_narrow<T, PACKED, 1, 1>(a, d, st)
           : rows <= 48 && a.n <= 24 ? launch_narrow<T, PACKED, 3, 3>(a, d, st)
           : a.n <= 16               ? launch_narrow<T, PACKED, 5, 2>(a, d, st)
                                     : launch_narrow<T, PACKED, 5, 4>(a, d, st);
}

template <typename T>
static int launch_wide(const MixBackArgs& a, const pl_mix_gradients& d, cudaStream_t st) {
    mix_dz<T><<<grid_for(a.rows, 8, 8), 256, 0, st>>>(a);
    PL_COUNT_LAUNCHES(1);
    PL_CUDA(cudaGetLastError());
    for (int second = 0; second < 2; second++) {
        void* to = second ? a.dx2 : a.dx;
        if (!to) continue;
        MixArgs f = {};
        f.rows = a.rows;
        f.k = a.n, f.n = second ? a.k2 : a.k;
        f.activation = PL_ACT_NONE;
        f.x = a.dz, f.out = to;
        f.weight = second ? a.weight2 : a.weight;
        f.weight_dtype = a.weight_dtype, f.transposed = 1;
        PL_TRY((forward_any<float, T>(f, st)));
    }
    if (!a.shares) return PL_OK;
    PL_TRY((ensure_dynamic_smem<mix_backward_weights<T>>(WIDE_SMEM)));
    const unsigned ctas = grid_for(a.rows, WIDE_ROWS, 1);
    mix_backward_weights<T><<<dim3(ctas, a.want_x2 ? 2 : 1), 256, WIDE_SMEM, st>>>(a);
    PL_COUNT_LAUNCHES(1);
    PL_CUDA(cudaGetLastError());
    return add_shares(a, d, (int)ctas, st);
}
template <typename T>
static int launch_back(const pl_mix* m, const MixBackArgs& a, const pl_mix_gradients& d, cudaStream_t st) {
    if (!narrow(m)) return launch_wide<T>(a, d, st);
    if (tiny(a.k, a.k2, a.n)) {
        const unsigned ctas = grid_for(a.rows, 256 * TINY_BACK_ROWS, 2);
        const void* rows[] = {a.grad, a.out.full, a.x.full, a.x2.full, a.dx, a.dx2, a.dresidual};
        const int v = tiny_channels(a.k, a.k2, a.n, sizeof(T), rows, 7);
        if (v == 4) mix_tiny_backward<T, 4><<<ctas, 256, 0, st>>>(a);
        else if (v == 2) mix_tiny_backward<T, 2><<<ctas, 256, 0, st>>>(a);
        else mix_tiny_backward<T, 0><<<ctas, 256, 0, st>>>(a);
        PL_COUNT_LAUNCHES(1);
        PL_CUDA(cudaGetLastError());
        return a.shares ? add_shares(a, d, (int)ctas, st) : PL_OK;
    }
    return a.out.codes || a.x.codes || a.x2.codes ? narrow_any<T, true>(a, d, st) : narrow_any<T, false>(a, d, st);
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
    const bool fused = keeps_in_forward(m->n);
    if (fused) {
        a.x_codes = keep_x.codes, a.x_scales = keep_x.scales;
        a.x2_codes = keep_x2.codes, a.x2_scales = keep_x2.scales;
        a.out_codes = keep_out.codes, a.out_scales = keep_out.scales;
    }
    PL_TRY((m->dtype == PL_F32   ? forward_any<float, float>(a, st)
            : m->dtype == PL_F16 ? forward_any<__half, __half>(a, st)
                                 : forward_any<__nv_bfloat16, __nv_bfloat16>(a, st)));
    if (fused) return PL_OK;
    if (keep_x.codes) PL_TRY(pack_any(keep_x, x, m->rows * m->k, m->dtype, false, st));
    if (keep_x2.codes) PL_TRY(pack_any(keep_x2, x2, m->rows * m->k2, m->dtype, false, st));
    if (keep_out.codes) PL_TRY(pack_any(keep_out, out, m->rows * m->n, m->dtype, m->activation == PL_ACT_RELU, st));
    return PL_OK;
}

int pl_channel_mix_workspace_bytes(const pl_mix* m, size_t* bytes) {
    PL_TRY(check_shape(m));
    if (!bytes) return PL_INVALID_ARGUMENT;
    *bytes = shares_bytes(m) + (narrow(m) ? 0 : sizeof(float) * (size_t)m->rows * m->n);
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
    return m->dtype == PL_F32   ? launch_back<float>(m, a, d, st)
           : m->dtype == PL_F16 ? launch_back<__half>(m, a, d, st)
                                : launch_back<__nv_bfloat16>(m, a, d, st);
}

}  // extern "C"
