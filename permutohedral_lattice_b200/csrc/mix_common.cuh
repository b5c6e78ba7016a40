// Shared device code of the channel products: number types, products of floats on the tensor cores, 8-bit blocks, and the
// copies of a tile's rows between global and shared memory.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include "common.cuh"

namespace pl {

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

// Weights and biases: few, of a type known at run time (pl_dtype).
__device__ __forceinline__ float load_weight(const void* w, int i, int dtype) {
    return dtype == PL_F32   ? static_cast<const float*>(w)[i]
           : dtype == PL_F16 ? __half2float(static_cast<const __half*>(w)[i])
                             : __bfloat162float(static_cast<const __nv_bfloat16*>(w)[i]);
}

// ---------------------------------------------------------------------------------------------
// Products: m16n8k8 on numbers of 11 significant bits (tf32), sums in float.  A float is the sum of two such numbers up to
// 2^-23 of it: v = hi + lo, hi the nearest one, lo what is left cut to 11 bits; a product of two floats is then hi hi + hi lo +
// lo hi up to 2^-22.  Numbers of 16 bits and 8-bit codes are their own hi, which saves a term.  Lane 4 g + t of a warp holds
//   a: (g, t), (g + 8, t), (g, t + 4), (g + 8, t + 4)    b: (t, g), (t + 4, g)    c: (g, 2t), (g, 2t + 1), (g + 8, 2t), (g + 8, 2t + 1)
// ---------------------------------------------------------------------------------------------
__device__ __forceinline__ void mma8(float (&c)[4], const u32 (&a)[4], const u32 (&b)[2]) {
    asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
__device__ __forceinline__ void split(float v, u32& hi, u32& lo) {
    hi = (__float_as_uint(v) + 0x1000u) & 0xFFFFE000u;
    lo = __float_as_uint(v - __uint_as_float(hi)) & 0xFFFFE000u;
}

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
__device__ __forceinline__ u32 encode_value(float v, u32 header, bool keep_nonzero) {
    if ((header & 255u) == 255u) return 0;
    const int e = (int)(header & 255u) - 127;
    int code = __float2int_rn(v * power_of_two(-e));   // exact but for values far below half a step
    if (e >= 120) code = (header & 256u) ? min(max(code, -127), 127) : min(code, 255);
    if (keep_nonzero && code == 0 && v != 0.f) code = v < 0.f ? -1 : 1;
    return (u32)code & 255u;
}
// What a code is multiplied by; NaN for a block of NaN.
__device__ __forceinline__ float block_step(u32 header) {
    const u32 low = header & 255u;
    return low == 255u ? __int_as_float(0x7FC00000) : power_of_two((int)low - 127);
}
__device__ __forceinline__ float decode_value(u32 code, u32 header) {
    return (float)((header & 256u) ? (int)(signed char)code : (int)code) * block_step(header);
}

// Four consecutive values.
__device__ __forceinline__ void load4(float (&v)[4], const float* p) {
    const float4 q = *reinterpret_cast<const float4*>(p);
    v[0] = q.x, v[1] = q.y, v[2] = q.z, v[3] = q.w;
}
template <typename T>
__device__ __forceinline__ void load4(float (&v)[4], const T* p) {
    static_assert(sizeof(T) == 2);
    const uint2 q = *reinterpret_cast<const uint2*>(p);
    const T* h = reinterpret_cast<const T*>(&q);
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = to_float(h[i]);
}
__device__ __forceinline__ void store4(float* p, const float (&v)[4]) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
}
template <typename T>
__device__ __forceinline__ void store4(T* p, const float (&v)[4]) {
    static_assert(sizeof(T) == 2);
    uint2 q;
    T* h = reinterpret_cast<T*>(&q);
#pragma unroll
    for (int i = 0; i < 4; i++) h[i] = from_float<T>(v[i]);
    *reinterpret_cast<uint2*>(p) = q;
}

// Four values of a block to codes, eight lanes a block (all lanes of the warp take part).  Returns the four codes.
__device__ __forceinline__ u32 encode4(const float (&v)[4], u32& header, bool keep_nonzero) {
    u32 most = 0, negative = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const u32 bits = __float_as_uint(v[i]);
        most = max(most, bits & 0x7FFFFFFFu);
        negative |= v[i] < 0.f ? 1u : 0u;
    }
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) {
        most = max(most, __shfl_xor_sync(~0u, most, o));
        negative |= __shfl_xor_sync(~0u, negative, o);
    }
    header = block_header(most, negative != 0);
    u32 codes = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) codes |= encode_value(v[i], header, keep_nonzero) << (8 * i);
    return codes;
}
__device__ __forceinline__ void decode4(float (&v)[4], u32 codes, u32 header) {
    const float step = block_step(header);
    const bool is_signed = (header & 256u) != 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const u32 c = (codes >> (8 * i)) & 255u;
        v[i] = (float)(is_signed ? (int)(signed char)c : (int)c) * step;
    }
}

// `count` values in shared memory, whole blocks from the first one on, to 8 bits by one warp.  wide: codes is 4-byte aligned.
template <typename T>
__device__ __forceinline__ void pack_by_warp(const T* values, int count, uint8_t* __restrict__ codes, int16_t* __restrict__ scales,
                                             bool keep_nonzero, bool wide) {
    const int lane = threadIdx.x & 31, blocks = (count + PACK_BLOCK - 1) / PACK_BLOCK;
    for (int b0 = 0; b0 < blocks; b0 += 4) {
        const int b = b0 + (lane >> 3), i = b * PACK_BLOCK + 4 * (lane & 7);
        float v[4] = {0.f, 0.f, 0.f, 0.f};
        if (i + 3 < count) load4(v, values + i);
        else
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (i + j < count) v[j] = to_float(values[i + j]);
        u32 header;
        const u32 c = encode4(v, header, keep_nonzero);
        if (wide && i + 3 < count) *reinterpret_cast<u32*>(codes + i) = c;
        else
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (i + j < count) codes[i + j] = (uint8_t)(c >> (8 * j));
        if ((lane & 7) == 0 && b < blocks) scales[b] = (int16_t)header;
    }
}

// ---------------------------------------------------------------------------------------------
// Rows of a tile between global and shared memory.  A producer warp fills stages; a stage's `full` barrier counts its 32
// lanes and the bytes of the bulk copies, its `empty` barrier the consumer warps.
// ---------------------------------------------------------------------------------------------
__device__ __forceinline__ void mbar_arrive(u64* bar) {
    const unsigned a = (unsigned)__cvta_generic_to_shared(bar);
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(a) : "memory");
}
__device__ __forceinline__ void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
__device__ __forceinline__ void bulk_wait_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }

// The lanes of a warp copy `bytes` from global to shared memory, any alignment of the source that its type has.
template <int SIZE>
__device__ __forceinline__ void copy_in(void* to, const void* from, int count) {
    const int lane = threadIdx.x & 31;
    if constexpr (SIZE == 4) {
        for (int i = lane; i < count; i += 32) cp_async4(static_cast<u32*>(to) + i, static_cast<const u32*>(from) + i);
    } else if constexpr (SIZE == 2) {
        for (int i = lane; i < count; i += 32) static_cast<u16*>(to)[i] = static_cast<const u16*>(from)[i];
    } else {
        for (int i = lane; i < count; i += 32) static_cast<uint8_t*>(to)[i] = static_cast<const uint8_t*>(from)[i];
    }
}
// A warp's finished rows from shared to global memory: one bulk copy, or plain stores.  Lane 0 waits later (bulk_wait_read).
template <typename T>
__device__ __forceinline__ void copy_out(T* to, const T* from, int count, bool bulk) {
    const int lane = threadIdx.x & 31;
    if (bulk) {
        if (lane == 0) bulk_store(to, from, (unsigned)(count * sizeof(T)));
    } else {
        for (int i = lane; i < count; i += 32) to[i] = from[i];
    }
}
__device__ __forceinline__ bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace pl
