// Shared device code of the channel products: number types, products of floats on the tensor cores, 8-bit blocks, and the
// copies of a tile's rows between global and shared memory.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <type_traits>
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

// put(r, c, weight of input channel r (those of a second input from first_rows on) and output channel c) for a grid of rows x columns, zeros
// where there is no such channel.  Four at a time: in a small call this is half of what a CTA does, and each is a trip to L2.
// transposed: the (first and only) weight is [n][k].
template <int COLUMNS, typename Put>
__device__ __forceinline__ void for_weights(int rows, int first_rows, int k, int k2, int n, const void* weight, const void* weight2, int transposed,
                                            int dtype, Put put) {
    constexpr int U = 4;
    for (int i0 = threadIdx.x; i0 < rows * COLUMNS; i0 += U * blockDim.x) {
        float v[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int i = i0 + u * (int)blockDim.x, r = i / COLUMNS, c = i - r * COLUMNS;
            const bool second = r >= first_rows;
            const int j = second ? r - first_rows : r;
            const void* w = second ? weight2 : weight;
            v[u] = i < rows * COLUMNS && c < n && j < (second ? k2 : k) && w ? load_weight(w, transposed ? c * k + j : j * n + c, dtype) : 0.f;
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int i = i0 + u * (int)blockDim.x;
            if (i < rows * COLUMNS) put(i / COLUMNS, i % COLUMNS, v[u]);
        }
    }
}

// ---------------------------------------------------------------------------------------------
// Products: m16n8k8 on numbers of 11 significant bits (tf32), sums in float.  A float is the sum of two such numbers up to
// 2^-23 of it: v = hi + lo, hi the nearest one, lo what is left cut to 11 bits; a product of two floats is then hi hi + hi lo +
// lo hi up to 2^-22.  Numbers of 16 bits and 8-bit codes are their own hi, which saves a term.  Lane 4 g + t of a warp holds
//   a: (g, t), (g + 8, t), (g, t + 4), (g + 8, t + 4)    b: (t, g), (t + 4, g)    c: (g, 2t), (g, 2t + 1), (g + 8, 2t), (g + 8, 2t + 1)
// and wants each of them in registers that follow one another.  So b's that are read more than once lie in shared memory as the
// lanes take them, 16 bytes a lane: the high terms of both, then the low ones.  (Lying row by row as pairs of terms they took two accesses
// and four moves: a quarter of all instructions of the gradients at 21 labels.)
// ---------------------------------------------------------------------------------------------
__device__ __forceinline__ void mma8(float (&c)[4], const u32 (&a)[4], const u32 (&b)[2]) {
    asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
__device__ __forceinline__ void mma8_first(float (&c)[4], const u32 (&a)[4], const u32 (&b)[2]) {   // to nothing
    asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]), "f"(0.f));
}
// Two 16-bit values a register, m16n8k16, products exact and sums in float: a: channels 2t, 2t + 1 of rows g and g + 8, then 2t + 8, 2t + 9;
// b: rows 2t, 2t + 1 of column g, then 2t + 8, 2t + 9.
template <typename T>
__device__ __forceinline__ void mma16(float (&c)[4], const u32 (&a)[4], const u32 (&b)[2]) {
    if constexpr (std::is_same<T, __half>::value)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
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

// Eight values of a block to codes, four lanes a block (all lanes of the warp take part): v[0..3] and v[4..7] are two runs of four
// consecutive values, their codes the two words.  A product with a power of two, rounded to a whole number by adding 1.5 2^23 to
// it: the sum's low byte is the code.
__device__ __forceinline__ uint2 encode8(const float (&v)[8], u32& header, bool keep_nonzero) {
    const int lane = threadIdx.x & 31;
    u32 bits[8], any = 0, most = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        bits[i] = __float_as_uint(v[i]);
        any |= bits[i];
    }
    bool is_signed = false;
    if (__any_sync(~0u, any >> 31)) {   // (signs of zeros do not count)
        float least = 0.f;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            bits[i] &= 0x7FFFFFFFu;
            least = fminf(least, v[i]);
        }
        is_signed = (__ballot_sync(~0u, least < 0.f) >> (lane & 28) & 15u) != 0;
    }
#pragma unroll
    for (int i = 0; i < 8; i++) most = max(most, bits[i]);
    most = max(most, __shfl_xor_sync(~0u, most, 1));
    most = max(most, __shfl_xor_sync(~0u, most, 2));
    // block_header, but for its upper limit and for NaN: adding what the fraction may lack carries into the exponent where it has more
    const u32 low = (u32)max((int)((most + (is_signed ? 0x1FFFFu : 0xFFFFu)) >> 23) - (is_signed ? 6 : 7), 1);
    header = low | (is_signed ? 256u : 0u);
    if (low >= 247 || keep_nonzero) {
        header = block_header(most, is_signed);
        u32 c[2] = {0, 0};
#pragma unroll
        for (int i = 0; i < 8; i++) c[i / 4] |= encode_value(v[i], header, keep_nonzero) << (8 * (i & 3));
        return make_uint2(c[0], c[1]);
    }
    const float per_step = __uint_as_float((254u - low) << 23), whole = 12582912.f;
    u32 c[8];
#pragma unroll
    for (int i = 0; i < 8; i++) c[i] = __float_as_uint(fmaf(v[i], per_step, whole));
    return make_uint2(__byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410),
                      __byte_perm(__byte_perm(c[4], c[5], 0x0040), __byte_perm(c[6], c[7], 0x0040), 0x5410));
}
// Where a lane's two runs of four lie in the 256 values of its warp: blocks take their halves in another order each, so that the
// lanes that access memory together lie in different banks.
__device__ __forceinline__ void runs_of_lane(int& first, int& second) {
    const int lane = threadIdx.x & 31, block = lane >> 2, at = block * PACK_BLOCK + 4 * (lane & 3), swap = 16 * (block & 1);
    first = at + swap, second = at + 16 - swap;
}
// Four codes to values: a byte in the last place of 2^23 is 2^23 more than it stands for, and so is a signed one with its sign
// turned round, but for another 128.
__device__ __forceinline__ void decode4(float (&v)[4], u32 codes, u32 header) {
    const float step = block_step(header);
    const bool is_signed = (header & 256u) != 0;
    const float less = is_signed ? 8388608.f + 128.f : 8388608.f;
    if (is_signed) codes ^= 0x80808080u;
    v[0] = (__uint_as_float(__byte_perm(codes, 0x4B000000u, 0x7440)) - less) * step;
    v[1] = (__uint_as_float(__byte_perm(codes, 0x4B000000u, 0x7441)) - less) * step;
    v[2] = (__uint_as_float(__byte_perm(codes, 0x4B000000u, 0x7442)) - less) * step;
    v[3] = (__uint_as_float(__byte_perm(codes, 0x4B000000u, 0x7443)) - less) * step;
}

// Up to 256 values, whole blocks from the first one on, to 8 bits by one warp: any number of them, any alignment.
template <typename T>
__device__ __noinline__ void pack_rest(const T* values, int count, uint8_t* codes, int16_t* scales, bool keep_nonzero) {
    int at[2];
    runs_of_lane(at[0], at[1]);
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = at[i / 4] + (i & 3) < count ? to_float(values[at[i / 4] + (i & 3)]) : 0.f;
    u32 header;
    const uint2 c = encode8(v, header, keep_nonzero);
#pragma unroll
    for (int i = 0; i < 8; i++)
        if (at[i / 4] + (i & 3) < count) codes[at[i / 4] + (i & 3)] = (uint8_t)((i < 4 ? c.x : c.y) >> (8 * (i & 3)));
    const int lane = threadIdx.x & 31;
    if ((lane & 3) == 0 && (lane >> 2) * PACK_BLOCK < count) scales[lane >> 2] = (int16_t)header;
}
// `count` values in shared memory, whole blocks from the first one on, to 8 bits by one warp: where(i) says where the i-th lies (four from
// a multiple of four on lie together).  wide: codes is 4-byte aligned and the blocks are whole.  (All cases in one loop took 150 instructions
// for 256 values, whole blocks by themselves take 60.)
template <typename T, typename Where>
__device__ __forceinline__ void pack_blocks_of(const T* values, int count, uint8_t* __restrict__ codes, int16_t* __restrict__ scales, bool keep_nonzero,
                                               Where where) {
    const int lane = threadIdx.x & 31;
    int first, second;
    runs_of_lane(first, second);
    uint8_t *c0 = codes + first, *c1 = codes + second;
    int16_t* head = scales + (lane >> 2);
    int left = count / PACK_BLOCK - (lane >> 2);   // blocks, from this lane's on
    for (int i = 0; i < count; i += 256, left -= 8, c0 += 256, c1 += 256, head += 8) {
        float v[8], q[4];
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = 0.f;
        if (left > 0) {
            load4(q, values + where(i + first));
#pragma unroll
            for (int e = 0; e < 4; e++) v[e] = q[e];
            load4(q, values + where(i + second));
#pragma unroll
            for (int e = 0; e < 4; e++) v[4 + e] = q[e];
        }
        u32 header;
        const uint2 c = encode8(v, header, keep_nonzero);
        if (left > 0) {
            *reinterpret_cast<u32*>(c0) = c.x;
            *reinterpret_cast<u32*>(c1) = c.y;
            if ((lane & 3) == 0) *head = (int16_t)header;
        }
    }
}
template <typename T>
__device__ __forceinline__ void pack_by_warp(const T* values, int count, uint8_t* __restrict__ codes, int16_t* __restrict__ scales,
                                             bool keep_nonzero, bool wide) {
    if (wide && count % PACK_BLOCK == 0) pack_blocks_of(values, count, codes, scales, keep_nonzero, [](int i) { return i; });
    else
        for (int i = 0; i < count; i += 256) pack_rest(values + i, min(256, count - i), codes + i, scales + i / PACK_BLOCK, keep_nonzero);
}

// ---------------------------------------------------------------------------------------------
// Tiles.  Every warp has its own: some rows of every operand, contiguous in memory whatever the number of channels, in a stage
// of shared memory of its own, fetched and sent out by bulk copies (one lane asks for them), the results in the place of what
// has been read.  Warps share the weights of their CTA and nothing else, and meet nobody at a tile.  What does not start on a
// 16-byte boundary, and the last rows, are copied by the lanes.
//
// Rows of 32, 64, ... 512 bytes would begin in the same few banks, and eight of them are read together (64 channels of 16 bits: up
// to 8 accesses for one, 259 us a forward pass over a million rows, so 160).  They lie 16 bytes further apart and are copied by the lanes,
// 16 bytes each.
// ---------------------------------------------------------------------------------------------
constexpr int MIX_WARPS = 4, MIX_STAGES = 2;   // of a CTA and of a warp, at most

__device__ __forceinline__ bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Values of `c` channels from one row to the next in shared memory: whether rows lie apart (RowsApart) is asked for by the caller, who knows
// that they are 16-byte aligned in memory.
struct RowsApart {
    int stride, shift;   // elements; log2 of the channels, or -1: one after another
    __host__ __device__ RowsApart(int c, int size, bool aligned) : stride(c), shift(-1) {
        const int bytes = c * size;
        if (!aligned || bytes < 32 || (bytes & (bytes - 1))) return;
        stride = c + 16 / size;
        shift = 0;
        while (1 << shift < c) shift++;
    }
    __host__ __device__ bool apart() const { return shift >= 0; }
    __device__ __forceinline__ int at(int i) const { return shift < 0 ? i : i + (i >> shift) * (stride - (1 << shift)); }   // of element i
};
template <typename T>
__device__ __forceinline__ void copy_rows_in(T* to, const T* from, int rows, const RowsApart& r) {   // there after the group's wait
    constexpr int PER = 16 / sizeof(T);
    const int lane = threadIdx.x & 31, count = rows << r.shift;
    for (int i = lane * PER; i < count; i += 32 * PER) cp_async16(to + r.at(i), from + i);
}
template <typename T>
__device__ __forceinline__ void copy_rows_out(T* to, const T* from, int rows, const RowsApart& r) {
    constexpr int PER = 16 / sizeof(T);
    const int lane = threadIdx.x & 31, count = rows << r.shift;
    for (int i = lane * PER; i < count; i += 32 * PER) *reinterpret_cast<uint4*>(to + i) = *reinterpret_cast<const uint4*>(from + r.at(i));
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void cp_async_wait_one() { asm volatile("cp.async.wait_group 1;" ::: "memory"); }   // one group may be on its way

// A warp copies `count` elements to shared memory; they are there after cp_async_wait_all and __syncwarp.
template <typename E>
__device__ __forceinline__ void copy_in(void* to, const E* from, int count) {
    const int lane = threadIdx.x & 31;
    if constexpr (sizeof(E) == 4) {
        for (int i = lane; i < count; i += 32) cp_async4(static_cast<E*>(to) + i, from + i);
    } else {
        for (int i = lane; i < count; i += 32) static_cast<E*>(to)[i] = from[i];
    }
}
// Shared memory by its own 32-bit addresses.
__device__ __forceinline__ u32 shared_address(const void* p) { return (u32)__cvta_generic_to_shared(p); }
__device__ __forceinline__ float lds(u32 at) {
    float v;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(at));
    return v;
}
// The accesses of which some lanes have none are predicated here: as branches around them they took a seventh of all instructions.
__device__ __forceinline__ u32 lds_u32_if(bool there, u32 at) {
    u32 v;
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %2, 0;\n\tmov.b32 %0, 0;\n\t@p ld.shared.u32 %0, [%1];\n\t}" : "=&r"(v) : "r"(at), "r"((int)there));
    return v;
}
__device__ __forceinline__ u32 lds_u16_if(bool there, u32 at) {
    u16 v;
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %2, 0;\n\tmov.b16 %0, 0;\n\t@p ld.shared.u16 %0, [%1];\n\t}" : "=&h"(v) : "r"(at), "r"((int)there));
    return v;
}
template <typename T>
__device__ __forceinline__ float value_of_bits(u32 bits) {
    if constexpr (sizeof(T) == 4) {
        return __uint_as_float(bits);
    } else {
        const u16 half = (u16)bits;
        return to_float(*reinterpret_cast<const T*>(&half));
    }
}
template <typename T>
__device__ __forceinline__ float lds_value(u32 at) {
    if constexpr (sizeof(T) == 4) {
        return lds(at);
    } else {
        u16 bits;
        asm volatile("ld.shared.u16 %0, [%1];" : "=h"(bits) : "r"(at));
        return value_of_bits<T>(bits);
    }
}
template <typename T>
__device__ __forceinline__ float lds_value_if(bool there, u32 at) {   // else zero
    if constexpr (sizeof(T) == 4) return value_of_bits<T>(lds_u32_if(there, at));
    else return value_of_bits<T>(lds_u16_if(there, at));
}
__device__ __forceinline__ uint4 lds4(u32 at) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at));
    return v;
}
__device__ __forceinline__ uint2 lds2(u32 at) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(at));
    return v;
}
template <typename T>
__device__ __forceinline__ void sts_value_if(bool there, u32 at, float v) {
    if constexpr (sizeof(T) == 4) {
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %2, 0;\n\t@p st.shared.f32 [%0], %1;\n\t}" ::"r"(at), "f"(v), "r"((int)there) : "memory");
    } else {
        T h = from_float<T>(v);
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %2, 0;\n\t@p st.shared.u16 [%0], %1;\n\t}" ::"r"(at), "h"(*reinterpret_cast<u16*>(&h)), "r"((int)there) : "memory");
    }
}
template <typename T>
__device__ __forceinline__ void sts_value(u32 at, float v) {
    if constexpr (sizeof(T) == 4) {
        asm volatile("st.shared.f32 [%0], %1;" ::"r"(at), "f"(v) : "memory");
    } else {
        T h = from_float<T>(v);
        asm volatile("st.shared.u16 [%0], %1;" ::"r"(at), "h"(*reinterpret_cast<u16*>(&h)) : "memory");
    }
}
__device__ __forceinline__ void sts(u32 at, float v) { asm volatile("st.shared.f32 [%0], %1;" ::"r"(at), "f"(v) : "memory"); }

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
__device__ __forceinline__ void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
__device__ __forceinline__ void bulk_wait_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }

__device__ __forceinline__ float exp2_approx(float v) {   // 2^v, within 2^-22 of it
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}

}  // namespace pl
