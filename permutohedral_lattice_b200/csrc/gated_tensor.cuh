// Fifth-generation tensor cores for the gated feed-forward block: 16-bit operands in shared memory, sums in tensor memory.
//
// Operands.  A tile of rows x columns lies as blocks of 8 rows by 8 columns, 16 bytes a row and 128 a block, blocks of the same columns
// one after another.  The same bytes serve as an operand whose sums run over the columns (K-major) and as one whose sums run over the
// rows (MN-major): nothing is ever transposed, x and what is made of it are operands both ways.  Threads with eight rows of a block access it
// together, in all banks.
//
// Terms.  A float is the sum of three bfloat16 numbers up to 2^-27 of it, each the nearest to what is left, and a product of two
// floats that of the six pairs whose orders of magnitude are above 2^-24 of it: as many steps as three products of tf32 numbers would
// take, 2^-22 off then, from 6 bytes a value in place of 8, and either major.  16-bit values are their own only term.
//
// Sums.  The tensor cores cut what they add to, a part in 2^24 a step of 16 on average toward zero.  Small products come first, or (over more
// than 128 terms) have sums of their own.
#pragma once
#include "mix_common.cuh"

namespace pl {

template <typename T>
struct Tensor {
    static constexpr int TERMS = sizeof(T) == 4 ? 3 : 1;
    static constexpr u32 FORMAT = std::is_same<T, __half>::value ? 0 : 1;   // of an operand: float16, bfloat16
    using Term = typename std::conditional<sizeof(T) == 4, __nv_bfloat16, T>::type;
};

// Bytes from one block of columns to the next, of a tile of so many rows, and of a tile.
__host__ __device__ constexpr int column_blocks(int rows) { return rows * 16; }
__host__ __device__ constexpr int tile_bytes(int rows, int columns) { return rows * columns * 2; }   // of a term

struct Operand {   // of a product: its first 16 terms of the sum, how far the next 16 are, the next 64, and the next term (in 16 bytes)
    u64 first;
    u32 step, jump, plane, transposed;
    __device__ __forceinline__ u64 at(int s, int term) const {   // (addresses are below 2^18: nothing is carried)
        return first + (u32)((s & 3) * step + (s >> 2) * jump + term * plane);
    }
};
__device__ __forceinline__ u64 operand_of(u32 at, u32 along, u32 across) {   // strides of blocks, along the sums and across
    return (u64)(at >> 4) | (u64)(along >> 4) << 16 | (u64)(across >> 4) << 32 | 1ull << 46;
}
// The tile's rows are the operand's rows, sums run over its columns.
__device__ __forceinline__ Operand over_columns(u32 at, int rows, int columns) {
    return {operand_of(at, column_blocks(rows), 128), (u32)column_blocks(rows) / 8, (u32)column_blocks(rows) / 2, (u32)tile_bytes(rows, columns) / 16, 0};
}
// The tile's columns are the operand's rows, sums run over its rows.
__device__ __forceinline__ Operand over_rows(u32 at, int rows, int columns) {
    return {operand_of(at, 128, column_blocks(rows)), 16, 64, (u32)tile_bytes(rows, columns) / 16, 1};
}
// Tiles of rows of 16-bit values, which the TMA brings: 64 columns after another, rows of 128 bytes whose 16-byte pieces lie at their number
// xor the row's (mod 8).  Either way round as well.
constexpr u64 SWIZZLED = 2ull << 61;
__host__ __device__ constexpr int swizzled_bytes(int rows, int row_bytes) { return (row_bytes + 127) / 128 * rows * 128; }
__device__ __forceinline__ int swizzled_at(int rows, int row, int piece) { return (piece >> 3) * rows * 128 + row * 128 + ((piece & 7) ^ (row & 7)) * 16; }
__device__ __forceinline__ Operand swizzled_over_columns(u32 at, int rows) { return {operand_of(at, 16, 1024) | SWIZZLED, 2, (u32)rows * 8, 0, 0}; }
__device__ __forceinline__ Operand swizzled_over_rows(u32 at, int rows) { return {operand_of(at, rows * 128, 1024) | SWIZZLED, 128, 512, 0, 1}; }
__device__ __forceinline__ void tensor_product(u32 d, u64 a, u64 b, u32 shape, bool add) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b),
                 "r"(shape), "r"((u32)add)
                 : "memory");
}
template <typename T>
__device__ __forceinline__ u32 product_shape(const Operand& a, const Operand& b, int n) {   // 128 x n
    return 1u << 4 | Tensor<T>::FORMAT << 7 | Tensor<T>::FORMAT << 10 | a.transposed << 15 | b.transposed << 16 | (u32)(n / 8) << 17 | 8u << 24;
}
// The same of 16-bit operands, one of which may be of two terms: the small one's products first.
template <typename T, int A_TERMS, int B_TERMS>
__device__ __forceinline__ void few_products(u32 d, const Operand& a, const Operand& b, int n, int steps, bool add) {
    static_assert(A_TERMS * B_TERMS <= 2);
    const u32 shape = product_shape<T>(a, b, n);
#pragma unroll
    for (int i = A_TERMS * B_TERMS - 1; i >= 0; i--) {
#pragma unroll 4
        for (int s = 0; s < steps; s++) {
            tensor_product(d, a.at(s, A_TERMS == 2 ? i : 0), b.at(s, B_TERMS == 2 ? i : 0), shape, add);
            add = true;
        }
    }
}
// d (+)= a b^T over 16 `steps` terms, 128 x n; small: where products with a term but the first go (may be d).  add, add_small: to what is there.
template <typename T>
__device__ __forceinline__ void products(u32 d, u32 small, const Operand& a, const Operand& b, int n, int steps, bool add, bool add_small) {
    const u32 shape = product_shape<T>(a, b, n);
    if constexpr (Tensor<T>::TERMS == 3) {
        bool more = add_small;
#pragma unroll
        for (int order = 2; order >= 1; order--)
#pragma unroll
            for (int i = 0; i <= order; i++)
#pragma unroll 2
                for (int s = 0; s < steps; s++) {
                    tensor_product(small, a.at(s, i), b.at(s, order - i), shape, more);
                    more = true;
                }
        if (small == d) add = true;
    }
#pragma unroll 4
    for (int s = 0; s < steps; s++) {
        tensor_product(d, a.at(s, 0), b.at(s, 0), shape, add);
        add = true;
    }
}
// The same with b's three terms side by side (as they lie behind one another in a tile whose columns are the operand's rows): three products in place
// of six, whose first operands, which take as long to read as 64 columns to multiply, are read half as often.  What is n columns further on is a part in 2^8 of it.
template <typename T>
__device__ __forceinline__ void stacked_products(u32 d, const Operand& a, const Operand& b, int n, int steps, bool add) {
#pragma unroll
    for (int i = 0; i < 3; i++) {
        const u32 shape = product_shape<T>(a, b, (3 - i) * n);
#pragma unroll 2
        for (int s = 0; s < steps; s++) tensor_product(d + i * n, a.at(s, i), b.at(s, 0), shape, add || i > 0 || s > 0);
    }
}
__device__ __forceinline__ void tensor_commit(u64* bar) {   // the barrier's phase ends when all products asked for so far are done
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(shared_address(bar)) : "memory");
}
__device__ __forceinline__ void tensor_load(float (&v)[16], u32 at) {   // columns of the lane's row; there after tensor_loaded
    u32* r = reinterpret_cast<u32*>(v);
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
                   "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(at));
}
__device__ __forceinline__ void tensor_load(float (&v)[8], u32 at) {
    u32* r = reinterpret_cast<u32*>(v);
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(at));
}
__device__ __forceinline__ void tensor_loaded() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tensor_before_sync() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tensor_after_sync() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void mbar_arrive(u64* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(shared_address(bar)) : "memory");
}

__device__ __forceinline__ bool mbar_done(u64* bar, u32 parity) {   // sleeps for up to 20 us
    u32 done;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(done)
                 : "r"(shared_address(bar)), "r"(parity), "r"(20000u)
                 : "memory");
    return done != 0;
}
__device__ __forceinline__ u64 global_timer() {   // nanoseconds
    u64 t;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
    return t;
}

__device__ __forceinline__ bool one_of_warp() {   // one lane, known as such to the compiler: what is the same for a warp stays in its uniform registers
    u32 one;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
    return one != 0;
}
// Boxes of a matrix in memory to shared memory and back by the TMA: columns from x on, rows from y on; what lies outside comes as zeros and is not
// written.
__device__ __forceinline__ void box_load(void* to, const void* map, int x, int y, u64* bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(shared_address(to)),
                 "l"(map), "r"(x), "r"(y), "r"(shared_address(bar))
                 : "memory");
}
__device__ __forceinline__ void box_store(const void* map, int x, int y, const void* from) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(map), "r"(x), "r"(y), "r"(shared_address(from)) : "memory");
}
__device__ __forceinline__ void bulk_wait_all() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

// Eight values as terms to a row of a block, 16 bytes each.
template <typename T, int TERMS = Tensor<T>::TERMS>
__device__ __forceinline__ void store_terms8(unsigned char* to, int plane, const float (&v)[8]) {
    using Term = typename Tensor<T>::Term;
    float left[8];
#pragma unroll
    for (int i = 0; i < 8; i++) left[i] = v[i];
#pragma unroll
    for (int t = 0; t < TERMS; t++) {
        uint4 q;
        Term* e = reinterpret_cast<Term*>(&q);
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
            if constexpr (std::is_same<Term, __half>::value) reinterpret_cast<__half2*>(&q)[i / 2] = __floats2half2_rn(left[i], left[i + 1]);
            else reinterpret_cast<__nv_bfloat162*>(&q)[i / 2] = __floats2bfloat162_rn(left[i], left[i + 1]);
            if (t + 1 < TERMS) left[i] -= to_float(e[i]), left[i + 1] -= to_float(e[i + 1]);
        }
        *reinterpret_cast<uint4*>(to + t * plane) = q;
    }
}

}  // namespace pl
