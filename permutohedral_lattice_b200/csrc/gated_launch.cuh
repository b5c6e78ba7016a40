// The launches of the gated block's kernels, for the translation units that compile them.
#pragma once
#include <algorithm>

#include "gated.cuh"
#include "host_calls.h"

namespace pl {

int gated_floats(GatedArgs p, GatedPass pass, bool pack, cudaStream_t st);
int gated_halves(GatedArgs p, int dtype, GatedPass pass, bool pack, cudaStream_t st);

constexpr size_t GATED_SMEM = 227 * 1024;   // of a CTA, at most

// CTAs of a chunk of hidden channels when the weights' gradients are summed up.
inline int gated_splits(int chunks, long long rows, int sms) { return (int)std::max(1ll, std::min<long long>(std::max(1, sms / chunks), (rows + 127) / 128)); }

// Buffers, as far as there is room: rows that leave together (or a thread stores its own), the weights of all chunks (else they come anew for every
// tile), of everything else two, so that what comes next is fetched while products run.
template <typename T, GatedPass PASS, int ROWS, bool FINE>
static bool gated_plan(GatedArgs& p) {
    const int chunks = PASS == GATED_DW ? 1 : p.chunks;
    p.box_x = sizeof(T) == 2 && p.wide_x, p.box_grad = sizeof(T) == 2 && PASS != GATED_OUT && p.wide_grad;
    auto fits = [&]() {
        // The weights of all chunks first, or of three: of a step's first products, of its second ones, and on their way; two tiles of rows, and rows
        // that leave together; more of all where there is room.  (154 401 rows of 128 to 512 to 128 float16 channels: 109 us with two buffers of weights
        // and rows that leave together, 119 with three and none.)
        const int io = PASS != GATED_DW && p.wide_out, two = std::min(2, chunks), three = std::min(3, chunks);
        const int before = PASS == GATED_DX ? 0 : io;      // (its operands are twice as large: two of them are worth more)
        const int tries[][4] = {{2, chunks, 2 * io, 2}, {2, chunks, io, 2}, {2, chunks, before, 2}, {2, chunks, 2 * io, 1}, {2, chunks, io, 1}, {1, chunks, io, 1}, {2, three, io, 2},
                                {2, three, io, 1}, {2, three, 0, 1}, {2, two, io, 2}, {2, two, io, 1}, {1, three, io, 2}, {1, three, io, 1}, {2, two, 0, 1},
                                {1, two, io, 2}, {1, two, io, 1}, {1, two, 0, 1}, {1, 1, io, 1}, {1, 1, 0, 1}};
        for (const auto& one : tries) {
            p.x_buffers = one[0], p.w_buffers[0] = p.w_buffers[1] = one[1], p.io_buffers = one[2], p.a_buffers = one[3];
            if (GatedSmem<T, PASS, ROWS, FINE>(p).total > (int)GATED_SMEM) continue;
            while (p.x_buffers >= 2 && p.x_buffers < 4) {
                p.x_buffers++;
                if (GatedSmem<T, PASS, ROWS, FINE>(p).total <= (int)GATED_SMEM) continue;
                p.x_buffers--;
                break;
            }
            return true;
        }
        return false;
    };
    auto columns = [&](int s, int d) {
        p.s_buffers = s, p.d_buffers = d;
        return GatedColumns<T, PASS>(p).total <= 512;
    };
    // What changes a result's bits (rows of a tile, sums side by side) goes by sizes and biases, not by which gradients are wanted.
    const int wanted = p.down_bias_wanted;
    p.down_bias_wanted = PASS == GATED_DW;
    p.stacked = 0, p.split = sizeof(T) == 4 && PASS != GATED_DW && p.h > 256;
    const bool room = fits();
    // float32: side by side as far as a product is wide, 256 columns, and as there is room
    if (PASS == GATED_DW && sizeof(T) == 4 && 3 * p.kx <= 256) {
        p.stacked = 1;
        if (!columns(1, 1)) p.stacked = 0;
    }
    p.down_bias_wanted = wanted;
    return room && ((PASS != GATED_DW && columns(2, 2)) || columns(2, 1) || columns(1, 1));
}

// A matrix of rows as the TMA takes it: boxes of 128 bytes by `box` rows, in shared memory as swizzled_at says.
int encode_matrix(CUtensorMap& map, const void* p, int dtype, unsigned long long rows, unsigned long long columns, unsigned box_columns, unsigned box_rows);
template <typename T>
static int matrix_map(CUtensorMap& map, const void* p, long long rows, int columns, int box) {
    const int dtype = sizeof(T) == 4 ? PL_F32 : std::is_same<T, __half>::value ? PL_F16 : PL_BF16;
    return encode_matrix(map, p, dtype, rows, columns, 128 / sizeof(T), box);
}

template <typename T, GatedPass PASS, int ROWS, bool FINE>
static int launch_gated_rows(GatedArgs& p, cudaStream_t st) {
    const int smem = GatedSmem<T, PASS, ROWS, FINE>(p).total;
    GatedMaps maps = {};
    if (p.box_x) PL_TRY(matrix_map<T>(maps.x, p.x, p.rows, p.k, ROWS));
    if (p.box_grad) PL_TRY(matrix_map<T>(maps.grad, p.grad, p.rows, p.n, ROWS));
    if (p.io_buffers) {
        PL_TRY(matrix_map<T>(maps.out, p.out, p.rows, PASS == GATED_OUT ? p.n : p.k, ROWS));
        if (PASS == GATED_OUT && p.residual) PL_TRY(matrix_map<T>(maps.residual, p.residual, p.rows, p.n, ROWS));
    }
    const long long tiles = (p.rows + ROWS - 1) / ROWS;
    const unsigned grid = PASS == GATED_DW ? p.chunks * p.splits : (unsigned)std::min<long long>(tiles, num_sms());
    PL_TRY((ensure_dynamic_smem<gated_kernel<T, PASS, ROWS, FINE>>(smem)));
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(grid), config.blockDim = dim3(GatedWarps<T>::THREADS), config.dynamicSmemBytes = smem, config.stream = st;
    cudaLaunchAttribute early[1];   // on the SMs, with its barriers set up, when the kernel before it (gated_pack, usually) ends
    early[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early[0].val.programmaticStreamSerializationAllowed = 1;
    config.attrs = early, config.numAttrs = 1;
    PL_CUDA(cudaLaunchKernelEx(&config, gated_kernel<T, PASS, ROWS, FINE>, (const GatedArgs)p, (const GatedMaps)maps));
    PL_COUNT_LAUNCHES(1);
    return PL_OK;
}
template <typename T, GatedPass PASS, bool FINE>
static int launch_gated(GatedArgs& p, cudaStream_t st) {
    // Tiles of 64 rows, the other half of a product idle, where 128 leave no room: the gradients of floats, three terms of everything, from some 90
    // channels on; and the sums over rows of 16-bit values where two tiles of 128 do not fit.
    const bool fits = gated_plan<T, PASS, 128, FINE>(p);
    if (fits && (PASS != GATED_DW || p.x_buffers >= 2)) return launch_gated_rows<T, PASS, 128, FINE>(p, st);
    if constexpr (PASS == GATED_DW || (PASS == GATED_DX && sizeof(T) == 4))
        if (gated_plan<T, PASS, 64, FINE>(p)) return launch_gated_rows<T, PASS, 64, FINE>(p, st);
    return fits && gated_plan<T, PASS, 128, FINE>(p) ? launch_gated_rows<T, PASS, 128, FINE>(p, st) : PL_INTERNAL_ERROR;
}
template <typename T>
static int pack_gated(const GatedArgs& p, cudaStream_t st) {
    const int items = gated_chunk<T>() * (p.np / 8) + p.kp * (2 * gated_chunk<T>() / 8);
    gated_pack<T><<<dim3((items + 255) / 256, p.chunks), 256, 0, st>>>(p);
    PL_COUNT_LAUNCHES(1);
    PL_CUDA(cudaGetLastError());
    return PL_OK;
}
template <typename T, bool FINE>
static int launch_pass(GatedArgs& p, GatedPass pass, cudaStream_t st) {
    return pass == GATED_OUT  ? launch_gated<T, GATED_OUT, FINE>(p, st)
           : pass == GATED_DX ? launch_gated<T, GATED_DX, FINE>(p, st)
                              : launch_gated<T, GATED_DW, FINE>(p, st);
}
// pack: the weights first (a backward pass packs them once for both of its kernels).
template <typename T>
static int gated_of(GatedArgs& p, GatedPass pass, bool pack, cudaStream_t st) {
    p.chunks = (p.h + gated_chunk<T>() - 1) / gated_chunk<T>();
    p.splits = gated_splits(p.chunks, p.rows, num_sms());
    // Tiles whose sums stay in tensor memory.  Floats: of 128, 256, 512 rows the gradients of weights of 75 776 rows of 16 to 32 to 16 are 2.7, 4.0, 7.0e-7 off, and a
    // training step of 3 409 920 of 32 to 128 to 32 takes 9200, 8190, 7720 us.  16-bit types, whose results are rounded at 2^-9 or 2^-12: 8192 rows.
    p.drain = sizeof(T) == 4 ? 2 : 64;
    if (pack) PL_TRY(pack_gated<T>(p, st));
    if constexpr (sizeof(T) == 2)
        if (!p.round_hidden) return launch_pass<T, true>(p, pass, st);
    return launch_pass<T, false>(p, pass, st);
}

}  // namespace pl
