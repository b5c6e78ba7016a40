// The gated feed-forward block: the C entry points (see gated.cuh).
#include "gated_launch.cuh"

namespace pl {

// The driver's function, asked for by name: the library links against the runtime alone.
int encode_matrix(CUtensorMap& map, const void* p, int dtype, unsigned long long rows, unsigned long long columns, unsigned box_columns, unsigned box_rows) {
    static const auto encode = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult found = cudaDriverEntryPointSymbolNotFound;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &found) != cudaSuccess || found != cudaDriverEntryPointSuccess) f = nullptr;
        return reinterpret_cast<decltype(&cuTensorMapEncodeTiled)>(f);
    }();
    if (!encode) return cuda_fail(cudaErrorNotSupported, "cuTensorMapEncodeTiled");
    const size_t size = dtype == PL_F32 ? 4 : 2;
    const cuuint64_t dims[2] = {columns, rows}, strides[1] = {columns * size};
    const cuuint32_t box[2] = {box_columns, box_rows}, steps[2] = {1, 1};
    const auto type = dtype == PL_F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : dtype == PL_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    const CUresult rc = encode(&map, type, 2, const_cast<void*>(p), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return rc == CUDA_SUCCESS ? PL_OK : cuda_fail(cudaErrorInvalidValue, "cuTensorMapEncodeTiled");
}

static int check_gated(const pl_gated_shape* m) {
    if (!m || m->rows < 0 || m->rows > ((long long)1 << 40) || m->k < 1 || m->h < 1 || m->n < 1) return PL_INVALID_ARGUMENT;
    if (m->activation < PL_GATE_SILU || m->activation > PL_GATE_RELU || m->dtype < PL_F32 || m->dtype > PL_BF16) return PL_INVALID_ARGUMENT;
    return m->k > MIX_MOST || m->n > MIX_MOST || m->h > GATED_HIDDEN ? PL_UNSUPPORTED_DIMS : PL_OK;
}
static int chunk_of(const pl_gated_shape* m) { return m->dtype == PL_F32 ? gated_chunk<float>() : gated_chunk<__half>(); }
static bool gated_aligned(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }
static GatedArgs gated_args(const pl_gated_shape* m, const void* x, const void* gate_weight, const void* up_weight, const void* down_weight,
                            const void* gate_bias, const void* up_bias) {
    GatedArgs p = {};
    p.rows = m->rows, p.k = m->k, p.h = m->h, p.n = m->n, p.activation = m->activation, p.scale = m->residual_scale;
    p.round_hidden = m->round_hidden != 0;
    p.x = x;
    p.gate_weight = gate_weight, p.up_weight = up_weight, p.down_weight = down_weight;
    p.gate_bias = gate_bias, p.up_bias = up_bias;
    p.biased = p.gate_bias || p.up_bias;
    p.np = (p.n + 15) / 16 * 16;
    p.wide_x = p.k % 8 == 0 && gated_aligned(x) && p.rows < (1ll << 31) - 128;   // (a row's number is 31 bits for the TMA)
    return p;
}
static void set_columns(GatedArgs& p) { p.kx = (p.k + 15) / 16 * 16, p.kp = p.kx + (p.biased ? 16 : 0); }
static int run_gated(const GatedArgs& p, int dtype, GatedPass pass, bool pack, cudaStream_t st) {
    return dtype == PL_F32 ? gated_floats(p, pass, pack, st) : gated_halves(p, dtype, pass, pack, st);
}
static int most_peaks() { return 2 * num_sms(); }   // CTAs of gated_peak
static size_t packed_bytes(const pl_gated_shape* m) {   // with all biases
    const int chunk = chunk_of(m), chunks = (m->h + chunk - 1) / chunk, kp = (m->k + 15) / 16 * 16 + 16, np = (m->n + 15) / 16 * 16;
    const size_t one = m->dtype == PL_F32 ? gated_down_bytes<float>(np) + gated_up_bytes<float>(kp) : gated_down_bytes<__half>(np) + gated_up_bytes<__half>(kp);
    return one * chunks;
}

}  // namespace pl

using namespace pl;

extern "C" {

int pl_gated_mix_workspace_bytes(const pl_gated_shape* m, int backward, size_t* bytes) {
    PL_TRY(check_gated(m));
    if (!bytes) return PL_INVALID_ARGUMENT;
    *bytes = packed_bytes(m);
    if (!backward) return PL_OK;
    const int chunk = chunk_of(m), chunks = (m->h + chunk - 1) / chunk;
    const size_t columns = (m->k + 15) / 16 * 16 + 16 + chunk + 16;   // with all biases
    *bytes += sizeof(float) * 128 * columns * chunks * gated_splits(chunks, m->rows, num_sms());
    if (m->dtype == PL_F16) *bytes += sizeof(u32) * most_peaks();
    return PL_OK;
}

int pl_gated_mix(const pl_gated_shape* m, void* out, const void* x, const void* gate_weight, const void* up_weight, const void* down_weight,
                 const void* gate_bias, const void* up_bias, const void* down_bias, const void* residual, void* workspace, size_t workspace_bytes,
                 void* stream) {
    PL_TRY(check_gated(m));
    if (m->rows == 0) return PL_OK;
    if (!out || !x || !gate_weight || !up_weight || !down_weight) return PL_INVALID_ARGUMENT;
    if (!workspace || workspace_bytes < packed_bytes(m)) return PL_WORKSPACE_TOO_SMALL;
    if (!gated_aligned(workspace)) return PL_INVALID_ARGUMENT;
    GatedArgs p = gated_args(m, x, gate_weight, up_weight, down_weight, gate_bias, up_bias);
    p.down_bias = down_bias;
    set_columns(p);
    p.packed = static_cast<unsigned char*>(workspace);
    p.out = out, p.residual = residual;
    p.wide_out = p.n % (m->dtype == PL_F32 ? 4 : 8) == 0 && gated_aligned(out) && gated_aligned(residual) && p.rows < (1ll << 31) - 128;
    return run_gated(p, m->dtype, GATED_OUT, true, (cudaStream_t)stream);
}

int pl_gated_mix_backward(const pl_gated_shape* m, const void* grad_out, const void* x, const void* gate_weight, const void* up_weight,
                          const void* down_weight, const void* gate_bias, const void* up_bias, pl_gated_gradients d, void* workspace,
                          size_t workspace_bytes, void* stream) {
    size_t need = 0;
    PL_TRY(pl_gated_mix_workspace_bytes(m, 1, &need));
    const cudaStream_t st = (cudaStream_t)stream;
    const size_t size = m->dtype == PL_F32 ? 4 : 2;
    const bool sums = d.gate_weight || d.up_weight || d.down_weight || d.gate_bias || d.up_bias || d.down_bias;
    if (m->rows == 0) {   // sums of nothing
        const struct { void* to; size_t count; } all[] = {{d.gate_weight, (size_t)m->k * m->h}, {d.up_weight, (size_t)m->k * m->h}, {d.down_weight, (size_t)m->h * m->n},
                                                          {d.gate_bias, (size_t)m->h}, {d.up_bias, (size_t)m->h}, {d.down_bias, (size_t)m->n}};
        for (const auto& a : all)
            if (a.to) PL_CUDA(cudaMemsetAsync(a.to, 0, size * a.count, st));
        return PL_OK;
    }
    if (!grad_out || !x || !gate_weight || !up_weight || !down_weight) return PL_INVALID_ARGUMENT;
    if (!workspace || workspace_bytes < need) return PL_WORKSPACE_TOO_SMALL;
    if (!gated_aligned(workspace)) return PL_INVALID_ARGUMENT;
    GatedArgs p = gated_args(m, x, gate_weight, up_weight, down_weight, gate_bias, up_bias);
    p.grad = grad_out;
    p.wide_grad = p.n % 8 == 0 && gated_aligned(grad_out) && p.rows < (1ll << 31) - 128;
    p.biased = p.biased || d.gate_bias || d.up_bias;   // (the ones' column sums dg and du)
    set_columns(p);
    p.packed = static_cast<unsigned char*>(workspace);
    // s dout by the kernel of dx where it has the rows at hand (16-bit rows by the TMA) or a loader to spare (floats), else by itself.
    const bool beside = d.x && (m->dtype == PL_F32 || (p.wide_x && p.wide_grad && gated_aligned(d.residual)));
    if (d.residual && !beside) {
        const pl_dropout none = {};
        PL_TRY(pl_channel_dropout(nullptr, d.residual, grad_out, nullptr, m->rows * m->n, m->dtype, m->residual_scale, &none, nullptr, stream));
    }
    if (m->dtype == PL_F16 && (d.x || sums)) {
        const long long count = m->rows * m->n, per = 256 * 8 * 4;
        u32* peaks = reinterpret_cast<u32*>(p.packed + need) - most_peaks();
        p.peaks = peaks, p.peak_count = (int)std::min<long long>((count + per - 1) / per, most_peaks());
        gated_peak<<<p.peak_count, 256, 0, st>>>(static_cast<const __half*>(grad_out), count, peaks);
        PL_COUNT_LAUNCHES(1);
        PL_CUDA(cudaGetLastError());
    }
    if (d.x) {
        p.out = d.x, p.dresidual = beside ? d.residual : nullptr;
        p.wide_out = p.k % (m->dtype == PL_F32 ? 4 : 8) == 0 && gated_aligned(d.x) && p.rows < (1ll << 31) - 128;
        p.wide_dresidual = gated_aligned(grad_out) && gated_aligned(d.residual);
        PL_TRY(run_gated(p, m->dtype, GATED_DX, true, st));
    }
    if (!sums) return PL_OK;
    p.down_bias_wanted = d.down_bias != nullptr;
    p.shares = reinterpret_cast<float*>(p.packed + packed_bytes(m));
    PL_TRY(run_gated(p, m->dtype, GATED_DW, !d.x, st));
    GatedSums s = {};
    s.shares = p.shares, s.k = p.k, s.h = p.h, s.n = p.n, s.kx = p.kx, s.chunk = chunk_of(m);
    s.chunks = (p.h + s.chunk - 1) / s.chunk, s.splits = gated_splits(s.chunks, m->rows, num_sms());
    s.down = p.kp, s.bias = s.down + s.chunk, s.columns = s.bias + (p.down_bias_wanted ? 16 : 0);
    s.gate_weight = d.gate_weight, s.up_weight = d.up_weight, s.down_weight = d.down_weight;
    s.gate_bias = d.gate_bias, s.up_bias = d.up_bias, s.down_bias = d.down_bias;
    const dim3 grid((std::max(p.h, p.n) + 255) / 256, 2 * (p.k + 1) + p.h + 1);
    if (m->dtype == PL_F32) gated_sums<float><<<grid, 256, 0, st>>>(s);
    else if (m->dtype == PL_F16) gated_sums<__half><<<grid, 256, 0, st>>>(s);
    else gated_sums<__nv_bfloat16><<<grid, 256, 0, st>>>(s);
    PL_COUNT_LAUNCHES(1);
    PL_CUDA(cudaGetLastError());
    return PL_OK;
}

}  // extern "C"
