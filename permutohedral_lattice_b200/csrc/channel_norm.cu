// Norms after and before a block with dropout, gate and residual, and dropout by itself: the C entry points (see channel_norm.cuh).
#include "norm_launch.cuh"

namespace pl {

constexpr int NORM_CTAS = 4;   // of an SM: as many shares of the sums there may be

static int check_norm(const pl_channel_norm_shape* m) {
    if (!m || m->rows < 0 || m->channels < 1 || m->rows > ((long long)1 << 40)) return PL_INVALID_ARGUMENT;
    if (m->dtype < PL_F32 || m->dtype > PL_BF16) return PL_INVALID_ARGUMENT;
    if (m->vector_dtype != PL_F32 && m->vector_dtype != m->dtype) return PL_INVALID_ARGUMENT;
    for (const pl_norm* n : {&m->after, &m->before}) {
        if (n->kind < PL_NORM_NONE || n->kind > PL_NORM_RMS) return PL_INVALID_ARGUMENT;
        if (n->kind != PL_NORM_NONE && !(n->eps > 0.f && n->eps <= 3.402e38f)) return PL_INVALID_ARGUMENT;
    }
    if (!(m->dropout.p >= 0.0 && m->dropout.p < 1.0)) return PL_INVALID_ARGUMENT;
    return m->channels > NORM_MOST ? PL_UNSUPPORTED_DIMS : PL_OK;
}
static Dropout dropout_of(const pl_dropout& d, const int64_t* seed) {
    Dropout r = {};
    r.threshold = (u32)std::min(d.p * 4294967296.0 + 0.5, 4294967295.0);
    r.scale = (float)(1.0 / (1.0 - d.p));
    r.key = d.key, r.offset = d.offset, r.seed = reinterpret_cast<const long long*>(seed);
    return r;
}
static NormArgs norm_args(const pl_channel_norm_shape* m, const void* x, const void* residual, const void* gate, const void* after_weight,
                          const void* after_bias, const void* before_weight, const void* before_bias, const int64_t* seed) {
    NormArgs a = {};
    a.rows = m->rows, a.c = m->channels;
    a.after = m->after.kind, a.before = m->before.kind;
    a.eps_after = m->after.eps, a.eps_before = m->before.eps, a.scale = m->residual_scale;
    a.x = x, a.residual = residual, a.gate = m->gate_of_values ? gate : nullptr;
    if (a.after) a.vectors[NORM_WA] = after_weight, a.vectors[NORM_BA] = after_bias;
    if (a.before) a.vectors[NORM_WB] = before_weight, a.vectors[NORM_BB] = before_bias;
    a.vectors[NORM_GATE] = m->gate_of_values ? nullptr : gate;
    a.vector_dtype = m->vector_dtype;
    a.drop = dropout_of(m->dropout, seed);
    return a;
}
static int run_norm(NormArgs& a, int dtype, bool backward, cudaStream_t st) {
    const int ctas = num_sms() * (backward ? NORM_CTAS : 8);
    return dtype == PL_F32 ? norm_of_floats(a, backward, ctas, st) : dtype == PL_F16 ? norm_of_halves(a, backward, ctas, st) : norm_of_bfloats(a, backward, ctas, st);
}
template <typename T>
static int launch_drop(const DropArgs& a, cudaStream_t st) {
    constexpr int V = Piece<T, true>::V;
    const long long per = 256 * V * DROP_PIECES;
    const unsigned grid = (unsigned)std::max(1ll, std::min((a.n + per - 1) / per, (long long)num_sms() * 8));
    if (norm_aligned(a.x) && norm_aligned(a.residual) && norm_aligned(a.out) && norm_aligned(a.scaled)) drop_values<T, true><<<grid, 256, 0, st>>>(a);
    else drop_values<T, false><<<grid, 256, 0, st>>>(a);
    PL_COUNT_LAUNCHES(1);
    PL_CUDA(cudaGetLastError());
    return PL_OK;
}

}  // namespace pl

using namespace pl;

extern "C" {

int pl_channel_norm(const pl_channel_norm_shape* m, void* h, void* y, const void* x, const void* residual, const void* gate, const void* after_weight,
                    const void* after_bias, const void* before_weight, const void* before_bias, const int64_t* seed, void* stream) {
    PL_TRY(check_norm(m));
    if (m->rows == 0) return PL_OK;
    if (!x || (!h && !y) || (y != nullptr) != (m->before.kind != PL_NORM_NONE)) return PL_INVALID_ARGUMENT;
    NormArgs a = norm_args(m, x, residual, gate, after_weight, after_bias, before_weight, before_bias, seed);
    a.h = h, a.y = y;
    return run_norm(a, m->dtype, false, (cudaStream_t)stream);
}

int pl_channel_norm_workspace_bytes(const pl_channel_norm_shape* m, size_t* bytes) {
    PL_TRY(check_norm(m));
    if (!bytes) return PL_INVALID_ARGUMENT;
    *bytes = sizeof(float) * NORM_VECTORS * (size_t)m->channels * num_sms() * NORM_CTAS;
    return PL_OK;
}

int pl_channel_norm_backward(const pl_channel_norm_shape* m, const void* dh, const void* dy, const void* x, const void* residual, const void* gate,
                             const void* after_weight, const void* after_bias, const void* before_weight, const int64_t* seed, pl_norm_gradients d,
                             void* workspace, size_t workspace_bytes, void* stream) {
    size_t need = 0;
    PL_TRY(pl_channel_norm_workspace_bytes(m, &need));
    const cudaStream_t st = (cudaStream_t)stream;
    const bool values = m->gate_of_values != 0;
    void* vectors[NORM_VECTORS] = {d.after_weight, d.after_bias, d.before_weight, d.before_bias, values ? nullptr : d.gate};
    if (m->rows == 0) {   // sums of nothing
        for (void* p : vectors)
            if (p) PL_CUDA(cudaMemsetAsync(p, 0, (m->vector_dtype == PL_F32 ? 4 : 2) * (size_t)m->channels, st));
        return PL_OK;
    }
    if ((!dh && !dy) || (dy != nullptr) != (m->before.kind != PL_NORM_NONE)) return PL_INVALID_ARGUMENT;
    if ((d.after_weight || d.after_bias) && !m->after.kind) return PL_INVALID_ARGUMENT;
    if ((d.before_weight || d.before_bias) && !m->before.kind) return PL_INVALID_ARGUMENT;
    if (!x && (m->after.kind || m->before.kind || d.gate)) return PL_INVALID_ARGUMENT;
    if (!workspace || workspace_bytes < need) return PL_WORKSPACE_TOO_SMALL;
    if (!norm_aligned(workspace)) return PL_INVALID_ARGUMENT;
    NormArgs a = norm_args(m, x, residual, gate, after_weight, after_bias, before_weight, nullptr, seed);
    a.dh = dh, a.dy = dy, a.dx = d.x, a.dresidual = d.residual, a.dgate = values ? d.gate : nullptr;
    for (int v = 0; v < NORM_VECTORS; v++) a.wanted |= vectors[v] ? 1 << v : 0;
    if (a.wanted) a.shares = static_cast<float*>(workspace);
    PL_TRY(run_norm(a, m->dtype, true, st));
    if (!a.wanted) return PL_OK;
    NormSums s = {a.shares, a.ctas, a.c, m->vector_dtype, {}};
    for (int v = 0; v < NORM_VECTORS; v++) s.to[v] = vectors[v];
    norm_sums<<<dim3((a.c + 31) / 32, NORM_VECTORS), NORM_THREADS, 0, st>>>(s);
    PL_COUNT_LAUNCHES(1);
    PL_CUDA(cudaGetLastError());
    return PL_OK;
}

int pl_channel_dropout(void* out, void* scaled, const void* x, const void* residual, int64_t n, int dtype, float residual_scale,
                       const pl_dropout* dropout, const int64_t* seed, void* stream) {
    if (n < 0 || dtype < PL_F32 || dtype > PL_BF16 || !dropout || !(dropout->p >= 0.0 && dropout->p < 1.0)) return PL_INVALID_ARGUMENT;
    if (n == 0) return PL_OK;
    if ((!out && !scaled) || !x) return PL_INVALID_ARGUMENT;
    const DropArgs a = {n, x, residual, out, scaled, residual_scale, dropout_of(*dropout, seed)};
    const cudaStream_t st = (cudaStream_t)stream;
    return dtype == PL_F32 ? launch_drop<float>(a, st) : dtype == PL_F16 ? launch_drop<__half>(a, st) : launch_drop<__nv_bfloat16>(a, st);
}

}  // extern "C"
