// taco_linear_attention, _backward, _step (include/taco_sequence.h)
#include "seq_host.hpp"
#include "seq_linear.hpp"

namespace seq {

static int check_args(const taco_linear_attention_args *a) {
    SEQ_NEED(a, "args: null");
    if (int rc = check_dims(a->heads, a->heads, a->dim, a->dtype)) return rc;
    SEQ_NEED(__builtin_fabsf(a->scale) >= 1.17549435e-38f && __builtin_fabsf(a->scale) < __builtin_inff(), "scale %g: finite and not 0 (nor below float32's normal range)", (double)a->scale);
    SEQ_NEED(a->n_sequences >= 0 && a->n_segments >= a->n_sequences, "%d segments of %d sequences", a->n_segments, a->n_sequences);
    SEQ_NEED((int64_t)a->n_sequences * a->heads <= 65535 || a->n_segments == a->n_sequences, "%d sequences of %d heads: at most 65535 in all where they are cut into segments",
             a->n_sequences, a->heads);
    return 0;
}
static size_t workspace_for(const taco_linear_attention_args *a, int modes) {
    const int64_t dp = padded_dim(a->dim);
    return a->n_segments == a->n_sequences ? 0 : (size_t)(modes * dp * dp * sizeof(float)) * a->n_segments * a->heads;
}

static int run(const taco_linear_attention_args *a, LinearParams &p, int modes, void *stream) {
    SEQ_NEED(a->log_decay && a->segments && a->first_segment, "log_decay, segments or first_segment: null");
    const size_t need = workspace_for(a, modes);
    if (need && (!a->workspace || (uintptr_t)a->workspace % 16 || a->workspace_bytes < need))
        return fail(TACO_SEQ_ERR_WORKSPACE, "workspace: %zu bytes, 16-byte aligned, are needed, %zu given", need, a->workspace ? a->workspace_bytes : (size_t)0);
    p.log_decay = a->log_decay;
    p.segments = a->segments;
    p.first_segment = a->first_segment;
    p.n_segments = a->n_segments;
    p.n_sequences = a->n_sequences;
    p.heads = a->heads;
    p.dim = a->dim;
    p.carry = need ? (float *)a->workspace : nullptr;
    return dispatch(a->dtype, a->dim, [&](auto type, auto dp) {
        typedef decltype(type) T;
        constexpr int DP = decltype(dp)::value;
        auto segments = [&](int threads, auto kernel) {
            in_launches(p.n_segments, threads, [&](int32_t first, uint32_t n) {
                p.first_block = first;
                kernel<<<dim3(n, (unsigned)p.heads, (unsigned)modes), threads, 0, (hipStream_t)stream>>>(p);
            });
        };
        if (p.carry) {
            segments(2 * DP * (chunk_of<T> / 32), linear_kernel<T, DP, true>);
            linear_scan_kernel<DP><<<dim3(DP * DP / 256, (unsigned)(p.n_sequences * p.heads), (unsigned)modes), 256, 0, (hipStream_t)stream>>>(p);
        }
        segments(4 * DP, linear_kernel<T, DP, false>);
        return launched("taco_linear_attention");
    });
}

}  // namespace seq

SEQ_API size_t taco_linear_attention_workspace_bytes(const taco_linear_attention_args *a, int backward) {
    return seq::check_args(a) ? 0 : seq::workspace_for(a, backward ? 3 : 1);
}

SEQ_API int taco_linear_attention(const taco_linear_attention_args *a, void *stream) {
    using namespace seq;
    if (int rc = check_args(a)) return rc;
    if (a->n_segments == 0) return TACO_SEQ_OK;
    LinearParams p{};
    LinearMode &m = p.mode[0];
    const struct { const char *name; const taco_seq_tensor *t; View *v; } all[] = {{"q", &a->q, &m.q}, {"k", &a->k, &m.k}, {"v", &a->v, &m.v}, {"o", &a->o, &m.o}};
    for (const auto &x : all) {
        if (int rc = check_tensor(x.name, *x.t, a->dim, a->dtype)) return rc;
        *x.v = view(*x.t, a->dtype);
    }
    m.s0 = a->state0;
    m.last = a->state_last;
    m.shift = 1;
    m.scale = a->scale;
    m.s0_scale = m.last_scale = 1.f;
    return run(a, p, 1, stream);
}

SEQ_API int taco_linear_attention_backward(const taco_linear_attention_args *a, void *stream) {
    using namespace seq;
    if (int rc = check_args(a)) return rc;
    if (a->n_segments == 0) return TACO_SEQ_OK;
    View q, k, v, g, dq, dk, dv;
    const struct { const char *name; const taco_seq_tensor *t; View *v; } all[] = {
        {"q", &a->q, &q}, {"k", &a->k, &k}, {"v", &a->v, &v}, {"d_o", &a->d_o, &g}, {"d_q", &a->d_q, &dq}, {"d_k", &a->d_k, &dk}, {"d_v", &a->d_v, &dv}};
    for (const auto &x : all) {
        if (int rc = check_tensor(x.name, *x.t, a->dim, a->dtype)) return rc;
        *x.v = view(*x.t, a->dtype);
    }
    LinearParams p{};
    const float s = a->scale;
    p.mode[0] = LinearMode{g, v, k, dq, a->state0, nullptr, 0, 1, 1, s, 1.f, 1.f};
    p.mode[1] = LinearMode{v, g, q, dk, a->d_state_last, nullptr, 1, 1, 0, s, 1.f / s, 1.f};
    p.mode[2] = LinearMode{k, q, g, dv, a->d_state_last, a->d_state0, 1, 0, 0, s, 1.f / s, s};
    return run(a, p, 3, stream);
}

SEQ_API int taco_linear_attention_step(const taco_linear_attention_step_args *a, void *stream) {
    using namespace seq;
    SEQ_NEED(a, "args: null");
    if (int rc = check_dims(a->heads, a->heads, a->dim, a->dtype)) return rc;
    SEQ_NEED(a->scale != 0.f && __builtin_fabsf(a->scale) < __builtin_inff(), "scale %g: finite and not 0", (double)a->scale);
    SEQ_NEED(a->rows >= 0 && (int64_t)a->rows * a->heads < (int64_t)1 << 31, "%d rows of %d heads: fewer than 2^31 in all", a->rows, a->heads);
    SEQ_NEED(!a->reset || a->reset_bytes == 1 || a->reset_bytes == 4 || a->reset_bytes == 8, "reset_bytes %d: 1, 4 or 8", a->reset_bytes);
    if (a->rows == 0) return TACO_SEQ_OK;
    LinearStepParams p{};
    const struct { const char *name; const taco_seq_tensor *t; View *v; } all[] = {{"q", &a->q, &p.q}, {"k", &a->k, &p.k}, {"v", &a->v, &p.v}, {"o", &a->o, &p.o}};
    for (const auto &x : all) {
        if (int rc = check_tensor(x.name, *x.t, a->dim, a->dtype)) return rc;
        *x.v = view(*x.t, a->dtype);
    }
    if (int rc = check_pointer("state", a->state)) return rc;
    SEQ_NEED(a->log_decay, "log_decay: null");
    p.log_decay = a->log_decay;
    p.state = a->state;
    p.reset = (const uint8_t *)a->reset;
    p.reset_bytes = a->reset_bytes;
    p.rows = a->rows;
    p.heads = a->heads;
    p.dim = a->dim;
    p.scale = a->scale;
    in_launches((int64_t)a->rows * a->heads, 256, [&](int32_t first, uint32_t grid) {
        p.first_block = first;
        if (a->dtype == TACO_SEQ_F32) linear_step_kernel<float><<<grid, 256, 0, (hipStream_t)stream>>>(p);
        else if (a->dtype == TACO_SEQ_F16) linear_step_kernel<f16><<<grid, 256, 0, (hipStream_t)stream>>>(p);
        else linear_step_kernel<bf16><<<grid, 256, 0, (hipStream_t)stream>>>(p);
    });
    return launched("taco_linear_attention_step");
}
