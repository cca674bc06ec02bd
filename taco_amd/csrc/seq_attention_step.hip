// taco_attention_step (include/taco_sequence.h)
#include "seq_host.hpp"
#include "seq_attention_step.hpp"

namespace seq {

// Keys per workgroup: enough workgroups to keep every CU's loads in flight (256 CUs, two workgroups on each, and some rounds of them because rows differ in
// length), but pieces long enough that a piece's partial result (written and read once, float32) stays small beside its keys.
static int32_t piece_of(const taco_attention_step_args *a) {
    const int64_t room = (int64_t)a->table_width * a->page_size, blocks = (a->heads / a->kv_heads + 31) / 32;
    const int64_t all = room * a->rows * a->kv_heads * blocks, want = (all / 2048 + 127) / 128 * 128;
    int64_t piece = want < 256 ? 256 : want;
    while ((room + piece - 1) / piece > 65535) piece *= 2;
    return (int32_t)(piece < (1 << 30) ? piece : 1 << 30);
}
static int64_t pieces_for(const taco_attention_step_args *a) {
    const int64_t room = (int64_t)a->table_width * a->page_size, piece = piece_of(a);
    return room <= 0 ? 1 : (room + piece - 1) / piece;
}
static int check_shape(const taco_attention_step_args *a) {
    SEQ_NEED(a, "args: null");
    if (int rc = check_dims(a->heads, a->kv_heads, a->dim, a->dtype)) return rc;
    SEQ_NEED(a->rows >= 0 && a->table_width >= 1 && a->page_size >= 1 && a->num_pages >= 1, "rows %d, table_width %d, page_size %d, num_pages %d: at least 0, 1, 1, 1",
             a->rows, a->table_width, a->page_size, a->num_pages);
    SEQ_NEED((int64_t)a->rows * a->heads < (int64_t)1 << 31, "%d rows of %d heads: fewer than 2^31 in all", a->rows, a->heads);
    return 0;
}
static size_t workspace_for(const taco_attention_step_args *a) {
    const int64_t n = pieces_for(a);
    return n == 1 ? 0 : (size_t)a->rows * a->heads * n * (padded_dim(a->dim) + 2) * sizeof(float);
}

}  // namespace seq

SEQ_API size_t taco_attention_step_workspace_bytes(const taco_attention_step_args *a) { return seq::check_shape(a) ? 0 : seq::workspace_for(a); }

SEQ_API int taco_attention_step(const taco_attention_step_args *a, void *stream) {
    using namespace seq;
    if (int rc = check_shape(a)) return rc;
    SEQ_NEED(a->scale > 0.f && a->scale < __builtin_inff(), "scale %g: positive and finite", (double)a->scale);
    if (a->rows == 0) return TACO_SEQ_OK;
    StepParams p{};
    const bool joins = a->k_new.ptr || a->v_new.ptr;
    const struct { const char *name; const taco_seq_tensor *t; View *v; int on; } all[] = {
        {"q", &a->q, &p.q, 1}, {"o", &a->o, &p.o, 1}, {"k_new", &a->k_new, &p.k_new, joins}, {"v_new", &a->v_new, &p.v_new, joins}};
    for (const auto &x : all)
        if (x.on) {
            if (int rc = check_tensor(x.name, *x.t, a->dim, a->dtype)) return rc;
            *x.v = view(*x.t, a->dtype);
        }
    if (int rc = check_stride("q head", a->q.head_stride, a->dim, a->dtype)) return rc;
    SEQ_NEED(a->q.head_stride <= (int64_t)1 << 21, "q: head stride of %lld elements: at most 2097152", (long long)a->q.head_stride);
    if (int rc = check_pointer("k_pages", a->k_pages)) return rc;
    if (int rc = check_pointer("v_pages", a->v_pages)) return rc;
    const struct { const char *name; int64_t from, *to; } strides[] = {
        {"k_pages page", a->k_page_stride, &p.k_ps}, {"k_pages token", a->k_token_stride, &p.k_ts}, {"k_pages head", a->k_head_stride, &p.k_hs},
        {"v_pages page", a->v_page_stride, &p.v_ps}, {"v_pages token", a->v_token_stride, &p.v_ts}, {"v_pages head", a->v_head_stride, &p.v_hs}};
    for (const auto &x : strides) {
        if (int rc = check_stride(x.name, x.from, 0, a->dtype)) return rc;
        *x.to = x.from * size_of(a->dtype);
    }
    SEQ_NEED(a->table && a->lengths, "table or lengths: null");
    const size_t need = workspace_for(a);
    if (need && (!a->workspace || (uintptr_t)a->workspace % 16 || a->workspace_bytes < need))
        return fail(TACO_SEQ_ERR_WORKSPACE, "workspace: %zu bytes, 16-byte aligned, are needed, %zu given", need, a->workspace ? a->workspace_bytes : (size_t)0);
    p.k_pages = (char *)a->k_pages;
    p.v_pages = (char *)a->v_pages;
    p.table = a->table;
    p.table_stride = a->table_stride;
    p.lengths = a->lengths;
    p.rows = a->rows;
    p.table_width = a->table_width;
    p.num_pages = a->num_pages;
    p.page_size = a->page_size;
    p.heads = a->heads;
    p.kv_heads = a->kv_heads;
    p.dim = a->dim;
    p.blocks = (a->heads / a->kv_heads + 31) / 32;
    p.piece = piece_of(a);
    p.pieces = (int32_t)pieces_for(a);
    p.scale = a->scale;
    const int64_t room = (int64_t)a->table_width * a->page_size;
    const int cols = a->heads / a->kv_heads < 32 ? a->heads / a->kv_heads : 32;
    const bool few = room <= 64;        // two tiles: one wavefront, no join
    return dispatch(a->dtype, a->dim, [&](auto type, auto dp) {
        typedef decltype(type) T;
        constexpr int DP = decltype(dp)::value;
        p.part_o = (float *)a->workspace;
        p.part_ml = p.part_o + (int64_t)p.rows * p.heads * p.pieces * DP;
        const int nw = few ? 1 : 4, tiles = nw * 32 * Tile<T, DP>::ROW, join = nw * cols * (DP + 2) * (int)sizeof(float);
        const size_t lds = tiles > join ? tiles : join;
        in_launches((int64_t)p.rows * p.kv_heads * p.blocks, 64 * nw, [&](int32_t first, uint32_t n) {
            const dim3 grid(n, (unsigned)p.pieces);
            p.first_block = first;
            if (few) attention_step_kernel<T, DP, 1><<<grid, 64, lds, (hipStream_t)stream>>>(p);
            else attention_step_kernel<T, DP, 4><<<grid, 256, lds, (hipStream_t)stream>>>(p);
        });
        if (p.pieces > 1)
            in_launches((int64_t)p.rows * p.heads, 64, [&](int32_t first, uint32_t n) {
                p.first_block = first;
                attention_join_kernel<T, DP><<<n, 64, 0, (hipStream_t)stream>>>(p);
            });
        return launched("taco_attention_step");
    });
}
