// What taco_attention and taco_attention_backward check and hand on.
#pragma once
#include "seq_host.hpp"

namespace seq {

inline int attention_params(const taco_attention_args *a, bool backward, AttentionParams &p) {
    SEQ_NEED(a, "args: null");
    if (int rc = check_dims(a->heads, a->kv_heads, a->dim, a->dtype)) return rc;
    SEQ_NEED(a->scale > 0.f && a->scale < __builtin_inff(), "scale %g: positive and finite", (double)a->scale);
    SEQ_NEED(a->tile_rows == 32 || a->tile_rows == 128, "tile_rows %d: 32 or 128", a->tile_rows);
    SEQ_NEED(!a->whole || a->tile_rows == 32, "whole sequences: tile_rows 32, not %d", a->tile_rows);
    SEQ_NEED(!backward || !a->whole || a->dtype != TACO_SEQ_F32 || a->dim <= 96, "whole sequences of float32 rows of %d: at most 96", a->dim);
    SEQ_NEED(a->n_tiles >= 0 && (int64_t)a->n_tiles * a->heads < (int64_t)1 << 31, "%d tiles of %d heads: fewer than 2^31 in all", a->n_tiles, a->heads);
    p = AttentionParams{};
    p.n_tiles = a->n_tiles;
    if (a->n_tiles == 0) return TACO_SEQ_OK;
    const struct { const char *name; const taco_seq_tensor *t; View *v; } all[] = {
        {"q", &a->q, &p.q}, {"k", &a->k, &p.k}, {"v", &a->v, &p.v}, {"o", &a->o, &p.o},
        {"d_o", &a->d_o, &p.d_o}, {"d_q", &a->d_q, &p.d_q}, {"d_k", &a->d_k, &p.d_k}, {"d_v", &a->d_v, &p.d_v}};
    for (int i = 0; i < (backward ? 8 : 4); ++i) {
        if (int rc = check_tensor(all[i].name, *all[i].t, a->dim, a->dtype)) return rc;
        *all[i].v = view(*all[i].t, a->dtype);
    }
    SEQ_NEED(a->lse && a->tiles, "lse or tiles: null");
    SEQ_NEED(!backward || a->delta, "delta: null");
    p.parts = 1;
    if (backward && a->tile_rows == 128) {
        SEQ_NEED(a->parts >= 1 && (a->heads / a->kv_heads) % a->parts == 0, "%d parts of a group of %d query heads", a->parts, a->heads / a->kv_heads);
        SEQ_NEED(a->parts == 1 || (a->partial && (uintptr_t)a->partial % 16 == 0), "partial: null or not 16-byte aligned");
        SEQ_NEED((int64_t)a->n_tiles * a->kv_heads * a->parts < (int64_t)1 << 31, "%d tiles of %d heads in %d parts: fewer than 2^31 in all", a->n_tiles, a->kv_heads, a->parts);
        p.parts = a->parts;
        p.partial = a->partial;
    }
    p.lse = a->lse;
    p.delta = a->delta;
    p.tiles = a->tiles;
    p.key_tiles = a->key_tiles ? a->key_tiles : a->tiles;
    p.heads = a->heads;
    p.kv_heads = a->kv_heads;
    p.dim = a->dim;
    p.causal = a->causal != 0;
    p.scale = a->scale;
    return TACO_SEQ_OK;
}

}  // namespace seq
