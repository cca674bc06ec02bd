// taco_attention (include/taco_sequence.h)
#include "seq_attention_host.hpp"

SEQ_API int taco_attention(const taco_attention_args *a, void *stream) {
    using namespace seq;
    AttentionParams p;
    if (int rc = attention_params(a, false, p)) return rc;
    if (p.n_tiles == 0) return TACO_SEQ_OK;
    return dispatch(a->dtype, a->dim, [&](auto type, auto dp) {
        typedef decltype(type) T;
        constexpr int DP = decltype(dp)::value;
        in_launches((int64_t)p.n_tiles * p.heads, 2 * a->tile_rows, [&](int32_t first, uint32_t grid) {
            p.first_block = first;
            if (a->tile_rows == 32) attention_kernel<T, DP, 1><<<grid, 64, 0, (hipStream_t)stream>>>(p);
            else attention_kernel<T, DP, 4><<<grid, 256, 0, (hipStream_t)stream>>>(p);
        });
        return launched("taco_attention");
    });
}
