// taco_attention_backward (include/taco_sequence.h)
#include "seq_attention_host.hpp"

SEQ_API int taco_attention_backward(const taco_attention_args *a, void *stream) {
    using namespace seq;
    AttentionParams p;
    if (int rc = attention_params(a, true, p)) return rc;
    if (p.n_tiles == 0) return TACO_SEQ_OK;
    return dispatch(a->dtype, a->dim, [&](auto type, auto dp) {
        typedef decltype(type) T;
        constexpr int DP = decltype(dp)::value;
        const dim3 grid((unsigned)(p.n_tiles * p.heads)), grid_kv((unsigned)(p.n_tiles * p.kv_heads));
        const hipStream_t s = (hipStream_t)stream;
        if constexpr (short_gradients<T, DP>) {
            if (a->whole) {
                attention_short_grad_kernel<T, DP><<<grid_kv, 64, 0, s>>>(p);
                return launched("taco_attention_backward");
            }
        }
        if (a->tile_rows == 32) {
            attention_dq_kernel<T, DP, 1><<<grid, 64, 0, s>>>(p);
            attention_dkv_kernel<T, DP, 1><<<grid_kv, 64, 0, s>>>(p);
        } else {
            attention_dq_kernel<T, DP, 4><<<grid, 256, 0, s>>>(p);
            if constexpr (keys_in_lds<T, DP>) attention_dkv_pair_kernel<T, DP><<<grid_kv.x * p.parts, 512, 0, s>>>(p);
            else attention_dkv_kernel<T, DP, 4><<<grid_kv.x * p.parts, 256, 0, s>>>(p);
            if (p.parts > 1) attention_sum_kernel<T, DP><<<grid_kv, 256, 0, s>>>(p);
        }
        return launched("taco_attention_backward");
    });
}
