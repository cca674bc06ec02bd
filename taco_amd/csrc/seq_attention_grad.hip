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
        const int64_t blocks = (int64_t)p.n_tiles * p.heads, blocks_kv = (int64_t)p.n_tiles * p.kv_heads;
        const hipStream_t s = (hipStream_t)stream;
        auto run = [&](int64_t all, int threads, auto kernel) {
            in_launches(all, threads, [&](int32_t first, uint32_t grid) {
                p.first_block = first;
                kernel<<<grid, threads, 0, s>>>(p);
            });
        };
        if constexpr (short_gradients<T, DP>) {
            if (a->whole) {
                run(blocks_kv, 64, attention_short_grad_kernel<T, DP>);
                return launched("taco_attention_backward");
            }
        }
        if (a->tile_rows == 32) {
            run(blocks, 64, attention_dq_kernel<T, DP, 1>);
            run(blocks_kv, 64, attention_dkv_kernel<T, DP, 1>);
        } else {
            run(blocks, 256, attention_dq_kernel<T, DP, 4>);
            if constexpr (keys_in_lds<T, DP>) run(blocks_kv * p.parts, 512, attention_dkv_pair_kernel<T, DP>);
            else run(blocks_kv * p.parts, 256, attention_dkv_kernel<T, DP, 4>);
            if (p.parts > 1) run(blocks_kv, 256, attention_sum_kernel<T, DP>);
        }
        return launched("taco_attention_backward");
    });
}
