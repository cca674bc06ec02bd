// Attention of one new token per row over a paged cache (include/taco_sequence.h taco_attention_step).
#pragma once
#include "seq_attention.hpp"
#include "seq_pages.hpp"

namespace seq {

struct StepParams {
    View q, o, k_new, v_new;            // byte strides
    char *k_pages, *v_pages;
    int64_t k_ps, k_ts, k_hs, v_ps, v_ts, v_hs;     // bytes
    const int32_t *table, *lengths;
    int64_t table_stride;
    int32_t rows, table_width, num_pages, page_size, heads, kv_heads, dim, blocks;      // blocks: of 32 query heads in a group
    int32_t piece, pieces, first_block;     // first_block: of this launch
    float scale;
    float *part_o, *part_ml;            // [rows][heads][pieces][DP], [rows][heads][pieces][2]
};

// One workgroup: a row, a key-value head, (up to) 32 query heads of its group as the columns of every product, and a piece of the keys; its NW wavefronts
// take tiles of 32 keys in turn, each with an LDS tile of its own (no barrier in the loop) that holds K, then V.  The cache is read once, in whole rows,
// 16 bytes a lane; the next K (V) tile is on its way in registers while this one is used, its page numbers one tile further ahead.
// Bound by HBM: 64 rows of up to 8 192 tokens, 32 heads of 128 over 8, bf16: 243 us, 4.8 TB/s (a copy of 2 GiB: 4.7); 4 rows of 65 536: 220 us, 4.9 TB/s.
// The new token is read from the call's own k and v; the one workgroup whose piece holds it writes it into the cache, which no other reads there.
template <typename T, int DP, int NW>
__global__ __launch_bounds__(64 * NW, sizeof(T) == 2 ? 2 : 1) void attention_step_kernel(StepParams p) {
    typedef Tile<T, DP> tile;
    constexpr int NS = DP / 16, DB = DP / 32, N = 32 * tile::NC / 64;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, h = lane >> 5, d = p.dim;
    const int block = p.first_block + blockIdx.x, blk = block % p.blocks, kvh = block / p.blocks % p.kv_heads, b = block / p.blocks / p.kv_heads;
    const int G = p.heads / p.kv_heads, g0 = 32 * blk, cols = min(32, G - g0), head0 = kvh * G + g0;
    const bool joins = p.k_new.p != nullptr;
    const int len = p.lengths[b], keys = keys_of(len, p.table_width, p.page_size, joins);
    const int64_t from = (int64_t)blockIdx.y * p.piece;         // (a table may have room for more than 2^31 tokens)
    if (blockIdx.y > 0 && from >= keys) return;
    const int begin = (int)from, end = (int)(from + p.piece < keys ? from + p.piece : max(keys, 0));
    const int32_t *table = p.table + b * p.table_stride;
    char *mine = lds + wave * 32 * tile::ROW;
    const float c = p.scale * LOG2E;
    const uint32_t rb = d * sizeof(T);

    frag<T> qf[NS];
    {
        rsrc r = rows_of(p.q.p + b * p.q.ts + head0 * p.q.hs, cols, p.q.hs, rb);
#pragma unroll
        for (int s = 0; s < NS; ++s) qf[s] = rows_global<T>(r, p.q.hs, d, 0, s, lane);
    }
    const char *kc = p.k_pages + kvh * p.k_hs, *vc = p.v_pages + kvh * p.v_hs;
    const char *kn = p.k_new.p + b * p.k_new.ts + kvh * p.k_new.hs, *vn = p.v_new.p + b * p.v_new.ts + kvh * p.v_new.hs;
    bool bad = keys < 0;
    // lane r (and r + 32) knows the place of key t0 + r
    auto look = [&](int t0) {
        const int token = t0 + (lane & 31);
        Place at{0, 0, false};
        if (token < end) at = place_of(table, token, p.page_size, p.num_pages);
        return at;
    };
    u32x4 kx[N], vx[N];
    auto fetch = [&](u32x4 (&x)[N], const char *cache, int64_t ps, int64_t ts, const char *fresh, Place at, int t0) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int e = i * 64 + lane, row = e / tile::NC, ch = e % tile::NC, token = t0 + row;
            const Place pl{__shfl(at.page, row), __shfl(at.slot, row), false};
            const bool in = token < end && ch * tile::CE < d;
            const char *src = joins && token == len ? fresh : cache + element_of(pl, ps, ts);       // (byte strides)
            const u32x4 y = *(const u32x4 *)(src + (ch * tile::CE < d ? ch * 16 : 0));
            x[i] = in ? y : u32x4{0, 0, 0, 0};
        }
    };
    auto put = [&](const u32x4 (&x)[N]) {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int e = i * 64 + lane;
            tile::put(mine, e / tile::NC, e % tile::NC, x[i]);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    };

    f32x16 o[DB];
    clear(o);
    float m = -__builtin_inff(), mu = -__builtin_inff(), l = 0.f;        // the running maximum, as it is and in the exponent's unit, and the sum
    int t0 = begin + 32 * wave;
    Place now{0, 0, false}, next{0, 0, false};
    if (t0 < end) {
        now = look(t0);
        bad |= now.bad;
        fetch(kx, kc, p.k_ps, p.k_ts, kn, now, t0);
        fetch(vx, vc, p.v_ps, p.v_ts, vn, now, t0);
        next = look(t0 + 32 * NW);
    }
    for (; t0 < end; t0 += 32 * NW) {
        const int t1 = t0 + 32 * NW;
        put(kx);
        f32x16 s[1];
        clear(s);
#pragma unroll
        for (int x = 0; x < NS; ++x) s[0] = mma(tile::rows(mine, 0, x, lane), qf[x], s[0]);
        bad |= next.bad;
        if (t1 < end) fetch(kx, kc, p.k_ps, p.k_ts, kn, next, t1);
        if (t0 + 32 > end) {
#pragma unroll
            for (int i = 0; i < 16; ++i) s[0][i] = t0 + row_of(i, h) < end ? s[0][i] : -__builtin_inff();
        }
        float mx = s[0][0];
#pragma unroll
        for (int i = 1; i < 16; ++i) mx = fmaxf(mx, s[0][i]);
        mx = fmaxf(mx, other_half(mx));
        if (__any(mx > m)) {
            m = fmaxf(m, mx);
            const float next = rounded(m * c), a = next == mu ? 1.f : exp2_(mu - next);
            mu = next;
            l *= a;
#pragma unroll
            for (int x = 0; x < DB; ++x) o[x] *= a;
        }
        const float sub = mu == -__builtin_inff() ? 0.f : mu;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            s[0][i] = exp2_(s[0][i] * c - sub);
            l += s[0][i];
        }
        put(vx);
        if (t1 < end) {
            fetch(vx, vc, p.v_ps, p.v_ts, vn, next, t1);
            next = look(t1 + 32 * NW);
        }
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            frag<T> pf = to_frag<T>(s[0] * WEIGHT<T>, x);
#pragma unroll
            for (int y = 0; y < DB; ++y) o[y] = mma(tile::cols(mine, 16 * x, 32 * y, lane), pf, o[y]);
        }
    }
    l += other_half(l);
    if (__any(bad)) l = __builtin_nanf("");

    // join the wavefronts: [NW][cols][DP] sums, then [NW][cols][2] maxima and weights
    float *so = (float *)lds, *sm = so + NW * cols * DP;
    __syncthreads();
    const int col = lane & 31;
    if (col < cols) {
#pragma unroll
        for (int x = 0; x < DB; ++x)
#pragma unroll
            for (int i = 0; i < 16; i += 4)
                *(f32x4 *)(so + (wave * cols + col) * DP + 32 * x + row_of(i, h)) = f32x4{o[x][i], o[x][i + 1], o[x][i + 2], o[x][i + 3]};
        if (h == 0) {
            sm[(wave * cols + col) * 2] = mu;
            sm[(wave * cols + col) * 2 + 1] = l;
        }
    }
    __syncthreads();
    for (int e = t; e < cols * (DP / 4); e += 64 * NW) {
        const int g = e / (DP / 4), x = e % (DP / 4) * 4;
        float M = -__builtin_inff(), L = 0.f;
#pragma unroll
        for (int y = 0; y < NW; ++y) M = fmaxf(M, sm[(y * cols + g) * 2]);
        f32x4 a{0, 0, 0, 0};
#pragma unroll
        for (int y = 0; y < NW; ++y) {
            const float my = sm[(y * cols + g) * 2], f = my == -__builtin_inff() ? 0.f : exp2_(my - M);
            L += sm[(y * cols + g) * 2 + 1] * f;
            a += *(const f32x4 *)(so + (y * cols + g) * DP + x) * f;
        }
        if (p.pieces == 1) {
            const float f = L == 0.f ? 0.f : 1.f / (L * WEIGHT<T>);
            if (x < d) store4((T *)(p.o.p + b * p.o.ts + (head0 + g) * p.o.hs) + x, a[0] * f, a[1] * f, a[2] * f, a[3] * f);
        } else {
            const int64_t at = ((int64_t)b * p.heads + head0 + g) * p.pieces + blockIdx.y;
            *(f32x4 *)(p.part_o + at * DP + x) = a;
            if (x == 0) {
                p.part_ml[at * 2] = M;
                p.part_ml[at * 2 + 1] = L;
            }
        }
    }
    if (joins && blk == 0 && keys > 0 && len >= begin && len < end) {
        const Place at = place_of(table, len, p.page_size, p.num_pages);
        if (!at.bad && t < 2 * tile::NC) {
            const int ch = t % tile::NC;
            if (ch * tile::CE < d) {
                if (t < tile::NC) *(u32x4 *)(p.k_pages + kvh * p.k_hs + element_of(at, p.k_ps, p.k_ts) + ch * 16) = *(const u32x4 *)(kn + ch * 16);
                else *(u32x4 *)(p.v_pages + kvh * p.v_hs + element_of(at, p.v_ps, p.v_ts) + ch * 16) = *(const u32x4 *)(vn + ch * 16);
            }
        }
    }
}

// The pieces of a row and head joined: one wavefront, DP / 4 lanes across the dimension (32 for 96), the other lanes take other pieces.
template <typename T, int DP>
__global__ __launch_bounds__(64) void attention_join_kernel(StepParams p) {
    constexpr int W = DP == 96 ? 32 : DP / 4, S = 64 / W;
    const int block = p.first_block + blockIdx.x, b = block / p.heads, head = block % p.heads, lane = threadIdx.x, x = lane % W * 4, s = lane / W;
    const int n = pieces_of(keys_of(p.lengths[b], p.table_width, p.page_size, p.k_new.p != nullptr), p.piece);
    const int64_t at = (int64_t)block * p.pieces;
    float M = -__builtin_inff();
    for (int i = lane; i < n; i += 64) M = fmaxf(M, p.part_ml[(at + i) * 2]);
#pragma unroll
    for (int i = 32; i > 0; i >>= 1) M = fmaxf(M, __shfl_xor(M, i));
    float L = 0.f;
    f32x4 a{0, 0, 0, 0};
    for (int i = s; i < n; i += S) {
        const float m = p.part_ml[(at + i) * 2], f = m == -__builtin_inff() ? 0.f : exp2_(m - M);
        L += p.part_ml[(at + i) * 2 + 1] * f;
        if (x < DP) a += *(const f32x4 *)(p.part_o + (at + i) * DP + x) * f;
    }
#pragma unroll
    for (int i = W; i < 64; i <<= 1) {
        L += __shfl_xor(L, i);
#pragma unroll
        for (int j = 0; j < 4; ++j) a[j] += __shfl_xor(a[j], i);
    }
    const float f = L == 0.f ? 0.f : 1.f / (L * WEIGHT<T>);
    if (s == 0 && x < p.dim) store4((T *)(p.o.p + b * p.o.ts + head * p.o.hs) + x, a[0] * f, a[1] * f, a[2] * f, a[3] * f);
}

}  // namespace seq
