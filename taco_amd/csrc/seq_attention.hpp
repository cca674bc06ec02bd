// Attention inside packed sequences, forward and backward (include/taco_sequence.h taco_attention, taco_attention_backward).
#pragma once
#include "seq_core.hpp"
#include "../../include/taco_sequence.h"

namespace seq {

struct View {            // a tensor [tokens][heads][dim]: strides in bytes
    char *p;
    int64_t ts, hs;
};

struct AttentionParams {
    View q, k, v, o, d_o, d_q, d_k, d_v;
    float *lse, *delta;
    const taco_seq_tile *tiles, *key_tiles;
    int32_t n_tiles, heads, kv_heads, dim, causal;
    float scale;
};

// Workgroups go to the 8 XCDs in turn, each with an L2 of its own: with a multiple of 8 heads, neighbouring heads (one group's, which read the same keys and
// values) take the same XCD.  The tiles come longest first, all heads of a tile behind one another.
__device__ __forceinline__ void locate(int block, int heads, int &tile, int &head) {
    tile = block / heads;
    head = block % heads;
    if (heads % 8 == 0) head = (head % 8) * (heads / 8) + head / 8;
}

template <typename T> constexpr int waves_per_simd(int nw) { return nw == 4 && sizeof(T) == 2 ? 2 : 1; }

// Forward.  A wavefront owns 32 queries (columns of all its products), a workgroup NW of them and one K and one V tile of BN keys in LDS; the next tiles travel
// in registers meanwhile.  S^T = K Q^T leaves a query's scores in one lane and its other half: the softmax needs one exchange per tile, and P^T is the next
// product's operand as it stands (O^T = V^T P^T).  P is rounded to the inputs' type for that product (half a step, independent from key to key, so about
// as much as the output's own rounding); its sum stays float32.
// Keys run from the diagonal to the first one: the only tile with hidden keys of the sequence comes first, while O is zero, so if a hidden NaN got into O
// it shows there and the tile is done again without it.
template <typename T, int DP, int NW>
__global__ __launch_bounds__(64 * NW, waves_per_simd<T>(NW)) void attention_kernel(AttentionParams p) {
    typedef Tile<T, DP> tile;
    constexpr int BM = 32 * NW, BN = NW == 1 ? 32 : 64, NB = BN / 32, NS = DP / 16, DB = DP / 32, NT = 64 * NW;
    __shared__ __attribute__((aligned(16))) char lds_k[BN * tile::ROW], lds_v[BN * tile::ROW];
    int ti, head;
    locate(blockIdx.x, p.heads, ti, head);
    const taco_seq_tile w = p.tiles[ti];
    const int kvh = head / (p.heads / p.kv_heads), t = threadIdx.x, lane = t & 63, wave = t >> 6, h = lane >> 5, d = p.dim;
    const int first = w.first + 32 * wave, row = first + (lane & 31);
    const uint32_t rb = d * sizeof(T);
    const float c = p.scale * LOG2E;

    frag<T> qf[NS];
    {
        rsrc r = rows_of(p.q.p + (int64_t)(w.start + w.first) * p.q.ts + head * p.q.hs, min(BM, w.length - w.first), p.q.ts, rb);
#pragma unroll
        for (int s = 0; s < NS; ++s) qf[s] = rows_global<T>(r, p.q.ts, d, 32 * wave, s, lane);
    }
    const char *kp = p.k.p + (int64_t)w.start * p.k.ts + kvh * p.k.hs, *vp = p.v.p + (int64_t)w.start * p.v.ts + kvh * p.v.hs;
    Staged<T, DP, BN, NT> sk, sv;
    auto fetch = [&](int kt) {
        int n = min(BN, w.length - kt * BN);
        sk.load(rows_of(kp + (int64_t)kt * BN * p.k.ts, n, p.k.ts, rb), p.k.ts, d, t);
        sv.load(rows_of(vp + (int64_t)kt * BN * p.v.ts, n, p.v.ts, rb), p.v.ts, d, t);
    };

    f32x16 o[DB];
    clear(o);
    float m = -__builtin_inff(), l = 0.f;
    const int last = p.causal ? min(w.length, w.first + BM) - 1 : w.length - 1;
    const int limit = p.causal ? row : w.length - 1;       // the last key this lane's query sees
    int kt = last / BN;
    fetch(kt);
    for (; kt >= 0; --kt) {
        __syncthreads();
        sk.put(lds_k, t);
        sv.put(lds_v, t);
        __syncthreads();
        if (kt > 0) fetch(kt - 1);
        const int k0 = kt * BN;
        if (p.causal && k0 > first + 31) continue;      // (the wavefront's: all of the tile is hidden)
        f32x16 s[NB];
        clear(s);
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int x = 0; x < NS; ++x) s[n] = mma(tile::rows(lds_k, 32 * n, x, lane), qf[x], s[n]);
        const bool masked = k0 + BN - 1 > (p.causal ? first : w.length - 1);
        if (masked) {
#pragma unroll
            for (int n = 0; n < NB; ++n)
#pragma unroll
                for (int i = 0; i < 16; ++i) s[n][i] = k0 + 32 * n + row_of(i, h) <= limit ? s[n][i] : -__builtin_inff();
        }
        float mx = s[0][0];
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[n][i]);
        mx = fmaxf(mx, other_half(mx));
        const float mn = fmaxf(m, mx), mu = mn == -__builtin_inff() ? 0.f : mn * c;
        if (__any(mn > m)) {
            float a = exp2_(m * c - mu);
            l *= a;
#pragma unroll
            for (int b = 0; b < DB; ++b)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[b][i] *= a;
            m = mn;
        }
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                s[n][i] = exp2_(s[n][i] * c - mu);
                l += s[n][i];
            }
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                frag<T> pf = to_frag<T>(s[n], x);
#pragma unroll
                for (int b = 0; b < DB; ++b) o[b] = mma(tile::cols(lds_v, 32 * n + 16 * x, 32 * b, lane), pf, o[b]);
            }
        if (masked && p.causal && any_nan(o)) {
            clear(o);
#pragma unroll
            for (int n = 0; n < NB; ++n)
                accumulate_seen<T, DP>(lds_v, 32 * n, 0, s[n], [&](int r) { return k0 + 32 * n + r <= limit; }, o, lane);
        }
    }
    l += other_half(l);
    if (row < w.length) {
        store_row<T>((T *)(p.o.p + (int64_t)(w.start + row) * p.o.ts + head * p.o.hs), o, l == 0.f ? 0.f : 1.f / l, d, lane);
        if (h == 0) p.lse[(int64_t)(w.start + row) * p.heads + head] = m * p.scale + log2_(l) * LN2;
    }
}

// Backward, first launch: dQ, and delta = rowsum(dO O) for the second.  The forward kernel's shape: dS^T = P^T (dP^T - delta) from S^T = K Q^T and
// dP^T = V dO^T, then dQ^T = K^T dS^T, K read both ways from one LDS tile.  dQ and dK / dV take a kernel each, which computes S and dP twice (seven
// products for five), because neither then needs an atomic or a float32 copy of a gradient.
template <typename T, int DP, int NW>
__global__ __launch_bounds__(64 * NW, 1) void attention_dq_kernel(AttentionParams p) {
    typedef Tile<T, DP> tile;
    constexpr int BM = 32 * NW, BN = NW == 1 ? 32 : 64, NB = BN / 32, NS = DP / 16, DB = DP / 32, NT = 64 * NW;
    __shared__ __attribute__((aligned(16))) char lds_k[BN * tile::ROW], lds_v[BN * tile::ROW];
    int ti, head;
    locate(blockIdx.x, p.heads, ti, head);
    const taco_seq_tile w = p.tiles[ti];
    const int kvh = head / (p.heads / p.kv_heads), t = threadIdx.x, lane = t & 63, wave = t >> 6, h = lane >> 5, d = p.dim;
    const int first = w.first + 32 * wave, row = first + (lane & 31);
    const uint32_t rb = d * sizeof(T);
    const float c = p.scale * LOG2E;

    frag<T> qf[NS], gf[NS];
    float delta = 0.f;
    {
        const int64_t at = w.start + w.first;
        const int n = min(BM, w.length - w.first);
        rsrc rq = rows_of(p.q.p + at * p.q.ts + head * p.q.hs, n, p.q.ts, rb), rg = rows_of(p.d_o.p + at * p.d_o.ts + head * p.d_o.hs, n, p.d_o.ts, rb),
             ro = rows_of(p.o.p + at * p.o.ts + head * p.o.hs, n, p.o.ts, rb);
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            qf[s] = rows_global<T>(rq, p.q.ts, d, 32 * wave, s, lane);
            gf[s] = rows_global<T>(rg, p.d_o.ts, d, 32 * wave, s, lane);
            frag<T> of = rows_global<T>(ro, p.o.ts, d, 32 * wave, s, lane);
#pragma unroll
            for (int j = 0; j < 8; ++j) delta += (float)gf[s][j] * (float)of[j];
        }
        delta += other_half(delta);
    }
    float lse = 0.f;
    if (row < w.length) {
        const int64_t at = (int64_t)(w.start + row) * p.heads + head;
        lse = p.lse[at];
        if (h == 0) p.delta[at] = delta;
    }
    const float mu = lse == -__builtin_inff() ? __builtin_inff() : lse * LOG2E;      // (a row that attends to nothing: P = 0)
    const char *kp = p.k.p + (int64_t)w.start * p.k.ts + kvh * p.k.hs, *vp = p.v.p + (int64_t)w.start * p.v.ts + kvh * p.v.hs;
    Staged<T, DP, BN, NT> sk, sv;
    auto fetch = [&](int kt) {
        int n = min(BN, w.length - kt * BN);
        sk.load(rows_of(kp + (int64_t)kt * BN * p.k.ts, n, p.k.ts, rb), p.k.ts, d, t);
        sv.load(rows_of(vp + (int64_t)kt * BN * p.v.ts, n, p.v.ts, rb), p.v.ts, d, t);
    };

    f32x16 dq[DB];
    clear(dq);
    const int last = p.causal ? min(w.length, w.first + BM) - 1 : w.length - 1;
    const int limit = p.causal ? row : w.length - 1;
    int kt = last / BN;
    fetch(kt);
    for (; kt >= 0; --kt) {
        __syncthreads();
        sk.put(lds_k, t);
        sv.put(lds_v, t);
        __syncthreads();
        if (kt > 0) fetch(kt - 1);
        const int k0 = kt * BN;
        if (p.causal && k0 > first + 31) continue;
        const bool masked = k0 + BN - 1 > (p.causal ? first : w.length - 1);
        f32x16 ds[NB];
#pragma unroll
        for (int n = 0; n < NB; ++n) {
            f32x16 x[2];
            clear(x);
#pragma unroll
            for (int y = 0; y < NS; ++y) x[0] = mma(tile::rows(lds_k, 32 * n, y, lane), qf[y], x[0]);
#pragma unroll
            for (int y = 0; y < NS; ++y) x[1] = mma(tile::rows(lds_v, 32 * n, y, lane), gf[y], x[1]);
#pragma unroll
            for (int i = 0; i < 16; ++i) ds[n][i] = exp2_(x[0][i] * c - mu) * (x[1][i] - delta);
            if (masked) {
#pragma unroll
                for (int i = 0; i < 16; ++i) ds[n][i] = k0 + 32 * n + row_of(i, h) <= limit ? ds[n][i] : 0.f;
            }
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                frag<T> f = to_frag<T>(ds[n], y);
#pragma unroll
                for (int b = 0; b < DB; ++b) dq[b] = mma(tile::cols(lds_k, 32 * n + 16 * y, 32 * b, lane), f, dq[b]);
            }
        }
        if (masked && p.causal && any_nan(dq)) {
            clear(dq);
#pragma unroll
            for (int n = 0; n < NB; ++n)
                accumulate_seen<T, DP>(lds_k, 32 * n, 0, ds[n], [&](int r) { return k0 + 32 * n + r <= limit; }, dq, lane);
        }
    }
    if (row < w.length) store_row<T>((T *)(p.d_q.p + (int64_t)(w.start + row) * p.d_q.ts + head * p.d_q.hs), dq, p.scale, d, lane);
}

// Backward, second launch: dK and dV.  A wavefront owns 32 keys, whose K and V rows stay in registers as operands; Q and dO tiles of BQ queries pass through LDS,
// for every query head of the group in turn, so the gradients of a shared head are sums in registers.  S = Q K^T and dP = dO V^T have the keys in
// the lanes; P and dS are the operands of dV^T = dO^T P and dK^T = Q^T dS as they stand.
template <typename T, int DP, int NW>
__global__ __launch_bounds__(64 * NW, 1) void attention_dkv_kernel(AttentionParams p) {
    typedef Tile<T, DP> tile;
    constexpr int BK = 32 * NW, BQ = NW == 1 ? 32 : 64, NB = BQ / 32, NS = DP / 16, DB = DP / 32, NT = 64 * NW;
    __shared__ __attribute__((aligned(16))) char lds_q[BQ * tile::ROW], lds_g[BQ * tile::ROW];
    __shared__ __attribute__((aligned(16))) float lds_mu[BQ], lds_delta[BQ];
    int ti, kvh;
    locate(blockIdx.x, p.kv_heads, ti, kvh);
    const taco_seq_tile w = p.key_tiles[ti];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, h = lane >> 5, d = p.dim, G = p.heads / p.kv_heads;
    const int first = w.first + 32 * wave, key = first + (lane & 31);
    const uint32_t rb = d * sizeof(T);
    const float c = p.scale * LOG2E;

    frag<T> kf[NS], vf[NS];
    {
        const int64_t at = w.start + w.first;
        const int n = min(BK, w.length - w.first);
        rsrc rk = rows_of(p.k.p + at * p.k.ts + kvh * p.k.hs, n, p.k.ts, rb), rv = rows_of(p.v.p + at * p.v.ts + kvh * p.v.hs, n, p.v.ts, rb);
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            kf[s] = rows_global<T>(rk, p.k.ts, d, 32 * wave, s, lane);
            vf[s] = rows_global<T>(rv, p.v.ts, d, 32 * wave, s, lane);
        }
    }
    const int qt0 = p.causal ? w.first / BQ : 0, nq = (w.length - 1) / BQ + 1 - qt0;
    Staged<T, DP, BQ, NT> sq, sg;
    float mu_r = 0.f, delta_r = 0.f;
    auto fetch = [&](int it) {
        const int head = kvh * G + it / nq, q0 = (qt0 + it % nq) * BQ, n = min(BQ, w.length - q0);
        const int64_t at = w.start + q0;
        sq.load(rows_of(p.q.p + at * p.q.ts + head * p.q.hs, n, p.q.ts, rb), p.q.ts, d, t);
        sg.load(rows_of(p.d_o.p + at * p.d_o.ts + head * p.d_o.hs, n, p.d_o.ts, rb), p.d_o.ts, d, t);
        if (t < BQ) {
            float lse = t < n ? p.lse[(at + t) * p.heads + head] : -__builtin_inff();
            delta_r = t < n ? p.delta[(at + t) * p.heads + head] : 0.f;
            mu_r = lse == -__builtin_inff() ? __builtin_inff() : lse * LOG2E;
        }
    };

    f32x16 dk[DB], dv[DB];
    clear(dk);
    clear(dv);
    fetch(0);
    for (int it = 0; it < G * nq; ++it) {
        __syncthreads();
        sq.put(lds_q, t);
        sg.put(lds_g, t);
        if (t < BQ) {
            lds_mu[t] = mu_r;
            lds_delta[t] = delta_r;
        }
        __syncthreads();
        if (it + 1 < G * nq) fetch(it + 1);
        const int q0 = (qt0 + it % nq) * BQ;
#pragma unroll
        for (int n = 0; n < NB; ++n) {
            const int qb = q0 + 32 * n;
            if (p.causal && qb < first) continue;       // (all of the block comes before the wavefront's keys)
            f32x16 x[2];
            clear(x);
#pragma unroll
            for (int y = 0; y < NS; ++y) x[0] = mma(tile::rows(lds_q, 32 * n, y, lane), kf[y], x[0]);
#pragma unroll
            for (int y = 0; y < NS; ++y) x[1] = mma(tile::rows(lds_g, 32 * n, y, lane), vf[y], x[1]);
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                f32x4 mu = *(const f32x4 *)(lds_mu + 32 * n + row_of(i, h)), de = *(const f32x4 *)(lds_delta + 32 * n + row_of(i, h));
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    x[0][i + j] = exp2_(x[0][i + j] * c - mu[j]);
                    x[1][i + j] = x[0][i + j] * (x[1][i + j] - de[j]);
                }
            }
            const bool masked = p.causal && qb == first;
            bool apart = false;
            if (masked) {
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    bool seen = key <= qb + row_of(i, h);
                    x[0][i] = seen ? x[0][i] : 0.f;
                    x[1][i] = seen ? x[1][i] : 0.f;
                }
                apart = tile::any_nonfinite(lds_q, 32 * n, 32, lane) || tile::any_nonfinite(lds_g, 32 * n, 32, lane);
            }
            if (apart) {
                auto seen = [&](int r) { return key <= qb + r; };
                accumulate_seen<T, DP>(lds_g, 32 * n, 0, x[0], seen, dv, lane);
                accumulate_seen<T, DP>(lds_q, 32 * n, 0, x[1], seen, dk, lane);
            } else {
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    frag<T> pf = to_frag<T>(x[0], y), sf = to_frag<T>(x[1], y);
#pragma unroll
                    for (int b = 0; b < DB; ++b) dv[b] = mma(tile::cols(lds_g, 32 * n + 16 * y, 32 * b, lane), pf, dv[b]);
#pragma unroll
                    for (int b = 0; b < DB; ++b) dk[b] = mma(tile::cols(lds_q, 32 * n + 16 * y, 32 * b, lane), sf, dk[b]);
                }
            }
        }
    }
    if (key < w.length) {
        store_row<T>((T *)(p.d_k.p + (int64_t)(w.start + key) * p.d_k.ts + kvh * p.d_k.hs), dk, p.scale, d, lane);
        store_row<T>((T *)(p.d_v.p + (int64_t)(w.start + key) * p.d_v.ts + kvh * p.d_v.hs), dv, 1.f, d, lane);
    }
}

}  // namespace seq
