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
    int32_t n_tiles, heads, kv_heads, dim, causal, parts, first_block;      // first_block: of this launch
    float scale;
    float *partial;          // [n_tiles][128][kv_heads][parts][2][DP], by the key tiles' order
};

// Workgroups go to the 8 XCDs in turn, each with an L2 of its own: with a multiple of 8 heads, neighbouring heads (one group's, which read the same keys and
// values) take the same XCD.  The tiles come longest first, all heads of a tile behind one another.
__device__ __forceinline__ void locate(int block, int heads, int &tile, int &head) {
    tile = block / heads;
    head = block % heads;
    if (heads % 8 == 0) head = (head % 8) * (heads / 8) + head / 8;
}

// Wavefronts per SIMD that the registers are cut for: as many as spill nothing, or little.  Nothing else hides the latency of loads and of the chain of products, least
// of all where a sequence is one tile.  Cut for two, these spill at rows of 128 in 16 bits: the forward 15 to 17 registers, dQ 58, dK / dV 9 to 12.  Cut for one: float32
// dQ of 128 in 32-row tiles 104, the forward there 29, the short gradients of 96 29; fp16's short gradients of 128 12, dK / dV of 64 2.
template <typename T, int DP, int NW> constexpr int waves_forward = sizeof(T) == 4 ? (DP == 32 ? 2 : 1) : DP == 32 ? 4 : DP == 64 || NW == 4 ? 2 : 1;
template <typename T, int DP, int NW> constexpr int waves_dq = sizeof(T) == 4 ? (DP == 32 ? 2 : 1) : DP <= 64 || NW == 4 ? 2 : 1;
template <typename T, int DP> constexpr int waves_dkv = sizeof(T) == 4 ? (DP == 32 ? 2 : 1) : DP <= 64 ? 2 : 1;
// The next tiles travel in registers while these are used, except where that would spill: wide float32 rows hold half the registers as operands already.
template <typename T, int DP> constexpr bool ahead = !(sizeof(T) == 4 && DP >= 96);

// (and there the compiler must not ask LDS for many operands at once either)
template <typename T, int DP> __device__ __forceinline__ void in_order() {
    if (!ahead<T, DP>) __builtin_amdgcn_sched_barrier(0);
}

// acc += X w for a product whose tile X of 32 rows is read by columns: one step of a running sum in acc.  float32 sums each tile apart first: the sum over a long
// sequence then has a rounding per tile in it, not per pair of rows (its error is the float32 result's own; the 16-bit types' roundings are larger).
template <typename T, int DP> __device__ __forceinline__ void add_columns(const char *lds, int row0, const f32x16 &w, f32x16 (&acc)[DP / 32], int lane, float factor = 1.f) {
    frag<T> f[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) f[x] = to_frag<T>(w * factor, x);
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int b = 0; b < DP / 32; ++b) {
            f32x16 y[1];
            clear(y);
#pragma unroll
            for (int x = 0; x < 2; ++x) y[0] = mma(Tile<T, DP>::cols(lds, row0 + 16 * x, 32 * b, lane), f[x], y[0]);
            acc[b] += y[0];
            in_order<T, DP>();
        }
    } else {
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int b = 0; b < DP / 32; ++b) acc[b] = mma(Tile<T, DP>::cols(lds, row0 + 16 * x, 32 * b, lane), f[x], acc[b]);
    }
}

// Forward.  A wavefront owns 32 queries (columns of all its products), a workgroup NW of them and one K and one V tile of BN keys in LDS; the next tiles travel
// in registers meanwhile.  S^T = K Q^T leaves a query's scores in one lane and its other half: the softmax needs one exchange per tile, and P^T is the next
// product's operand as it stands (O^T = V^T P^T).  P is rounded to the inputs' type for that product (half a step, independent from key to key, so about
// as much as the output's own rounding; in float16 lifted by 2^15, or one key that draws nearly all the weight and has no value would leave the others' below the
// type's normal range); its sum stays float32.
// Keys run from the diagonal to the first one.  The tiles that hide keys come first, in a loop of their own, and the others run without a mask.
// Bound by LDS (32 KB a wavefront and tile for 1 024 clocks of matrix work) and the exponentials, which only the second wavefront of the SIMD hides.  One
// sequence of 16 384 tokens, 16 heads of 128 over 4, bf16: 1.10 to 1.13 ms, 975 to 1 000 TFLOP/s (a library product of 8 192^3: 1 138); with the masks and the test for
// NaN in the one loop, and what that spilled, 9.3 ms.  24 sequences of up to 2 048: 0.25 ms, 627: tiles of 12 turns on average, whose first loads and
// half-hidden tiles nothing covers.  fp16, with its lift: 1.28 ms for the one of 16 384 (1.26 without).
template <typename T, int DP, int NW>
__global__ __launch_bounds__(64 * NW, (waves_forward<T, DP, NW>)) void attention_kernel(AttentionParams p) {
    typedef Tile<T, DP> tile;
    constexpr int BM = 32 * NW, BN = NW == 1 ? 32 : 64, NB = BN / 32, NS = DP / 16, DB = DP / 32, NT = 64 * NW;
    __shared__ __attribute__((aligned(16))) char lds_k[BN * tile::ROW], lds_v[BN * tile::ROW];
    __shared__ int nonfinite;
    int ti, head;
    locate(p.first_block + blockIdx.x, p.heads, ti, head);
    const taco_seq_tile w = p.tiles[ti];
    const int kvh = head / (p.heads / p.kv_heads), t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), h = lane >> 5, d = p.dim;
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
        const int n = min(BN, w.length - kt * BN);
        sk.load(rows_of(kp + (int64_t)kt * BN * p.k.ts, n, p.k.ts, rb), p.k.ts, d, t);
        sv.load(rows_of(vp + (int64_t)kt * BN * p.v.ts, n, p.v.ts, rb), p.v.ts, d, t);
    };

    f32x16 o[DB];
    clear(o);
    float m = -__builtin_inff(), mu = -__builtin_inff(), l = 0.f;        // the running maximum, as it is and in the exponent's unit, and the sum
    const int last = p.causal ? min(w.length, w.first + BM) - 1 : w.length - 1;
    const int limit = p.causal ? row : w.length - 1;       // the last key this lane's query sees
    auto scores = [&](f32x16 (&s)[NB]) {
        clear(s);
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int x = 0; x < NS; ++x) {
                s[n] = mma(tile::rows(lds_k, 32 * n, x, lane), qf[x], s[n]);
                in_order<T, DP>();
            }
    };
    auto softmax = [&](f32x16 (&s)[NB]) {
        float mx = s[0][0];
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[n][i]);
        mx = fmaxf(mx, other_half(mx));
        if (__any(mx > m)) {
            m = fmaxf(m, mx);
            const float next = rounded(m * c), a = next == mu ? 1.f : exp2_(mu - next);
            mu = next;
            l *= a;
#pragma unroll
            for (int b = 0; b < DB; ++b) o[b] *= a;
        }
        const float sub = mu == -__builtin_inff() ? 0.f : mu;
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                s[n][i] = exp2_(s[n][i] * c - sub);
                sum[i % 4] += s[n][i];
            }
        l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
    };

    int kt = last / BN;
    // tiles from here up hide keys of the sequence from some query of the workgroup (causal), or hold rows behind its end
    const int whole = p.causal ? w.first / BN : w.length / BN;
    if (ahead<T, DP>) fetch(kt);
    if (t == 0) nonfinite = 0;
    for (; kt >= whole; --kt) {
        __syncthreads();
        if (!ahead<T, DP>) fetch(kt);
        const bool bad = p.causal && __any(sv.any_nonfinite());
        if (bad) {
            sv.nonfinite_to_zero();
            if (lane == 0) nonfinite = kt + 1;
        }
        sk.put(lds_k, t);
        sv.put(lds_v, t);
        __syncthreads();
        if (ahead<T, DP> && kt > 0) fetch(kt - 1);
        const int k0 = kt * BN;
        if (p.causal && k0 > first + 31) continue;      // (the wavefront's: all of the tile is hidden)
        f32x16 s[NB];
        scores(s);
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int i = 0; i < 16; ++i) s[n][i] = k0 + 32 * n + row_of(i, h) <= limit ? s[n][i] : -__builtin_inff();
        softmax(s);
#pragma unroll
        for (int n = 0; n < NB; ++n) add_columns<T, DP>(lds_v, 32 * n, s[n], o, lane, WEIGHT<T>);
        if (nonfinite == kt + 1) {
            for (int b = 0; b < DP; b += 64) {
                int plus, minus;
                const int n = min(BN, w.length - k0);
                first_nonfinite<T>(vp + (int64_t)k0 * p.v.ts, p.v.ts, b + lane < d ? n : 0, b + lane < d ? b + lane : 0, plus, minus);
                if (b + lane >= d) plus = minus = n;
                plus += k0;
                minus += k0;
                const int end = k0 + n;
#pragma unroll
                for (int x = 0; x < DB; ++x)
                    if (32 * x >= b && 32 * x < b + 64)
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            const int from = 32 * x - b + row_of(i, h), fp = __shfl(plus, from), fm = __shfl(minus, from);
                            o[x][i] += (fp < end && fp <= limit ? __builtin_inff() : 0.f) + (fm < end && fm <= limit ? -__builtin_inff() : 0.f);
                        }
            }
        }
    }
    for (; kt >= 0; --kt) {
        __syncthreads();
        if (!ahead<T, DP>) fetch(kt);
        sk.put(lds_k, t);
        sv.put(lds_v, t);
        __syncthreads();
        if (ahead<T, DP> && kt > 0) fetch(kt - 1);
        f32x16 s[NB];
        scores(s);
        softmax(s);
#pragma unroll
        for (int n = 0; n < NB; ++n) add_columns<T, DP>(lds_v, 32 * n, s[n], o, lane, WEIGHT<T>);
    }
    l += other_half(l);
    if (row < w.length) {
        store_row<T>((T *)(p.o.p + (int64_t)(w.start + row) * p.o.ts + head * p.o.hs), o, l == 0.f ? 0.f : 1.f / (l * WEIGHT<T>), d, lane);
        if (h == 0) p.lse[(int64_t)(w.start + row) * p.heads + head] = (mu + log2_(l)) * LN2;
    }
}

// Backward, first launch: dQ, and delta = scale rowsum(dO O) for the second.  dP, delta and so dS carry the scale from the start.  In float16 dS, a product of a weight (of
// 1 / length), an upstream gradient and the scale, is lifted by a power of two for each query (here) or key (dK) before it is rounded: without, an upstream
// gradient of a thousandth over 2 048 tokens left dq and dk 25 times as far off as a value rounded once.  The forward kernel's shape: dS^T = P^T (dP^T - delta) from S^T = K Q^T and
// dP^T = V dO^T, then dQ^T = K^T dS^T, K read both ways from one LDS tile.  dQ and dK / dV take a kernel each, which computes S and dP twice (seven
// products for five), because neither then needs an atomic or a float32 copy of a gradient.
// A query that sees few keys has gradients that are small differences of dP and delta, and o as it was rounded would set their error.  Where all its keys
// lie in one tile, delta is the sum of P dP over that tile instead, in float32 (from o, dq and dk of sequences of two tokens were 2.3 roundings off, now 1.4).
// Six sequences of up to 4 096, 16 heads of 128 over 4, bf16: 0.41 ms, 740 TFLOP/s of its three products (fp16 0.45); bound as the forward, and by what it spills
// (243 MB written, 65 of them dQ).
template <typename T, int DP, int NW>
__global__ __launch_bounds__(64 * NW, (waves_dq<T, DP, NW>)) void attention_dq_kernel(AttentionParams p) {
    typedef Tile<T, DP> tile;
    constexpr int BM = 32 * NW, BN = NW == 1 ? 32 : 64, NB = BN / 32, NS = DP / 16, DB = DP / 32, NT = 64 * NW;
    __shared__ __attribute__((aligned(16))) char lds_k[BN * tile::ROW], lds_v[BN * tile::ROW];
    __shared__ int nonfinite;       // the first key of the tile with something not finite in it
    int ti, head;
    locate(p.first_block + blockIdx.x, p.heads, ti, head);
    const taco_seq_tile w = p.tiles[ti];
    const int kvh = head / (p.heads / p.kv_heads), t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), h = lane >> 5, d = p.dim;
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
        delta = (delta + other_half(delta)) * p.scale;
    }
    const int64_t at = (int64_t)(w.start + row) * p.heads + head;
    const float lse = row < w.length ? p.lse[at] : 0.f;
    const float mu = lse == -__builtin_inff() ? __builtin_inff() : lse * LOG2E;      // (a row that attends to nothing: P = 0)
    const char *kp = p.k.p + (int64_t)w.start * p.k.ts + kvh * p.k.hs, *vp = p.v.p + (int64_t)w.start * p.v.ts + kvh * p.v.hs;
    Staged<T, DP, BN, NT> sk, sv;
    auto fetch = [&](int kt) {
        const int n = min(BN, w.length - kt * BN), t_ = afresh(t);
        sk.load(rows_of(kp + (int64_t)kt * BN * p.k.ts, n, p.k.ts, rb), p.k.ts, d, t_);
        sv.load(rows_of(vp + (int64_t)kt * BN * p.v.ts, n, p.v.ts, rb), p.v.ts, d, t_);
    };

    f32x16 dq[DB];
    clear(dq);
    float f = lift_start<T>;
    const int last = p.causal ? min(w.length, w.first + BM) - 1 : w.length - 1;
    const int limit = p.causal ? row : w.length - 1;
    // P and scale dP of 32 keys
    auto weights = [&](int n, f32x16 &pr, f32x16 &dp) {
        f32x16 x[2];
        clear(x);
        mma_rows<T>([&](int y) { return tile::rows(lds_k, 32 * n, y, lane); }, qf, x[0]);
        mma_rows<T>([&](int y) { return tile::rows(lds_v, 32 * n, y, lane); }, gf, x[1]);
#pragma unroll
        for (int i = 0; i < 16; ++i) pr[i] = exp2_(x[0][i] * c - mu);
        dp = x[1] * p.scale;
    };
    int kt = last / BN;
    const int whole = p.causal ? w.first / BN : w.length / BN;
    if (ahead<T, DP>) fetch(kt);
    if (t == 0) nonfinite = BN;
    for (; kt >= whole; --kt) {
        __syncthreads();
        if (!ahead<T, DP>) fetch(kt);
        if (p.causal && __any(sk.any_nonfinite())) {
            int r = BN;
#pragma unroll
            for (int i = Staged<T, DP, BN, NT>::N - 1; i >= 0; --i)
                if (sk.chunk_nonfinite(i)) r = (i * NT + t) / tile::NC;
            sk.nonfinite_to_zero();
            atomicMin(&nonfinite, r);
        }
        sk.put(lds_k, t);
        sv.put(lds_v, t);
        __syncthreads();
        const int seen_bad = nonfinite;
        if (ahead<T, DP> && kt > 0) fetch(kt - 1);
        const int k0 = kt * BN;
        if (!(p.causal && k0 > first + 31)) {      // (else: all of the tile is hidden from the wavefront)
            f32x16 pr, ds;
            if (k0 == 0) {
                float x = 0.f;
#pragma unroll 1
                for (int n = 0; n < NB; ++n) {
                    weights(n, pr, ds);
#pragma unroll
                    for (int i = 0; i < 16; ++i) x += k0 + 32 * n + row_of(i, h) <= limit ? pr[i] * ds[i] : 0.f;
                }
                delta = limit < BN ? x + other_half(x) : delta;
            }
#pragma unroll 1
            for (int n = 0; n < NB; ++n) {
                weights(n, pr, ds);
#pragma unroll
                for (int i = 0; i < 16; ++i) ds[i] = k0 + 32 * n + row_of(i, h) <= limit ? pr[i] * (ds[i] - delta) : 0.f;
                lift<T>(ds, f, dq);
                add_columns<T, DP>(lds_k, 32 * n, ds, dq, lane);
            }
            if (k0 + seen_bad <= limit && seen_bad < BN) {      // (a key that is not finite: its weight is not either)
#pragma unroll
                for (int b = 0; b < DB; ++b) dq[b] += __builtin_nanf("");
            }
        }
        if (p.causal) {
            __syncthreads();
            if (t == 0) nonfinite = BN;
        }
    }
    for (; kt >= 0; --kt) {
        __syncthreads();
        if (!ahead<T, DP>) fetch(kt);
        sk.put(lds_k, t);
        sv.put(lds_v, t);
        __syncthreads();
        if (ahead<T, DP> && kt > 0) fetch(kt - 1);
#pragma unroll
        for (int n = 0; n < NB; ++n) {
            f32x16 pr, ds;
            weights(n, pr, ds);
#pragma unroll
            for (int i = 0; i < 16; ++i) ds[i] = pr[i] * (ds[i] - delta);
            lift<T>(ds, f, dq);
            add_columns<T, DP>(lds_k, 32 * n, ds, dq, lane);
        }
    }
    if (row < w.length) {
        store_row<T>((T *)(p.d_q.p + (int64_t)(w.start + row) * p.d_q.ts + head * p.d_q.hs), dq, inverse(f), d, lane);
        if (h == 0) p.delta[at] = delta;
    }
}

// Backward, second launch: dK and dV.  A wavefront owns 32 keys, whose K and V rows stay in registers as operands; Q and dO tiles of BQ queries pass through LDS,
// for every query head of the group in turn, so the gradients of a shared head are sums in registers.  S = Q K^T and dP = dO V^T have the keys in
// the lanes; P and dS are the operands of dV^T = dO^T P and dK^T = Q^T dS as they stand.
// Where the longest sequence's first keys would outlast everything else (all queries of all heads of the group behind one another), the group's heads are
// shared out to `parts` workgroups, whose float32 sums a third launch adds up, always in the same order (six sequences of up to 4 096: 0.84 -> 0.70 ms + 0.03).
// Rows of 96 and 128 float32 leave some 150 registers beside the operands and sums: there a tile is 32 queries, Q and dO come in the same registers one after
// the other, and addresses are computed again for each tile.  100 sequences of up to 200, 8 heads of 128 over 2: 0.20 ms; with tiles of 64 and both at once,
// which spilled 180 registers, 0.36.
template <typename T, int DP, int NW>
__global__ __launch_bounds__(64 * NW, (waves_dkv<T, DP>)) void attention_dkv_kernel(AttentionParams p) {
    typedef Tile<T, DP> tile;
    constexpr int BK = 32 * NW, BQ = NW == 1 || !ahead<T, DP> ? 32 : 64, NB = BQ / 32, NS = DP / 16, DB = DP / 32, NT = 64 * NW;
    __shared__ __attribute__((aligned(16))) char lds_q[BQ * tile::ROW], lds_g[BQ * tile::ROW];
    __shared__ __attribute__((aligned(16))) float lds_mu[BQ], lds_delta[BQ];
    __shared__ int nonfinite;       // the last query of the tile with something not finite in its row or its gradient's
    int ti, kvh;
    locate(p.first_block + blockIdx.x, p.kv_heads * p.parts, ti, kvh);
    const int part = kvh % p.parts;
    kvh /= p.parts;
    const taco_seq_tile w = p.key_tiles[ti];
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), h = lane >> 5, d = p.dim, G = p.heads / p.kv_heads / p.parts, head0 = (kvh * p.parts + part) * G;
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
    const int qt0 = p.causal ? w.first / BQ : 0, qt1 = (w.length - 1) / BQ + 1;
    const int whole = p.causal ? min(qt1, (w.first + BK) / BQ) : 0;      // tiles from here on hide no key of the workgroup
    Staged<T, DP, BQ, NT> sq, sg;
    float mu_r = 0.f, delta_r = 0.f;
    auto place = [&]() { return ahead<T, DP> ? t : afresh(t); };      // (wide float32 rows: no register holds an address from tile to tile)
    auto fetch_q = [&](int head, int qt) {
        const int q0 = qt * BQ, n = min(BQ, w.length - q0);
        const int64_t at = w.start + q0;
        sq.load(rows_of(p.q.p + at * p.q.ts + head * p.q.hs, n, p.q.ts, rb), p.q.ts, d, place());
        if (t < BQ) {
            float lse = t < n ? p.lse[(at + t) * p.heads + head] : -__builtin_inff();
            delta_r = t < n ? p.delta[(at + t) * p.heads + head] : 0.f;
            mu_r = lse == -__builtin_inff() ? __builtin_inff() : __builtin_fmaf(lse, LOG2E, -LIFT<T>);     // (P comes lifted)
        }
    };
    auto fetch_g = [&](int head, int qt) {
        const int q0 = qt * BQ, n = min(BQ, w.length - q0);
        const int64_t at = w.start + q0;
        sg.load(rows_of(p.d_o.p + at * p.d_o.ts + head * p.d_o.hs, n, p.d_o.ts, rb), p.d_o.ts, d, place());
    };
    auto fetch = [&](int head, int qt) {
        fetch_q(head, qt);
        fetch_g(head, qt);
    };
    auto hide_nonfinite = [&](auto &s) {
        if (!__any(s.any_nonfinite())) return;
        int r = -1;
#pragma unroll
        for (int i = 0; i < Staged<T, DP, BQ, NT>::N; ++i)
            if (s.chunk_nonfinite(i)) r = (i * NT + t) / tile::NC;
        s.nonfinite_to_zero();
        atomicMax(&nonfinite, r);
    };
    auto column = [&]() { return ahead<T, DP> ? lane : afresh(lane); };
    // the tile to LDS; where nothing travels ahead, Q first and dO after it, in the same registers
    auto bring = [&](int head, int qt, auto masked) {
        if (!ahead<T, DP>) fetch_q(head, qt);
        if (decltype(masked)::value) hide_nonfinite(sq);
        sq.put(lds_q, place());
        if (t < BQ) {
            lds_mu[t] = mu_r;
            lds_delta[t] = delta_r;
        }
        if (!ahead<T, DP>) {
            in_order<T, DP>();
            fetch_g(head, qt);
        }
        if (decltype(masked)::value) hide_nonfinite(sg);
        sg.put(lds_g, place());
    };

    f32x16 dk[DB], dv[DB];
    clear(dk);
    clear(dv);
    float f = lift_start<T>;
    // P and dS of 32 queries
    auto weights = [&](int n, f32x16 (&x)[2]) {
        clear(x);
        mma_rows<T>([&](int y) { return tile::rows(lds_q, 32 * n, y, column()); }, kf, x[0]);
        mma_rows<T>([&](int y) { return tile::rows(lds_g, 32 * n, y, column()); }, vf, x[1]);
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            f32x4 mu = *(const f32x4 *)(lds_mu + 32 * n + row_of(i, h)), de = *(const f32x4 *)(lds_delta + 32 * n + row_of(i, h));
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                x[0][i + j] = exp2_(x[0][i + j] * c - mu[j]);
                x[1][i + j] = x[0][i + j] * (x[1][i + j] * p.scale - de[j]);
            }
        }
    };
    if (ahead<T, DP>) fetch(head0, qt0);
    if (t == 0) nonfinite = -1;
    for (int head = head0; head < head0 + G; ++head) {
        int qt = qt0;
        auto next = [&]() {
            if (!ahead<T, DP>) return;
            if (qt + 1 < qt1) fetch(head, qt + 1);
            else if (head + 1 < head0 + G) fetch(head + 1, qt0);
        };
        for (; qt < whole; ++qt) {
            __syncthreads();
            bring(head, qt, std::true_type());
            __syncthreads();
            const int seen_bad = nonfinite;
            next();
#pragma unroll
            for (int n = 0; n < NB; ++n) {
                const int qb = qt * BQ + 32 * n;
                if (qb < first) continue;       // (all of the block comes before the wavefront's keys)
                f32x16 x[2];
                weights(n, x);
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const bool seen = key <= qb + row_of(i, h);
                    x[0][i] = seen ? x[0][i] : 0.f;
                    x[1][i] = seen ? x[1][i] : 0.f;
                }
                lift<T>(x[1], f, dk);
                add_columns<T, DP>(lds_g, 32 * n, x[0], dv, column());
                add_columns<T, DP>(lds_q, 32 * n, x[1], dk, column());
            }
            if (seen_bad >= 0 && key <= qt * BQ + seen_bad) {       // (a key that such a query sees: its gradients are not finite)
#pragma unroll
                for (int b = 0; b < DB; ++b) {
                    dk[b] += __builtin_nanf("");
                    dv[b] += __builtin_nanf("");
                }
            }
            __syncthreads();
            if (t == 0) nonfinite = -1;
        }
        for (; qt < qt1; ++qt) {
            __syncthreads();
            bring(head, qt, std::false_type());
            __syncthreads();
            next();
#pragma unroll
            for (int n = 0; n < NB; ++n) {
                f32x16 x[2];
                weights(n, x);
                lift<T>(x[1], f, dk);
                add_columns<T, DP>(lds_g, 32 * n, x[0], dv, column());
                add_columns<T, DP>(lds_q, 32 * n, x[1], dk, column());
            }
        }
    }
    if constexpr (narrow<T>) {
#pragma unroll
        for (int b = 0; b < DB; ++b) {
            dk[b] *= inverse(f) * (1.f / WEIGHT<T>);
            dv[b] *= 1.f / WEIGHT<T>;
        }
    }
    if (NW == 4 && p.parts > 1) {
        float *to = p.partial + ((((int64_t)ti * 128 + key - w.first) * p.kv_heads + kvh) * p.parts + part) * 2 * DP;
        if (key < w.length) {
            store_row<float>(to, dk, 1.f, DP, lane);
            store_row<float>(to + DP, dv, 1.f, DP, lane);
        }
    } else if (key < w.length) {
        store_row<T>((T *)(p.d_k.p + (int64_t)(w.start + key) * p.d_k.ts + kvh * p.d_k.hs), dk, 1.f, d, lane);
        store_row<T>((T *)(p.d_v.p + (int64_t)(w.start + key) * p.d_v.ts + kvh * p.d_v.hs), dv, 1.f, d, lane);
    }
}

// The same for 128 keys of 16 bits and rows of 128, where the operands and sums of 32 keys leave room for one wavefront on a SIMD only, and nothing to hide its
// waits behind.  K and V stay in LDS instead, and two wavefronts own the same 32 keys: one takes the first 32 queries of each tile, one the others; their
// sums meet in LDS at the end.  Six sequences of up to 4 096 tokens, 16 heads over 4, bf16: 0.57 ms, 710 TFLOP/s of its four products (0.70 ms with one
// wavefront); LDS (48 KB a wavefront and tile for 1 024 clocks of matrix work) is the nearer bound.  fp16 0.61 ms.
template <typename T, int DP> constexpr bool keys_in_lds = sizeof(T) == 2 && DP == 128;
template <typename T, int DP>
__global__ __launch_bounds__(512, 2) void attention_dkv_pair_kernel(AttentionParams p) {
    typedef Tile<T, DP> tile;
    constexpr int BK = 128, BQ = 64, NS = DP / 16, DB = DP / 32, NT = 512, KT = BK * tile::ROW, QT = BQ * tile::ROW;
    __shared__ __attribute__((aligned(16))) char lds[2 * KT + 2 * QT];
    __shared__ __attribute__((aligned(16))) float lds_mu[BQ], lds_delta[BQ];
    __shared__ int nonfinite;       // the last query of the tile with something not finite in its row or its gradient's
    char *const lds_k = lds, *const lds_v = lds + KT, *const lds_q = lds + 2 * KT, *const lds_g = lds + 2 * KT + QT;
    static_assert(4 * DB * 16 * 64 * sizeof(float) <= sizeof(lds), "the sums of four wavefronts");
    int ti, kvh;
    locate(p.first_block + blockIdx.x, p.kv_heads * p.parts, ti, kvh);
    const int part = kvh % p.parts;
    kvh /= p.parts;
    const taco_seq_tile w = p.key_tiles[ti];
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), keys = 32 * (wave & 3), half = wave >> 2, h = lane >> 5, d = p.dim;
    const int G = p.heads / p.kv_heads / p.parts, head0 = (kvh * p.parts + part) * G, first = w.first + keys, key = first + (lane & 31);
    const uint32_t rb = d * sizeof(T);
    const float c = p.scale * LOG2E;
    {
        const int64_t at = w.start + w.first;
        const int n = min(BK, w.length - w.first);
        Staged<T, DP, BK, NT> s;
        s.load(rows_of(p.k.p + at * p.k.ts + kvh * p.k.hs, n, p.k.ts, rb), p.k.ts, d, t);
        s.put(lds_k, t);
        s.load(rows_of(p.v.p + at * p.v.ts + kvh * p.v.hs, n, p.v.ts, rb), p.v.ts, d, t);
        s.put(lds_v, t);
    }
    const int qt0 = p.causal ? w.first / BQ : 0, qt1 = (w.length - 1) / BQ + 1;
    const int whole = p.causal ? min(qt1, (w.first + BK) / BQ) : 0;      // tiles from here on hide no key of the workgroup
    Staged<T, DP, BQ, NT> sq, sg;
    float mu_r = 0.f, delta_r = 0.f;
    auto fetch = [&](int head, int qt) {
        const int q0 = qt * BQ, n = min(BQ, w.length - q0), t_ = afresh(t);
        const int64_t at = w.start + q0;
        sq.load(rows_of(p.q.p + at * p.q.ts + head * p.q.hs, n, p.q.ts, rb), p.q.ts, d, t_);
        sg.load(rows_of(p.d_o.p + at * p.d_o.ts + head * p.d_o.hs, n, p.d_o.ts, rb), p.d_o.ts, d, t_);
        if (t < BQ) {
            float lse = t < n ? p.lse[(at + t) * p.heads + head] : -__builtin_inff();
            delta_r = t < n ? p.delta[(at + t) * p.heads + head] : 0.f;
            mu_r = lse == -__builtin_inff() ? __builtin_inff() : __builtin_fmaf(lse, LOG2E, -LIFT<T>);     // (P comes lifted)
        }
    };
    auto put = [&]() {
        sq.put(lds_q, t);
        sg.put(lds_g, t);
        if (t < BQ) {
            lds_mu[t] = mu_r;
            lds_delta[t] = delta_r;
        }
    };
    f32x16 dk[DB], dv[DB];
    clear(dk);
    clear(dv);
    float f = lift_start<T>;
    // P and dS of this wavefront's 32 queries
    auto weights = [&](f32x16 (&x)[2]) {
        clear(x);
#pragma unroll
        for (int z = 0; z < 2; ++z)
#pragma unroll
            for (int y0 = 0; y0 < NS; y0 += 4) {
                frag<T> a[4], b[4];
#pragma unroll
                for (int y = 0; y < 4; ++y) {
                    a[y] = tile::rows(z ? lds_g : lds_q, 32 * half, y0 + y, lane);
                    b[y] = tile::rows(z ? lds_v : lds_k, keys, y0 + y, lane);
                }
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int y = 0; y < 4; ++y) x[z] = mma(a[y], b[y], x[z]);
            }
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            f32x4 mu = *(const f32x4 *)(lds_mu + 32 * half + row_of(i, h)), de = *(const f32x4 *)(lds_delta + 32 * half + row_of(i, h));
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                x[0][i + j] = exp2_(x[0][i + j] * c - mu[j]);
                x[1][i + j] = x[0][i + j] * (x[1][i + j] * p.scale - de[j]);
            }
        }
    };
    fetch(head0, qt0);
    if (t == 0) nonfinite = -1;
    for (int head = head0; head < head0 + G; ++head) {
        int qt = qt0;
        auto next = [&]() {
            if (qt + 1 < qt1) fetch(head, qt + 1);
            else if (head + 1 < head0 + G) fetch(head + 1, qt0);
        };
        for (; qt < whole; ++qt) {
            __syncthreads();
            if (__any(sq.any_nonfinite() || sg.any_nonfinite())) {
                int r = -1;
#pragma unroll
                for (int i = 0; i < Staged<T, DP, BQ, NT>::N; ++i)
                    if (sq.chunk_nonfinite(i) || sg.chunk_nonfinite(i)) r = (i * NT + t) / tile::NC;
                sq.nonfinite_to_zero();
                sg.nonfinite_to_zero();
                atomicMax(&nonfinite, r);
            }
            put();
            __syncthreads();
            const int seen_bad = nonfinite, qb = qt * BQ + 32 * half;
            next();
            if (qb >= first) {       // (else: all of the block comes before the wavefront's keys)
                f32x16 x[2];
                weights(x);
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const bool seen = key <= qb + row_of(i, h);
                    x[0][i] = seen ? x[0][i] : 0.f;
                    x[1][i] = seen ? x[1][i] : 0.f;
                }
                lift<T>(x[1], f, dk);
                add_columns<T, DP>(lds_g, 32 * half, x[0], dv, lane);
                add_columns<T, DP>(lds_q, 32 * half, x[1], dk, lane);
            }
            if (seen_bad >= 0 && key <= qt * BQ + seen_bad) {       // (a key that such a query sees: its gradients are not finite)
#pragma unroll
                for (int b = 0; b < DB; ++b) {
                    dk[b] += __builtin_nanf("");
                    dv[b] += __builtin_nanf("");
                }
            }
            __syncthreads();
            if (t == 0) nonfinite = -1;
        }
        for (; qt < qt1; ++qt) {
            __syncthreads();
            put();
            __syncthreads();
            next();
            f32x16 x[2];
            weights(x);
            lift<T>(x[1], f, dk);
            add_columns<T, DP>(lds_g, 32 * half, x[0], dv, lane);
            add_columns<T, DP>(lds_q, 32 * half, x[1], dk, lane);
        }
    }
    auto join = [&](f32x16 (&x)[DB]) {
        float *mine = (float *)lds + (wave & 3) * DB * 16 * 64 + lane;
        __syncthreads();
        if (half) {
#pragma unroll
            for (int b = 0; b < DB; ++b)
#pragma unroll
                for (int i = 0; i < 16; ++i) mine[(b * 16 + i) * 64] = x[b][i];
        }
        __syncthreads();
        if (!half) {
#pragma unroll
            for (int b = 0; b < DB; ++b)
#pragma unroll
                for (int i = 0; i < 16; ++i) x[b][i] += mine[(b * 16 + i) * 64];
        }
    };
    if constexpr (narrow<T>) {      // (each of the two wavefronts has a lift of its own)
#pragma unroll
        for (int b = 0; b < DB; ++b) {
            dk[b] *= inverse(f) * (1.f / WEIGHT<T>);
            dv[b] *= 1.f / WEIGHT<T>;
        }
    }
    join(dk);
    join(dv);
    if (half || key >= w.length) return;
    if (p.parts > 1) {
        float *to = p.partial + ((((int64_t)ti * 128 + key - w.first) * p.kv_heads + kvh) * p.parts + part) * 2 * DP;
        store_row<float>(to, dk, 1.f, DP, lane);
        store_row<float>(to + DP, dv, 1.f, DP, lane);
    } else {
        store_row<T>((T *)(p.d_k.p + (int64_t)(w.start + key) * p.d_k.ts + kvh * p.d_k.hs), dk, 1.f, d, lane);
        store_row<T>((T *)(p.d_v.p + (int64_t)(w.start + key) * p.d_v.ts + kvh * p.d_v.hs), dv, 1.f, d, lane);
    }
}

template <typename T, int DP> __global__ __launch_bounds__(256) void attention_sum_kernel(AttentionParams p) {
    int ti, kvh;
    locate(p.first_block + blockIdx.x, p.kv_heads, ti, kvh);
    const taco_seq_tile w = p.key_tiles[ti];
    const int rows = min(128, w.length - w.first);
    for (int e = threadIdx.x; e < rows * (DP / 4); e += 256) {
        const int64_t token = w.start + w.first + e / (DP / 4);
        const int x = e % (DP / 4) * 4;
        const float *from = p.partial + (((int64_t)ti * 128 + e / (DP / 4)) * p.kv_heads + kvh) * p.parts * 2 * DP + x;
        f32x4 dk{0, 0, 0, 0}, dv{0, 0, 0, 0};
        for (int i = 0; i < p.parts; ++i) {
            dk += *(const f32x4 *)(from + i * 2 * DP);
            dv += *(const f32x4 *)(from + i * 2 * DP + DP);
        }
        if (x < p.dim) {
            store4((T *)(p.d_k.p + token * p.d_k.ts + kvh * p.d_k.hs) + x, dk[0], dk[1], dk[2], dk[3]);
            store4((T *)(p.d_v.p + token * p.d_v.ts + kvh * p.d_v.hs) + x, dv[0], dv[1], dv[2], dv[3]);
        }
    }
}

// Backward of sequences of at most 32 tokens, all of it: one wavefront for a sequence and a key-value head.  S and dP are made once (five products), delta is the
// sum of P dP, and dK and dV take P and dS turned around through LDS (a wavefront's own, no barrier).  q, k, v, d_o and lse are read once and the gradients
// written once, where the two launches above read q, k, v and d_o twice and o as well.  Not for float32 rows of 128: their operands leave no registers.
// 131 072 tokens in 6 700 sequences, 4 heads of 32, float32: 0.17 ms, 2.8 TB/s (the two launches: 0.25); each wavefront's chain of loads, products and LDS
// turns is the bound, at two on a SIMD.
template <typename T, int DP> constexpr bool short_gradients = !(sizeof(T) == 4 && DP == 128);
template <typename T, int DP>
__global__ __launch_bounds__(64, DP == 32 ? 2 : 1) void attention_short_grad_kernel(AttentionParams p) {
    typedef Tile<T, DP> tile;
    typedef Tile<T, 32> square;
    typedef Tile<float, 32> square32;       // dS in float16: lifted by key, once it is turned
    constexpr int NS = DP / 16, DB = DP / 32;
    __shared__ __attribute__((aligned(16))) char lds_k[32 * tile::ROW], lds_q[32 * tile::ROW], lds_g[32 * tile::ROW], lds_w[32 * (narrow<T> ? square32::ROW : square::ROW)];
    int ti, kvh;
    locate(p.first_block + blockIdx.x, p.kv_heads, ti, kvh);
    const taco_seq_tile w = p.key_tiles[ti];
    const int lane = threadIdx.x, h = lane >> 5, r = lane & 31, d = p.dim, G = p.heads / p.kv_heads, length = min(w.length, 32);
    const uint32_t rb = d * sizeof(T);
    const float c = p.scale * LOG2E;
    const int64_t at = w.start;
    // the first key, and the last query, with something not finite in its row (a query: or its gradient's); such rows leave the tiles as zeros
    auto stage = [&](char *lds, rsrc from, uint32_t stride, int &first, int &last) {
        Staged<T, DP, 32, 64> s;
        s.load(from, stride, d, lane);
        if (p.causal && __any(s.any_nonfinite())) {
#pragma unroll
            for (int i = 0; i < Staged<T, DP, 32, 64>::N; ++i)
                if (s.chunk_nonfinite(i)) {
                    first = min(first, (i * 64 + lane) / tile::NC);
                    last = max(last, (i * 64 + lane) / tile::NC);
                }
#pragma unroll
            for (int i = 32; i > 0; i >>= 1) {
                first = min(first, __shfl_xor(first, i));
                last = max(last, __shfl_xor(last, i));
            }
            s.nonfinite_to_zero();
        }
        s.put(lds, lane);
    };
    int bad_key = 32, unused = -1;
    stage(lds_k, rows_of(p.k.p + at * p.k.ts + kvh * p.k.hs, length, p.k.ts, rb), p.k.ts, bad_key, unused);
    frag<T> vf[NS];
    {
        const rsrc rv = rows_of(p.v.p + at * p.v.ts + kvh * p.v.hs, length, p.v.ts, rb);
#pragma unroll
        for (int s = 0; s < NS; ++s) vf[s] = rows_global<T>(rv, p.v.ts, d, 0, s, lane);
    }
    f32x16 dk[DB], dv[DB];
    clear(dk);
    clear(dv);
    float fk = lift_start<T>;
    int bad_query = -1;
    for (int head = kvh * G; head < (kvh + 1) * G; ++head) {
        const rsrc rq = rows_of(p.q.p + at * p.q.ts + head * p.q.hs, length, p.q.ts, rb), rg = rows_of(p.d_o.p + at * p.d_o.ts + head * p.d_o.hs, length, p.d_o.ts, rb);
        int ignored = 32;
        __syncthreads();
        stage(lds_q, rq, p.q.ts, ignored, bad_query);
        stage(lds_g, rg, p.d_o.ts, ignored, bad_query);
        const float lse = r < length ? p.lse[(at + r) * p.heads + head] : -__builtin_inff();
        const float mu = lse == -__builtin_inff() ? __builtin_inff() : lse * LOG2E;
        __syncthreads();
        // columns: the queries
        f32x16 x[2];
        clear(x);
#pragma unroll
        for (int s = 0; s < NS; ++s) x[0] = mma(tile::rows(lds_k, 0, s, lane), rows_global<T>(rq, p.q.ts, d, 0, s, lane), x[0]);
#pragma unroll
        for (int s = 0; s < NS; ++s) x[1] = mma(vf[s], rows_global<T>(rg, p.d_o.ts, d, 0, s, lane), x[1]);
        const int limit = p.causal ? r : length - 1;
        float delta = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const bool seen = row_of(i, h) <= limit;
            x[0][i] = seen ? exp2_(x[0][i] * c - mu) : 0.f;
            x[1][i] = seen ? x[1][i] * p.scale : 0.f;
            delta += x[0][i] * x[1][i];
        }
        delta += other_half(delta);
#pragma unroll
        for (int i = 0; i < 16; ++i) x[1][i] = row_of(i, h) <= limit ? x[0][i] * (x[1][i] - delta) : 0.f;
        f32x16 dq[DB];
        clear(dq);
        float fq = lift_start<T>;
        lift<T>(x[1], fq, dq);
        add_columns<T, DP>(lds_k, 0, x[1], dq, lane);
        if (bad_key <= limit) {
#pragma unroll
            for (int b = 0; b < DB; ++b) dq[b] += __builtin_nanf("");
        }
        if (r < length) store_row<T>((T *)(p.d_q.p + (at + r) * p.d_q.ts + head * p.d_q.hs), dq, inverse(fq), d, lane);
        // columns: the keys
#pragma unroll
        for (int y = 0; y < 2; ++y) {
            __syncthreads();
            frag<T> f[2];
            if (narrow<T> && y == 1) {
#pragma unroll
                for (int i = 0; i < 16; ++i) *(float *)(lds_w + square32::at(row_of(i, h), r / 4) + r % 4 * 4) = x[1][i] * inverse(fq);
                __syncthreads();
                f32x16 z;
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    const f32x8 a = square32::rows_permuted(lds_w, 0, 16 * s, lane);
#pragma unroll
                    for (int j = 0; j < 8; ++j) z[8 * s + j] = a[j];
                }
                lift<T>(z, fk, dk);
#pragma unroll
                for (int s = 0; s < 2; ++s) f[s] = to_frag<T>(z, s);
            } else {
#pragma unroll
                for (int i = 0; i < 16; ++i) *(T *)(lds_w + square::at(row_of(i, h), r / square::CE) + r % square::CE * (int)sizeof(T)) = (T)(x[y][i] * (y == 0 ? WEIGHT<T> : 1.f));
                __syncthreads();
#pragma unroll
                for (int s = 0; s < 2; ++s) f[s] = square::rows_permuted(lds_w, 0, 16 * s, lane);
            }
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int b = 0; b < DB; ++b) {
                    if (y == 0) dv[b] = mma(tile::cols(lds_g, 16 * s, 32 * b, lane), f[s], dv[b]);
                    else dk[b] = mma(tile::cols(lds_q, 16 * s, 32 * b, lane), f[s], dk[b]);
                }
        }
    }
    if constexpr (narrow<T>) {
#pragma unroll
        for (int b = 0; b < DB; ++b) {
            dk[b] *= inverse(fk);
            dv[b] *= 1.f / WEIGHT<T>;
        }
    }
    if (r < length) {
        if (r <= bad_query) {       // (a key that such a query sees: its gradients are not finite)
#pragma unroll
            for (int b = 0; b < DB; ++b) {
                dk[b] += __builtin_nanf("");
                dv[b] += __builtin_nanf("");
            }
        }
        store_row<T>((T *)(p.d_k.p + (at + r) * p.d_k.ts + kvh * p.d_k.hs), dk, 1.f, d, lane);
        store_row<T>((T *)(p.d_v.p + (at + r) * p.d_v.ts + kvh * p.d_v.hs), dv, 1.f, d, lane);
    }
}

}  // namespace seq
