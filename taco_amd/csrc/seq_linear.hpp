// Linear attention with a decay for each head: whole sequences in chunks, forward and backward, and the single-token step
// (include/taco_sequence.h taco_linear_attention*).
#pragma once
#include "seq_attention.hpp"

namespace seq {

// One product o_i = scale * (sum_{j <= i} g^(i-j) (q_i . k_j) v_j + g^(i+shift) q_i S_0): the forward, and each gradient with its roles exchanged:
//   o    q = q,   k = k,   v = v,   first to last token, S_0 = state0,             shift 1
//   dq   q = d_o, k = v,   v = k,   first to last,       S_0 = state0 transposed,  shift 1
//   dk   q = v,   k = d_o, v = q,   last to first,       S_0 = d_state transposed, shift 0
//   dv   q = k,   k = q,   v = d_o, last to first,       S_0 = d_state,            shift 0; its last state is d_state0
// What it carries is S with S_0 as given; a chunk of n tokens makes it g^n S + sum_j g^(n-shift-j) k_j v_j^T, which with shift 1 is the state behind the last
// token and with shift 0 (where S_0 itself does not decay on its way to token 0) that times g, what d_state0 wants.
struct LinearMode {
    View q, k, v, o;
    const float *s0;        // or NULL
    float *last;            // or NULL
    int32_t reverse, transposed, shift;
    float scale, s0_scale, last_scale;      // of o, of S_0 as it is read, of the last state as it is written
};
struct LinearParams {
    LinearMode mode[3];
    const float *log_decay;
    const taco_seq_segment *segments;
    const int32_t *first_segment;
    int32_t n_segments, n_sequences, heads, dim, first_block;      // first_block: of this launch, a segment
    float *carry;           // [modes][n_segments][heads][DP * DP], or NULL: one segment per sequence
};

// log2 of the decay; -inf (a memory of one token) becomes a number that still decays to nothing in one step but gives 1 for none
__device__ __forceinline__ float decay2(const float *log_decay, int head) {
    float x = log_decay[head] * LOG2E;
    return x < -1e30f ? -1e30f : x;
}

// acc[b] += K^T (V * tail), C tokens' part of the state, from row0.  tail decays per token, so V * tail has float32's 24 bits; it goes through the 16-bit product in
// parts that add up to it, and the state stays as exact as float32 sums: bf16 in three parts of 8 bits; fp16 in two of 11 (the second scaled by 2^11, with
// a sum of its own: what is lost of a value is below 2^-36, as much as float32 would lose of values of 2^-12 and more).
template <typename T, int DP, int C> __device__ __forceinline__ void add_outer(const char *lds_k, const char *lds_v, const float *tail, int row0, int col0, f32x16 (&acc)[DP / 32], int lane) {
    typedef Tile<T, DP> tile;
    constexpr int E = C / 16, PARTS = sizeof(T) == 4 ? 1 : __is_same(T, f16) ? 2 : 3;
    auto parts = [&](int e, frag<T> (&p)[PARTS]) {
        const frag<T> v = tile::cols(lds_v, row0 + 16 * e, col0, lane);
        const f32x4 t0 = *(const f32x4 *)(tail + row0 + 16 * e + 4 * (lane >> 5)), t1 = *(const f32x4 *)(tail + row0 + 16 * e + 8 + 4 * (lane >> 5));
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            float x = rounded((float)v[j] * (j < 4 ? t0[j % 4] : t1[j % 4]));      // (fused into one of its uses and not into the other: apart on a tie)
#pragma unroll
            for (int n = 0; n < PARTS; ++n) {
                p[n][j] = (T)x;
                x -= (float)p[n][j];
                if (__is_same(T, f16)) x *= 2048.f;
            }
        }
    };
    if constexpr (PARTS == 2) {
        frag<T> p[E][PARTS];
#pragma unroll
        for (int e = 0; e < E; ++e) parts(e, p[e]);
#pragma unroll
        for (int b = 0; b < DP / 32; ++b) {
            f32x16 low[1];
            clear(low);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const frag<T> k = tile::cols(lds_k, row0 + 16 * e, 32 * b, lane);
                acc[b] = mma(k, p[e][0], acc[b]);
                low[0] = mma(k, p[e][1], low[0]);
            }
            acc[b] += low[0] * (1.f / 2048.f);
        }
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            frag<T> p[PARTS], k[DP / 32];
#pragma unroll
            for (int b = 0; b < DP / 32; ++b) k[b] = tile::cols(lds_k, row0 + 16 * e, 32 * b, lane);
            __builtin_amdgcn_sched_barrier(0);
            parts(e, p);
            // (the same block's sums apart: a product does not wait for the one before it)
#pragma unroll
            for (int n = PARTS - 1; n >= 0; --n)
#pragma unroll
                for (int b = 0; b < DP / 32; ++b) acc[b] = mma(k[b], p[n], acc[b]);
        }
    }
}

// A segment of one sequence and head in chunks of C tokens.  For every 32 columns of the value dimension there are two wavefronts, on one SIMD, with about
// the same number of matrix instructions each: one holds the columns of the state, float32, in registers and updates them (K^T V with the decays); the
// other makes the outputs from the state before the chunk (P^T = K Q^T with the decays, O^T = V^T P^T + S^T Q^T), which the first leaves for it in LDS as
// the operand it will be.  One wavefront for both would need more registers than two on a SIMD can have, and then nothing hides its waits.
// P and S are rounded to the inputs' type for their products, the state itself never is.  In float16 a column of S that does not fit the type is lifted by a power of two (a
// gradient's state is divided by the scale: 5 800 is past 65 504 there with heads of 128).
// 28 700 tokens in 6 sequences, 16 heads of 128, bf16: 0.15 ms for the outputs, 3.1 TB/s (without the outputs' products 0.10: the rest is their latency), 0.07 for
// the segments' own states, 0.01 for joining them: 0.21 ms in all.  With one wavefront for both parts and its spills it took 0.58.  fp16 pays 1 to 5 % for looking at the states' and weights' range.
// STATES: only the state that the segment makes from nothing, for `carry`; there are fewer of these than CUs, so each chunk is shared out to QB keepers, 32
// tokens each, whose sums meet in LDS at the end.
template <typename T> constexpr int chunk_of = sizeof(T) == 4 ? 32 : 64;        // (float32: the tiles and the state's copy have to fit 160 KB of LDS)
template <typename T, int DP, bool STATES>
__global__ __launch_bounds__(STATES ? 2 * DP * (chunk_of<T> / 32) : 4 * DP, 2) void linear_kernel(LinearParams p) {
    typedef Tile<T, DP> tile;
    constexpr int C = chunk_of<T>, NT = STATES ? 2 * DP * (C / 32) : 4 * DP, NS = DP / 16, DB = DP / 32, QB = C / 32;
    __shared__ __attribute__((aligned(16))) char lds_k[C * tile::ROW], lds_v[C * tile::ROW], lds_q[STATES ? 16 : C * tile::ROW];
    __shared__ __attribute__((aligned(16))) char lds_s[STATES ? 16 : DP * tile::ROW];      // the state before the chunk, transposed
    __shared__ __attribute__((aligned(16))) float lowered[narrow<T> && !STATES ? DP : 4];   // what undoes the lift of each column of that state,
    __shared__ int lifted[DB];                                                              // where a block of 32 columns has one
    __shared__ __attribute__((aligned(16))) float tail[C], to_end[32];      // decay from each token to the last of the chunk; of 32 tokens
    __shared__ int first_bad[DP];
    __shared__ int nonfinite;        // the chunk (its first token) whose V holds something not finite
    const LinearMode m = p.mode[blockIdx.z];
    const int head = blockIdx.y, t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), slice = wave % DB, h = lane >> 5, d = p.dim;
    const bool keeper = STATES || wave >= DB;       // of the state; else: makes the outputs
    const int segment = p.first_block + blockIdx.x;
    const taco_seq_segment g = p.segments[segment];
    if (STATES && g.first + g.count == g.length) return;        // (nothing starts from the last segment's state)
    const uint32_t rb = d * sizeof(T);
    const float ld = decay2(p.log_decay, head);
    float *carry = p.carry ? p.carry + (((int64_t)blockIdx.z * p.n_segments + segment) * p.heads + head) * DP * DP : nullptr;
    const int col = 32 * slice + (lane & 31);       // this lane's value dimension

    Staged<T, DP, C, NT> sk, sv, sq;
    auto fetch = [&](int c) {
        const int n = min(C, g.count - c), f = g.first + c;
        const int64_t at = g.start + (m.reverse ? g.length - f - n : f);
        rsrc rk = rows_of(m.k.p + at * m.k.ts + head * m.k.hs, n, m.k.ts, rb), rv = rows_of(m.v.p + at * m.v.ts + head * m.v.hs, n, m.v.ts, rb);
        rsrc rq = rk;
        if (!STATES) rq = rows_of(m.q.p + at * m.q.ts + head * m.q.hs, n, m.q.ts, rb);
        if (m.reverse) {
            sk.load_reversed(rk, m.k.ts, d, n - 1, t);
            sv.load_reversed(rv, m.v.ts, d, n - 1, t);
            if (!STATES) sq.load_reversed(rq, m.q.ts, d, n - 1, t);
        } else {
            sk.load(rk, m.k.ts, d, t);
            sv.load(rv, m.v.ts, d, t);
            if (!STATES) sq.load(rq, m.q.ts, d, t);
        }
    };
    // the next chunk into LDS: `leave` between the barriers
    auto advance = [&](int c0, auto leave) {
        const int n = min(C, g.count - c0);
        __syncthreads();
        if (!STATES && __any(sv.any_nonfinite())) {
            sv.nonfinite_to_zero();
            if (lane == 0) nonfinite = c0;
        }
        sk.put(lds_k, t);
        sv.put(lds_v, t);
        if (!STATES) sq.put(lds_q, t);
        if (n < C && t < C) tail[t] = exp2_(ld * max(n - 1 - t, 0));     // (behind the last token: v = 0)
        leave();
        __syncthreads();
        if (c0 + C < g.count) fetch(c0 + C);
        return n;
    };
    // the first token of the chunk whose V is not finite in this lane's column (C: none)
    auto first_nonfinite_token = [&](int c0, int n) {
        const int f = g.first + c0;
        const char *v = m.v.p + (g.start + (m.reverse ? g.length - 1 - f : f)) * m.v.ts + head * m.v.hs;
        int plus, minus;
        first_nonfinite<T>(v, m.reverse ? -m.v.ts : m.v.ts, col < d ? n : 0, col < d ? col : 0, plus, minus);
        return col < d && min(plus, minus) < n ? min(plus, minus) : C;
    };
    if (g.count > 0) fetch(0);
    if (t == 0) nonfinite = -1;
    if (t < C) tail[t] = exp2_(ld * (C - 1 - t));
    if (t < 32) to_end[t] = exp2_(ld * (31 - t));

    if (keeper) {
        f32x16 s[DB];
        clear(s);
        if (!STATES) {
            const float *from = carry ? carry : m.s0 ? m.s0 + ((int64_t)g.sequence * p.heads + head) * d * d : nullptr;
            const int size = carry ? DP : d;
            const bool turned = !carry && m.transposed;
            const float f = carry ? 1.f : m.s0_scale;
            // (through a descriptor: outside reads as zero, and all loads are on their way at once)
            const rsrc state = rows_of(from, from ? 1 : 0, 0, size * size * 4);
#pragma unroll
            for (int b = 0; b < DB; ++b)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int r = 32 * b + row_of(i, h);
                    s[b][i] = load4(state, r < size && col < size ? (turned ? col * size + r : r * size + col) * 4 : OUTSIDE);
                }
#pragma unroll
            for (int b = 0; b < DB; ++b) s[b] *= f;
        }
        for (int c0 = 0; c0 < g.count; c0 += C) {
            bool lift = false;
            float f = 1.f;
            if constexpr (narrow<T> && !STATES) {
                float x = largest(s);
                lift = __any(!in_range(x));
                if (lift) {
                    x = fmaxf(x, other_half(x));
                    f = in_range(x) ? 1.f : lift_of(x);
                }
            }
            const int n = advance(c0, [&]() {
                if constexpr (!STATES) {
                    auto store = [&](auto g) {
#pragma unroll
                        for (int b = 0; b < DB; ++b)
#pragma unroll
                            for (int i = 0; i < 16; i += 4) {
                                const int r = 32 * b + row_of(i, h);
                                store4((T *)(lds_s + tile::at(col, r / tile::CE) + r % tile::CE * (int)sizeof(T)), g(s[b][i]), g(s[b][i + 1]), g(s[b][i + 2]), g(s[b][i + 3]));
                            }
                    };
                    if (narrow<T> && lift) store([&](float y) { return y * f; });
                    else store([](float y) { return y; });
                    if (narrow<T> && lift && h == 0) lowered[col] = inverse(f);
                    if (narrow<T> && lane == 0) lifted[slice] = lift;
                }
            });
            // (shift 0: the chunk's own part decays once more, behind its product: a strong decay would leave nothing of it in fp16)
            const float gn = exp2_(ld * (n - 1 + m.shift));
#pragma unroll
            for (int b = 0; b < DB; ++b) s[b] *= gn;
            if constexpr (STATES) add_outer<T, DP, 32>(lds_k, lds_v, tail, 32 * (wave / DB), 32 * slice, s, lane);
            else add_outer<T, DP, C>(lds_k, lds_v, tail, 0, 32 * slice, s, lane);
            if (!STATES && nonfinite == c0) {
                const bool bad = first_nonfinite_token(c0, n) < C;
#pragma unroll
                for (int b = 0; b < DB; ++b) s[b] += bad ? __builtin_nanf("") : 0.f;
            }
            if (!m.shift) {
                const float g1 = exp2_(ld);
#pragma unroll
                for (int b = 0; b < DB; ++b) s[b] *= g1;
            }
        }
        if (STATES) {
            if constexpr (QB == 2) {
                static_assert(DB * 16 * 64 * sizeof(float) <= sizeof(lds_k), "a block of every keeper's");
                float *sums = (float *)lds_k + slice * 16 * 64 + lane;
#pragma unroll
                for (int b = 0; b < DB; ++b) {
                    __syncthreads();
                    if (wave >= DB) {
#pragma unroll
                        for (int i = 0; i < 16; ++i) sums[i * 64] = s[b][i];
                    }
                    __syncthreads();
                    if (wave < DB) {
#pragma unroll
                        for (int i = 0; i < 16; ++i) s[b][i] += sums[i * 64];
                    }
                }
                if (wave >= DB) return;
            }
#pragma unroll
            for (int b = 0; b < DB; ++b)
#pragma unroll
                for (int i = 0; i < 16; ++i) carry[(32 * b + row_of(i, h)) * DP + col] = s[b][i];
        } else if (m.last && g.first + g.count == g.length && (g.count > 0 || g.length == 0)) {
            float *out = m.last + ((int64_t)g.sequence * p.heads + head) * d * d;
#pragma unroll
            for (int b = 0; b < DB; ++b)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int r = 32 * b + row_of(i, h);
                    if (r < d && col < d) out[r * d + col] = s[b][i] * m.last_scale;
                }
        }
        return;
    }
    if constexpr (!STATES) {
        // (the weights carry the scale before they are rounded; in float16, those of a block and query that do not fit the type are lifted by a power of two)
        // decay from key to query inside a block of 32; from an earlier block: the key's to that block's end (to_end), then this lane's query's from there
        float w0[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int n = (lane & 31) - row_of(i, h);
            w0[i] = n >= 0 ? exp2_(ld * n) * m.scale : 0.f;
        }
        const float q_entry = exp2_(ld * ((lane & 31) + 1)) * m.scale;
        for (int c0 = 0; c0 < g.count; c0 += C) {
            const int n = advance(c0, []() {});
            const bool bad = nonfinite == c0;
            if (bad) {
                first_bad[col] = first_nonfinite_token(c0, n);      // (both halves of the wavefront write the same)
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            }
#pragma unroll
            for (int qb = 0; qb < QB; ++qb) {
                if (32 * qb >= n) continue;
                frag<T> qf[NS];
#pragma unroll
                for (int e = 0; e < NS; ++e) qf[e] = tile::rows(lds_q, 32 * qb, e, lane);
                f32x16 o[1], x[1];
                clear(o);
                // what came before the chunk
                mma_rows<T>([&](int e) { return tile::rows(lds_s, 32 * slice, e, lane); }, qf, o[0]);
                o[0] *= exp2_(ld * (32 * qb + (lane & 31) + m.shift)) * m.scale;
                if (narrow<T> && lifted[slice]) {
#pragma unroll
                    for (int i = 0; i < 16; i += 4) {
                        const f32x4 u = *(const f32x4 *)(lowered + 32 * slice + row_of(i, h));
#pragma unroll
                        for (int j = 0; j < 4; ++j) o[0][i + j] *= u[j];
                    }
                }
                // the chunk itself
#pragma unroll
                for (int kb = qb; kb >= 0; --kb) {
                    frag<T> vf[2];
                    clear(x);
                    mma_rows<T>([&](int e) { return tile::rows(lds_k, 32 * kb, e, lane); }, qf, x[0]);
#pragma unroll
                    for (int e = 0; e < 2; ++e) vf[e] = tile::cols(lds_v, 32 * kb + 16 * e, 32 * slice, lane);
#pragma unroll
                    for (int i = 0; i < 16; i += 4) {
                        const f32x4 w = *(const f32x4 *)(to_end + row_of(i, h));
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            x[0][i + j] = kb == qb ? ((lane & 31) >= row_of(i + j, h) ? x[0][i + j] * w0[i + j] : 0.f) : x[0][i + j] * (w[j] * q_entry);
                    }
                    float f = 1.f;          // (outside: the whole sum is lifted with this block's weights, and lowered behind them)
                    bool lift = false;
                    if constexpr (narrow<T>) {
                        float y = largest(x);
                        lift = __any(!in_range(y));
                        if (lift) {
                            y = fmaxf(y, other_half(y));
                            f = in_range(y) ? 1.f : lift_of(y);
                            x[0] *= f;
                            o[0] *= f;
                        }
                    }
#pragma unroll
                    for (int e = 0; e < 2; ++e) o[0] = mma(vf[e], to_frag<T>(x[0], e), o[0]);
                    if (narrow<T> && lift) o[0] *= inverse(f);
                }
                if (bad) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[0][i] = first_bad[32 * slice + row_of(i, h)] <= 32 * qb + (lane & 31) ? __builtin_nanf("") : o[0][i];
                }
                const int at = c0 + 32 * qb + (lane & 31);
                if (at < g.count) {
                    const int64_t token = g.start + (m.reverse ? g.length - 1 - g.first - at : g.first + at);
                    T *row = (T *)(m.o.p + token * m.o.ts + head * m.o.hs);
#pragma unroll
                    for (int i = 0; i < 16; i += 4) {
                        const int c = 32 * slice + row_of(i, h);
                        if (c < d) store4(row + c, o[0][i], o[0][i + 1], o[0][i + 2], o[0][i + 3]);
                    }
                }
            }
        }
    }
}

// carry[segment]: from what the segment makes itself to the state it starts with, along the segments of each sequence
template <int DP> __global__ __launch_bounds__(256) void linear_scan_kernel(LinearParams p) {
    const LinearMode m = p.mode[blockIdx.z];
    const int seq = blockIdx.y / p.heads, head = blockIdx.y % p.heads, e = blockIdx.x * 256 + threadIdx.x, r = e / DP, c = e % DP, d = p.dim;
    const float ld = decay2(p.log_decay, head);
    float s = m.s0 && r < d && c < d ? m.s0[((int64_t)seq * p.heads + head) * d * d + (m.transposed ? c * d + r : r * d + c)] * m.s0_scale : 0.f;
    for (int i = p.first_segment[seq]; i < p.first_segment[seq + 1]; ++i) {
        float *x = p.carry + (((int64_t)blockIdx.z * p.n_segments + i) * p.heads + head) * DP * DP + e;
        const float own = i + 1 < p.first_segment[seq + 1] ? *x : 0.f;      // (the last segment's is not made, and nothing starts from it)
        *x = s;
        s = s * exp2_(ld * p.segments[i].count) + own;
    }
}

struct LinearStepParams {
    View q, k, v, o;
    const float *log_decay;
    float *state;
    const uint8_t *reset;
    int32_t reset_bytes, rows, heads, dim, first_block;
    float scale;
};

// One token: a workgroup per row and head streams the d x d state through registers once, 16 bytes a lane, and sums q S over the key dimension through
// LDS.  8 d^2 bytes for 5 d^2 operations: HBM is the only bound.  4 096 rows, 4 heads of 64: 103 us, 5.4 TB/s.
template <typename T> __global__ __launch_bounds__(256) void linear_step_kernel(LinearStepParams p) {
    __shared__ float lq[128], lk[128];
    __shared__ __attribute__((aligned(16))) float lv[128], part[1024];
    const int block = p.first_block + blockIdx.x, row = block / p.heads, head = block % p.heads, t = threadIdx.x, d = p.dim;
    if (t < d) {
        lq[t] = (float)((const T *)(p.q.p + row * p.q.ts + head * p.q.hs))[t];
        lk[t] = (float)((const T *)(p.k.p + row * p.k.ts + head * p.k.hs))[t];
        lv[t] = (float)((const T *)(p.v.p + row * p.v.ts + head * p.v.hs))[t];
    }
    bool fresh = false;
    if (p.reset)
        for (int i = 0; i < p.reset_bytes; ++i) fresh |= p.reset[(int64_t)row * p.reset_bytes + i] != 0;
    const float g = exp2_(decay2(p.log_decay, head));
    __syncthreads();
    float *s = p.state + (int64_t)block * d * d;
    const int w = d / 4, lanes = 256 / w * w, step = lanes / w, c = t % w * 4;      // w lanes across, `step` key rows at a time
    f32x4 a{0, 0, 0, 0};
    if (t < lanes) {
        const f32x4 v = *(const f32x4 *)(lv + c);
        for (int r = t / w; r < d; r += step) {
            f32x4 *x = (f32x4 *)(s + r * d + c);
            f32x4 y{0, 0, 0, 0};
            if (!fresh) y = *x * g;
            y += lk[r] * v;
            *x = y;
            a += lq[r] * y;
        }
        *(f32x4 *)(part + t * 4) = a;
    }
    __syncthreads();
    if (t < d) {
        float y = 0.f;
        for (int i = 0; i < step; ++i) y += part[i * d + t];
        ((T *)(p.o.p + row * p.o.ts + head * p.o.hs))[t] = (T)(y * p.scale);
    }
}

}  // namespace seq
