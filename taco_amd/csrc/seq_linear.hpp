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
    int32_t n_segments, n_sequences, heads, dim;
    float *carry;           // [modes][n_segments][heads][DP * DP], or NULL: one segment per sequence
};

// log2 of the decay; -inf (a memory of one token) becomes a number that still decays to nothing in one step but gives 1 for none
__device__ __forceinline__ float decay2(const float *log_decay, int head) {
    float x = log_decay[head] * LOG2E;
    return x < -1e30f ? -1e30f : x;
}

// Register i of this lane's part of the state: S[32 b + row_of(i, h)][32 wave + l % 32], block b of the key dimension
template <int DP> __device__ __forceinline__ void state_at(int b, int i, int lane, int wave, int &r, int &c) {
    r = 32 * b + row_of(i, lane >> 5);
    c = 32 * wave + (lane & 31);
}

// acc[b] += K^T (V * tail): the chunk's part of the state.  tail decays per token, so V * tail has float32's 24 bits; it goes through the 16-bit product
// in parts that add up to it, and the state stays as exact as float32 sums: bf16 in three parts of 8 bits; fp16 in two of 11 (the second scaled by
// 2^11, with a sum of its own, so that small values do not fall below fp16's range).
template <int DP, int NB> __device__ __forceinline__ void add_outer(const char *lds_k, int s, f32x8 x, f32x16 (&acc)[NB], f32x16 (&)[NB], int lane, float) {
#pragma unroll
    for (int b = 0; b < NB; ++b) acc[b] = mma(Tile<float, DP>::cols(lds_k, 16 * s, 32 * b, lane), x, acc[b]);
}
template <int DP, int NB> __device__ __forceinline__ void add_outer(const char *lds_k, int s, f32x8 x, f32x16 (&acc)[NB], f32x16 (&)[NB], int lane, bf16) {
    bf16x8 p[3];
#pragma unroll
    for (int n = 0; n < 3; ++n)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            p[n][j] = (bf16)x[j];
            x[j] -= (float)p[n][j];
        }
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        bf16x8 k = Tile<bf16, DP>::cols(lds_k, 16 * s, 32 * b, lane);
#pragma unroll
        for (int n = 2; n >= 0; --n) acc[b] = mma(k, p[n], acc[b]);
    }
}
template <int DP, int NB> __device__ __forceinline__ void add_outer(const char *lds_k, int s, f32x8 x, f32x16 (&acc)[NB], f32x16 (&low)[NB], int lane, f16) {
    f16x8 p, q;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        // x is one float32 from here on: a multiplication fused into one of its two uses and not into the other rounds them apart on a tie
        asm("" : "+v"(x[j]));
        p[j] = (f16)x[j];
        q[j] = (f16)((x[j] - (float)p[j]) * 2048.f);
    }
#pragma unroll
    for (int b = 0; b < NB; ++b) {
        f16x8 k = Tile<f16, DP>::cols(lds_k, 16 * s, 32 * b, lane);
        acc[b] = mma(k, p, acc[b]);
        low[b] = mma(k, q, low[b]);
    }
}

// A segment of one sequence and head in chunks of 64 tokens.  A wavefront owns 32 columns of the value dimension: DP / 32 of them share the chunk's Q, K and V
// tiles in LDS and each holds its columns of the state, float32, in registers.  Per chunk: P^T = K Q^T with the decays (every wavefront makes it for
// itself: cheaper than a turn through LDS), O^T = V^T P^T, plus S^T Q^T with S as the operand it already is, then the state's update.  P and S are rounded
// to the inputs' type for their products, the state itself never is.
// STATES: only the state that the segment makes from nothing, for `carry`.
template <typename T, int DP, bool STATES>
__global__ __launch_bounds__(2 * DP, 1) void linear_kernel(LinearParams p) {
    typedef Tile<T, DP> tile;
    constexpr int C = 64, NT = 2 * DP, NS = DP / 16, DB = DP / 32;
    __shared__ __attribute__((aligned(16))) char lds_k[C * tile::ROW], lds_v[C * tile::ROW], lds_q[STATES ? 16 : C * tile::ROW];
    __shared__ int nonfinite;        // the chunk (its first token) whose V holds something not finite
    const LinearMode m = p.mode[blockIdx.z];
    const int head = blockIdx.y, t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), h = lane >> 5, d = p.dim;
    const taco_seq_segment g = p.segments[blockIdx.x];
    const uint32_t rb = d * sizeof(T);
    const float ld = decay2(p.log_decay, head);
    float *carry = p.carry ? p.carry + (((int64_t)blockIdx.z * p.n_segments + blockIdx.x) * p.heads + head) * DP * DP : nullptr;

    f32x16 s[DB];
    clear(s);
    if (!STATES) {
        if (carry) {
#pragma unroll
            for (int b = 0; b < DB; ++b)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    int r, c;
                    state_at<DP>(b, i, lane, wave, r, c);
                    s[b][i] = carry[r * DP + c];
                }
        } else if (m.s0) {
            const float *s0 = m.s0 + ((int64_t)g.sequence * p.heads + head) * d * d;
#pragma unroll
            for (int b = 0; b < DB; ++b)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    int r, c;
                    state_at<DP>(b, i, lane, wave, r, c);
                    s[b][i] = r < d && c < d ? s0[m.transposed ? c * d + r : r * d + c] * m.s0_scale : 0.f;
                }
        }
    }
    // decays inside a chunk: from key to query (the two blocks of a 32 x 32 triangle's kinds), and to the state behind it
    float w0[16], w1[16];
    if (!STATES) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            int n = (lane & 31) - row_of(i, h);
            w0[i] = n >= 0 ? exp2_(ld * n) : 0.f;
            w1[i] = exp2_(ld * (n + 32));
        }
    }
    const float q_decay0 = exp2_(ld * ((lane & 31) + m.shift)), q_decay1 = exp2_(ld * ((lane & 31) + 32 + m.shift));

    Staged<T, DP, C, NT> sk, sv, sq;
    auto fetch = [&](int c) {
        const int n = min(C, g.count - c), f = g.first + c;
        const int64_t at = g.start + (m.reverse ? g.length - f - n : f);
        rsrc rk = rows_of(m.k.p + at * m.k.ts + head * m.k.hs, n, m.k.ts, rb), rv = rows_of(m.v.p + at * m.v.ts + head * m.v.hs, n, m.v.ts, rb);
        if (m.reverse) {
            sk.load_reversed(rk, m.k.ts, d, n - 1, t);
            sv.load_reversed(rv, m.v.ts, d, n - 1, t);
        } else {
            sk.load(rk, m.k.ts, d, t);
            sv.load(rv, m.v.ts, d, t);
        }
        if (!STATES) {
            rsrc rq = rows_of(m.q.p + at * m.q.ts + head * m.q.hs, n, m.q.ts, rb);
            if (m.reverse) sq.load_reversed(rq, m.q.ts, d, n - 1, t);
            else sq.load(rq, m.q.ts, d, t);
        }
    };
    if (g.count > 0) fetch(0);
    if (t == 0) nonfinite = -1;
    for (int c0 = 0; c0 < g.count; c0 += C) {
        const int n = min(C, g.count - c0);
        __syncthreads();
        if (!STATES && __any(sv.any_nonfinite())) {
            sv.nonfinite_to_zero();
            if (lane == 0) nonfinite = c0;
        }
        sk.put(lds_k, t);
        sv.put(lds_v, t);
        if (!STATES) sq.put(lds_q, t);
        __syncthreads();
        int bad = C;        // the first token of the chunk whose V is not finite in this lane's column
        if (!STATES && nonfinite == c0) {
            const int col = 32 * wave + (lane & 31), f = g.first + c0;
            const char *v = m.v.p + (g.start + (m.reverse ? g.length - 1 - f : f)) * m.v.ts + head * m.v.hs;
            int plus, minus;
            first_nonfinite<T>(v, m.reverse ? -m.v.ts : m.v.ts, col < d ? n : 0, col < d ? col : 0, plus, minus);
            if (col < d && min(plus, minus) < n) bad = min(plus, minus);
        }
        if (c0 + C < g.count) fetch(c0 + C);
        if (!STATES) {
#pragma unroll
            for (int qb = 0; qb < 2; ++qb) {
                if (32 * qb >= n) continue;
                f32x16 o[1], x[1], y[1];
                clear(o);
                clear(y);
                // the chunk itself
#pragma unroll
                for (int kb = qb; kb >= 0; --kb) {
                    clear(x);
#pragma unroll
                    for (int e = 0; e < NS; ++e) x[0] = mma(tile::rows(lds_k, 32 * kb, e, lane), tile::rows(lds_q, 32 * qb, e, lane), x[0]);
#pragma unroll
                    for (int i = 0; i < 16; ++i) x[0][i] = kb == qb ? ((lane & 31) >= row_of(i, h) ? x[0][i] * w0[i] : 0.f) : x[0][i] * w1[i];
#pragma unroll
                    for (int e = 0; e < 2; ++e) o[0] = mma(tile::cols(lds_v, 32 * kb + 16 * e, 32 * wave, lane), to_frag<T>(x[0], e), o[0]);
                }
                // what came before it
#pragma unroll
                for (int b = 0; b < DB; ++b)
#pragma unroll
                    for (int e = 0; e < 2; ++e) y[0] = mma(to_frag<T>(s[b], e), tile::rows_permuted(lds_q, 32 * qb, 32 * b + 16 * e, lane), y[0]);
                const float f = qb ? q_decay1 : q_decay0;
#pragma unroll
                for (int i = 0; i < 16; ++i) o[0][i] += y[0][i] * f;
                if (__any(bad < C)) {
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (__shfl(bad, row_of(i, h)) <= 32 * qb + (lane & 31)) o[0][i] = __builtin_nanf("");
                }
                const int at = c0 + 32 * qb + (lane & 31);
                if (at < g.count) {
                    const int64_t token = g.start + (m.reverse ? g.length - 1 - g.first - at : g.first + at);
                    T *row = (T *)(m.o.p + token * m.o.ts + head * m.o.hs);
#pragma unroll
                    for (int i = 0; i < 16; i += 4) {
                        const int c = 32 * wave + row_of(i, h);
                        if (c < d) store4(row + c, o[0][i] * m.scale, o[0][i + 1] * m.scale, o[0][i + 2] * m.scale, o[0][i + 3] * m.scale);
                    }
                }
            }
        }
        // (shift 0: the chunk's own part decays once more, behind its product: a strong decay would leave nothing of it in fp16)
        const float gn = exp2_(ld * (n - 1 + m.shift));
        f32x16 low[DB];
        clear(low);
#pragma unroll
        for (int b = 0; b < DB; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) s[b][i] *= gn;
#pragma unroll
        for (int e = 0; e < C / 16; ++e) {
            frag<T> v = tile::cols(lds_v, 16 * e, 32 * wave, lane);
            f32x8 x;
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = (float)v[j] * exp2_(ld * max(n - 1 - 16 * e - row_of(j, h), 0));      // (behind the last token: v = 0)
            add_outer<DP>(lds_k, e, x, s, low, lane, T());
        }
        if (__is_same(T, f16)) {
#pragma unroll
            for (int b = 0; b < DB; ++b)
#pragma unroll
                for (int i = 0; i < 16; ++i) s[b][i] += low[b][i] * (1.f / 2048.f);
        }
        if (__any(bad < C)) {
#pragma unroll
            for (int b = 0; b < DB; ++b)
#pragma unroll
                for (int i = 0; i < 16; ++i) s[b][i] = bad < C ? __builtin_nanf("") : s[b][i];
        }
        if (!m.shift) {
            const float g1 = exp2_(ld);
#pragma unroll
            for (int b = 0; b < DB; ++b)
#pragma unroll
                for (int i = 0; i < 16; ++i) s[b][i] *= g1;
        }
    }
    if (STATES) {
#pragma unroll
        for (int b = 0; b < DB; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                int r, c;
                state_at<DP>(b, i, lane, wave, r, c);
                carry[r * DP + c] = s[b][i];
            }
    } else if (m.last && g.first + g.count == g.length && (g.count > 0 || g.length == 0)) {
        float *out = m.last + ((int64_t)g.sequence * p.heads + head) * d * d;
#pragma unroll
        for (int b = 0; b < DB; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                int r, c;
                state_at<DP>(b, i, lane, wave, r, c);
                if (r < d && c < d) out[r * d + c] = s[b][i] * m.last_scale;
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
        const float own = *x;
        *x = s;
        s = s * exp2_(ld * p.segments[i].count) + own;
    }
}

struct LinearStepParams {
    View q, k, v, o;
    const float *log_decay;
    float *state;
    const uint8_t *reset;
    int32_t reset_bytes, rows, heads, dim;
    float scale;
};

// One token: a workgroup per row and head streams the d x d state through registers once, 16 bytes a lane, and sums q S over the key dimension through
// LDS.  8 d^2 bytes for 5 d^2 operations: HBM is the only bound.
template <typename T> __global__ __launch_bounds__(256) void linear_step_kernel(LinearStepParams p) {
    __shared__ float lq[128], lk[128];
    __shared__ __attribute__((aligned(16))) float lv[128], part[1024];
    const int row = blockIdx.x / p.heads, head = blockIdx.x % p.heads, t = threadIdx.x, d = p.dim;
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
    float *s = p.state + (int64_t)blockIdx.x * d * d;
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
