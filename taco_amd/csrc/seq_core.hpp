// What the sequence kernels share: element types, 32x32 matrix tiles, swizzled LDS tiles, bounds-checked loads.
//
// Every product runs on 32x32 MFMAs with 16 values of the contraction per step.  Lane l = 32 h + r of the A operand holds row r and the contraction's
// slots 8 h + j, j < 8; B the same for its columns; register i of the result is row 8 (i / 4) + 4 h + i % 4 of column r.  Two facts carry all kernels:
//  * a contraction may be permuted as long as A and B agree.  The result of one product (columns = lane) is therefore the B (or A) operand of the
//    next one as it stands: slot (h, j) of step s is row 16 s + 8 (j / 4) + 4 h + j % 4, "permuted order" below.  Scores never leave the registers.
//  * float32 runs through the same fragments: eight 32x32x2 MFMAs take element j of both operands in turn.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace seq {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16;
typedef _Float16 f16;

template <typename T> struct Frag;
template <> struct Frag<float> { typedef f32x8 type; };
template <> struct Frag<f16> { typedef f16x8 type; };
template <> struct Frag<bf16> { typedef bf16x8 type; };
template <typename T> using frag = typename Frag<T>::type;

__device__ __forceinline__ f32x16 mma(bf16x8 a, bf16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 mma(f16x8 a, f16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 mma(f32x8 a, f32x8 b, f32x16 c) {
#pragma unroll
    for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], c, 0, 0, 0);
    return c;
}

// row (of a product's result) that register i of half h holds; also the permuted order of a contraction, i = 8 (step % 2) + j
__device__ __forceinline__ int row_of(int i, int h) { return 8 * (i / 4) + 4 * h + i % 4; }

// registers 8 s .. 8 s + 7 of a result as an operand in permuted order: rounded to nearest even, once
template <typename T> __device__ __forceinline__ frag<T> to_frag(const f32x16 &x, int s) {
    frag<T> f;
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = (T)x[8 * s + j];
    return f;
}

template <int N> __device__ __forceinline__ void clear(f32x16 (&x)[N]) {
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i) x[n][i] = 0.f;
}

__device__ __forceinline__ float other_half(float x) { return __shfl_xor(x, 32); }
__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float log2_(float x) { return __builtin_amdgcn_logf(x); }
// a product as it was rounded, wherever it is used (not fused into one of its uses and rounded apart from the others).  The softmax keeps its maximum that way:
// the factor that joins two maxima is then exactly 1 where a row's own has not changed, and sums do not drift by a rounding each time another row's does.
__device__ __forceinline__ float rounded(float x) {
    asm("" : "+v"(x));
    return x;
}
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

// ---- float16's range.  An operand that is rounded for a product (a weight, its gradient, a state) may lie outside float16's range, or below 2^-14, where digits are
// lost, while the inputs and the result do not.  It is multiplied by a power of two first and the product divided by it, both exact.
template <typename T> constexpr bool narrow = __is_same(T, f16);
// the power of two that brings the largest absolute value m to [2^14, 2^15); at most 2^64
__device__ __forceinline__ float lift_of(float m) { return __builtin_bit_cast(float, (268 - max((int)(__builtin_bit_cast(uint32_t, m) >> 23), 77)) << 23); }
__device__ __forceinline__ float inverse(float power_of_two) { return __builtin_bit_cast(float, (254u << 23) - __builtin_bit_cast(uint32_t, power_of_two)); }
// The largest value of an operand is between: what is small beside it loses no more than 2^-17 of it (half a step below 2^-14 is 2^-25), less than a half step of the
// type does, and nothing is lifted.  Nothing but zeros needs no lift either.
__device__ __forceinline__ bool in_range(float m) { return m == 0.f || (m >= 0.00390625f && m < 32768.f); }
template <int N> __device__ __forceinline__ float largest(const f32x16 (&x)[N]) {
    float m[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i) m[i % 4] = fmaxf(m[i % 4], __builtin_fabsf(x[n][i]));
    return fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
}
// An operand that is made block by block while a product runs, a column (lane) at a time: x becomes x times a power of two `f` that the column keeps, chosen by its largest
// value so far, and the sums acc with it.  f starts at 2^64 and falls: what comes later and is smaller loses no more than 2^-39 of the largest.
template <typename T, int N> __device__ __forceinline__ void lift(f32x16 &x, float &f, f32x16 (&acc)[N]) {
    if constexpr (narrow<T>) {
        const f32x16 y[1] = {x};
        float m = largest(y);
        if (__any(m * f >= 32768.f)) {
            m = fmaxf(m, other_half(m));
            const float g = m * f >= 32768.f ? lift_of(m) : f, a = g * inverse(f);
            f = g;
#pragma unroll
            for (int n = 0; n < N; ++n) acc[n] *= a;
        }
        x *= f;
    }
}
// A softmax's weight is at most 1 (a rounding more as it is computed): always lifted by 2^15, and the sum lowered by as much
template <typename T> constexpr float LIFT = narrow<T> ? 15.f : 0.f;
template <typename T> constexpr float WEIGHT = narrow<T> ? 32768.f : 1.f;
template <typename T> constexpr float lift_start = narrow<T> ? 18446744073709551616.f : 1.f;

// ---- LDS tiles: rows of DP elements (the head dimension padded with zeros to 32, 64, 96 or 128; 96 in the room of 128), 16-byte chunks exchanged inside each row by an XOR that
// depends on the row.  256 bytes are one turn of the 64 banks.  A row-wise read (32 rows, the same chunk) wants 16 neighbouring rows in 16 different
// chunk positions; a column-wise read (4 neighbouring rows, 64 bytes each) wants the four rows in different quarters.  flip() gives both.
template <typename T, int DP> struct Tile {
    static constexpr int NC = DP * (int)sizeof(T) / 16;         // chunks of a row
    static constexpr int CE = 16 / (int)sizeof(T);              // elements of a chunk
    static constexpr int ROOM = DP == 96 ? NC / 3 * 4 : NC;     // chunks that a row has room for, a power of two
    static constexpr int ROW = ROOM * 16;                       // bytes of a row
    static __device__ __forceinline__ int flip(int r) {
        if (ROOM == 4) return (r >> 2) & 3;
        if (ROOM == 8) return ((r >> 1) & 1) << 2 | ((r >> 2) & 3);
        return (r & 3) << 2 | ((r >> 2) & 3);
    }
    static __device__ __forceinline__ int at(int r, int c) { return r * ROW + ((c ^ flip(r)) << 4); }
    static __device__ __forceinline__ void put(char *lds, int r, int c, u32x4 x) { *(u32x4 *)(lds + at(r, c)) = x; }
    static __device__ __forceinline__ T get(const char *lds, int r, int d) { return *(const T *)(lds + at(r, d / CE) + (d % CE) * (int)sizeof(T)); }

    // operand whose lane is a row of the tile (row0 + l % 32), contraction over the columns 16 s + 8 h + j
    static __device__ __forceinline__ frag<T> rows(const char *lds, int row0, int s, int lane) {
        int r = row0 + (lane & 31), h = lane >> 5;
        if constexpr (sizeof(T) == 2) {
            return *(const frag<T> *)(lds + at(r, 2 * s + h));
        } else {
            f32x4 a = *(const f32x4 *)(lds + at(r, 4 * s + 2 * h)), b = *(const f32x4 *)(lds + at(r, 4 * s + 2 * h + 1));
            return f32x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
        }
    }
    // the same with the columns col0 + (permuted order): the partner of a result used as an operand
    static __device__ __forceinline__ frag<T> rows_permuted(const char *lds, int row0, int col0, int lane) {
        int r = row0 + (lane & 31), h = lane >> 5;
        if constexpr (sizeof(T) == 2) {
            s16x4 a = *(const s16x4 *)(lds + at(r, col0 / 8) + 8 * h), b = *(const s16x4 *)(lds + at(r, col0 / 8 + 1) + 8 * h);
            return __builtin_bit_cast(frag<T>, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
        } else {
            f32x4 a = *(const f32x4 *)(lds + at(r, col0 / 4 + h)), b = *(const f32x4 *)(lds + at(r, col0 / 4 + 2 + h));
            return f32x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
        }
    }
    // operand whose lane is a column of the tile (col0 + l % 32), contraction over the rows row0 + (permuted order).  16 bit: the transposing LDS
    // read: 16 lanes name four rows of 16 columns, 8 bytes each, and receive a column of four.  All 64 lanes have to be active.
    static __device__ __forceinline__ frag<T> cols(const char *lds, int row0, int col0, int lane) {
        int h = lane >> 5;
        if constexpr (sizeof(T) == 2) {
            typedef s16x4 __attribute__((address_space(3))) *lds4;
            int i = lane & 15, r = row0 + 4 * h + (i >> 2), c = col0 / 8 + 2 * ((lane >> 4) & 1) + ((i & 3) >> 1), b = (i & 1) * 8;
            s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(lds + at(r, c) + b));
            s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(lds + at(r + 8, c) + b));
            return __builtin_bit_cast(frag<T>, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
        } else {
            f32x8 f;
            int d = col0 + (lane & 31);
#pragma unroll
            for (int j = 0; j < 8; ++j) f[j] = get(lds, row0 + row_of(j, h), d);
            return f;
        }
    }
};

// acc += A B over DP / 16 steps: A's fragments from `a(step)`, all asked of LDS before the first product waits for one (left to itself the compiler asks for each
// right before its use, and the matrix pipe idles for an LDS round trip every time)
template <typename T, int NS, typename A> __device__ __forceinline__ void mma_rows(A a, const frag<T> (&b)[NS], f32x16 &acc) {
    constexpr int AHEAD = sizeof(T) == 2 ? NS : 2;
#pragma unroll
    for (int s0 = 0; s0 < NS; s0 += AHEAD) {
        frag<T> f[AHEAD];
#pragma unroll
        for (int s = 0; s < AHEAD; ++s) f[s] = a(s0 + s);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int s = 0; s < AHEAD; ++s) acc = mma(f[s], b[s0 + s], acc);
    }
}

// the value itself, but not known to be the same from one turn of a loop to the next: what is computed from it is computed again each time instead of being
// kept in registers that the loop has no room for
__device__ __forceinline__ int afresh(int x) {
    asm volatile("" : "+v"(x));
    return x;
}

// ---- Global memory.  A buffer descriptor covers the rows of one tile that exist; what lies outside reads as zero, so no lane branches and padding rows and
// padding columns cost nothing.  The base is 64 bits and moves with the tile, offsets inside it are 32.
typedef __amdgpu_buffer_rsrc_t rsrc;
__device__ __forceinline__ rsrc rows_of(const void *base, int rows, uint32_t stride_bytes, uint32_t row_bytes) {
    uint32_t n = rows > 0 ? (uint32_t)(rows - 1) * stride_bytes + row_bytes : 0u;
    return __builtin_amdgcn_make_buffer_rsrc((void *)base, 0, n, 0x00020000);
}
__device__ __forceinline__ u32x4 load16(rsrc r, uint32_t off) { return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0)); }
__device__ __forceinline__ float load4(rsrc r, uint32_t off) { return __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(r, off, 0, 0)); }
constexpr uint32_t OUTSIDE = 0x80000000u;      // an offset no descriptor reaches (tiles stay below 2 GiB)

// a tile of ROWS rows in the registers of NT threads, on its way from global memory to LDS
template <typename T, int DP, int ROWS, int NT> struct Staged {
    typedef Tile<T, DP> tile;
    static constexpr int N = ROWS * tile::NC / NT;
    static_assert(ROWS * tile::NC % NT == 0, "whole chunks per thread");
    u32x4 x[N];
    __device__ __forceinline__ void load(rsrc r, uint32_t stride_bytes, int d, int t) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            int e = i * NT + t, row = e / tile::NC, c = e % tile::NC;
            x[i] = load16(r, c * tile::CE < d ? row * stride_bytes + c * 16 : OUTSIDE);
        }
    }
    // row j of the tile is row last - j of the descriptor (a sequence read backwards); negative rows wrap to offsets outside
    __device__ __forceinline__ void load_reversed(rsrc r, uint32_t stride_bytes, int d, int last, int t) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            int e = i * NT + t, row = last - e / tile::NC, c = e % tile::NC;
            x[i] = load16(r, c * tile::CE < d && row >= 0 ? row * stride_bytes + c * 16 : OUTSIDE);
        }
    }
    __device__ __forceinline__ void put(char *lds, int t) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            int e = i * NT + t;
            tile::put(lds, e / tile::NC, e % tile::NC, x[i]);
        }
    }
    // NaN and infinities have an exponent of all ones: adding one to its last place carries into the sign's bit, which is masked out first
    static constexpr uint32_t MAGNITUDE = sizeof(T) == 4 ? 0x7fffffffu : 0x7fff7fffu, SIGNS = ~MAGNITUDE,
                              STEP = sizeof(T) == 4 ? 0x00800000u : __is_same(T, f16) ? 0x04000400u : 0x00800080u;
    __device__ __forceinline__ bool any_nonfinite() const {
        bool bad = false;
#pragma unroll
        for (int i = 0; i < N; ++i) bad |= chunk_nonfinite(i);
        return bad;
    }
    __device__ __forceinline__ bool chunk_nonfinite(int i) const {
        uint32_t bad = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) bad |= (x[i][j] & MAGNITUDE) + STEP;
        return bad & SIGNS;
    }
    __device__ __forceinline__ void nonfinite_to_zero() {
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                uint32_t bad = ((x[i][j] & MAGNITUDE) + STEP) & SIGNS;      // the sign bits of what goes
                x[i][j] &= sizeof(T) == 4 ? (bad ? 0u : ~0u) : ~((bad >> 15) * 0xffffu);
            }
    }
};

// operand whose lane is a row of global memory (row0 + l % 32), contraction over the columns 16 s + 8 h + j
template <typename T> __device__ __forceinline__ frag<T> rows_global(rsrc r, uint32_t stride_bytes, int d, int row0, int s, int lane) {
    uint32_t off = (row0 + (lane & 31)) * stride_bytes;
    int c = 16 * s + 8 * (lane >> 5);
    u32x4 a = load16(r, c < d ? off + c * (int)sizeof(T) : OUTSIDE);
    if constexpr (sizeof(T) == 2) return __builtin_bit_cast(frag<T>, a);
    else {
        u32x4 b = load16(r, c < d ? off + c * 4 + 16 : OUTSIDE);
        return __builtin_bit_cast(f32x8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
    }
}

// four neighbouring elements of a row, rounded to T
template <typename T> __device__ __forceinline__ void store4(T *p, float a, float b, float c, float d) {
    if constexpr (sizeof(T) == 4) *(f32x4 *)p = f32x4{a, b, c, d};
    else {
        typedef T t4 __attribute__((ext_vector_type(4)));
        *(t4 *)p = t4{(T)a, (T)b, (T)c, (T)d};
    }
}

// acc[db] (rows = dimension, column = this lane's row) * f -> a row of global memory
template <typename T, int DB> __device__ __forceinline__ void store_row(T *row, const f32x16 (&acc)[DB], float f, int d, int lane) {
    int h = lane >> 5;
#pragma unroll
    for (int b = 0; b < DB; ++b)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            int c = 32 * b + 8 * (i / 4) + 4 * h;
            if (c < d) store4(row + c, acc[b][i] * f, acc[b][i + 1] * f, acc[b][i + 2] * f, acc[b][i + 3] * f);
        }
}

// ---- Hidden rows that are not finite.  A tile in which rows of a sequence are hidden from some columns goes through a matrix product with weights of 0 for
// them, and 0 * NaN is NaN.  Such a tile (only those on the diagonal) is therefore looked over on its way into LDS, three operations for four bytes; if
// anything in it is not finite, it is written without that, a flag says so, and the few lines below put what the columns do see back in: rare, and slow.

// Column `col` of n rows of global memory: the first row that holds +inf or NaN, and the first that holds -inf or NaN (n: none)
template <typename T> __device__ inline void first_nonfinite(const char *base, int64_t stride_bytes, int n, int col, int &plus, int &minus) {
    plus = minus = n;
    for (int r = n - 1; r >= 0; --r) {
        const float x = (float)((const T *)(base + r * stride_bytes))[col];
        if (__builtin_fabsf(x) < __builtin_inff()) continue;
        if (!(x < 0.f)) plus = r;
        if (!(x > 0.f)) minus = r;
    }
}

}  // namespace seq
