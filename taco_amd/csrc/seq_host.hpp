// Host side shared by the entry points of taco_sequence.h: argument checks, errors, type dispatch.
#pragma once
#include "seq_attention.hpp"
#include "seq_launches.hpp"

namespace seq {

int fail(int code, const char *fmt, ...) __attribute__((format(printf, 2, 3), visibility("hidden")));
#define SEQ_API extern "C" __attribute__((visibility("default")))
#define SEQ_NEED(cond, ...) do { if (!(cond)) return ::seq::fail(TACO_SEQ_ERR_INVALID_ARG, __VA_ARGS__); } while (0)

inline int64_t size_of(int dtype) { return dtype == TACO_SEQ_F32 ? 4 : 2; }
inline int padded_dim(int dim) { return (dim + 31) / 32 * 32; }

inline int check_dims(int heads, int kv_heads, int dim, int dtype) {
    SEQ_NEED(dtype >= TACO_SEQ_F32 && dtype <= TACO_SEQ_BF16, "dtype %d is none of TACO_SEQ_F32, TACO_SEQ_F16, TACO_SEQ_BF16", dtype);
    SEQ_NEED(dim >= 8 && dim <= 128 && dim % 8 == 0, "dim %d: a multiple of 8 from 8 to 128 is supported", dim);
    SEQ_NEED(heads >= 1 && kv_heads >= 1 && heads % kv_heads == 0, "%d heads cannot share %d key-value heads", heads, kv_heads);
    SEQ_NEED(heads <= 65535, "%d heads: at most 65535", heads);
    return 0;
}
inline int check_stride(const char *name, int64_t stride, int64_t least, int dtype) {
    SEQ_NEED(stride >= least && stride * size_of(dtype) % 16 == 0, "%s stride of %lld elements: at least %lld and a multiple of 16 bytes", name, (long long)stride, (long long)least);
    return 0;
}
inline int check_pointer(const char *name, const void *p) {
    SEQ_NEED(p && (uintptr_t)p % 16 == 0, "%s: null or not 16-byte aligned", name);
    return 0;
}
// a tile of 128 tokens has to stay inside the 31-bit offsets of a buffer descriptor
inline int check_tensor(const char *name, const taco_seq_tensor &t, int dim, int dtype) {
    if (int rc = check_pointer(name, t.ptr)) return rc;
    if (int rc = check_stride(name, t.token_stride, dim, dtype)) return rc;
    if (int rc = check_stride(name, t.head_stride, 0, dtype)) return rc;
    SEQ_NEED(t.token_stride <= (int64_t)1 << 21, "%s: token stride of %lld elements: at most 2097152", name, (long long)t.token_stride);
    return 0;
}
inline View view(const taco_seq_tensor &t, int dtype) { return View{(char *)t.ptr, t.token_stride * size_of(dtype), t.head_stride * size_of(dtype)}; }

inline int launched(const char *what) {
    hipError_t e = hipGetLastError();
    return e == hipSuccess ? TACO_SEQ_OK : fail(TACO_SEQ_ERR_HIP, "%s: %s", what, hipGetErrorString(e));
}

// f(T(), dim padded as an integral constant) for the call's type and head size
template <int N> struct Int { static constexpr int value = N; };
template <typename F> int dispatch(int dtype, int dim, F f) {
    auto by_dim = [&](auto type) { return dim <= 32 ? f(type, Int<32>()) : dim <= 64 ? f(type, Int<64>()) : dim <= 96 ? f(type, Int<96>()) : f(type, Int<128>()); };
    return dtype == TACO_SEQ_F32 ? by_dim(float()) : dtype == TACO_SEQ_F16 ? by_dim(f16()) : by_dim(bf16());
}

}  // namespace seq
