// Where a token of a paged cache lies: the index arithmetic of taco_attention_step, plain C++ so that it is checked on a host as well.
#pragma once
#include <stdint.h>
#ifndef SEQ_HD
#ifdef __HIPCC__
#define SEQ_HD __host__ __device__ __forceinline__
#else
#define SEQ_HD inline
#endif
#endif

namespace seq {

// How many keys a row has (its cache, and the new token if it joins), or -1: a negative length, or one that its table has no room for.
SEQ_HD int32_t keys_of(int32_t length, int32_t table_width, int32_t page_size, bool joins) {
    const int64_t n = (int64_t)length + (joins ? 1 : 0), room = (int64_t)table_width * page_size;
    return length < 0 || n > room || n > INT32_MAX - 4096 ? -1 : (int32_t)n;
}

struct Place {
    int32_t page, slot;     // page 0, slot 0 if it names none: always inside the cache
    bool bad;
};
// token < keys_of(...), so the table is read inside its width; a page outside [0, num_pages) is bad
SEQ_HD Place place_of(const int32_t *row_table, int32_t token, int32_t page_size, int32_t num_pages) {
    const int32_t n = token / page_size, e = row_table[n];
    const bool bad = e < 0 || e >= num_pages;
    return Place{bad ? 0 : e, bad ? 0 : token - n * page_size, bad};
}

// Offset in elements: 64 bits, a long cache passes 2^31
SEQ_HD int64_t element_of(Place at, int64_t page_stride, int64_t token_stride) { return at.page * page_stride + at.slot * token_stride; }

// The split of a row's keys over workgroups: pieces of `piece` keys, the last one shorter; a row without keys has one piece of none.
SEQ_HD int32_t pieces_of(int32_t keys, int32_t piece) { return keys <= 0 ? 1 : (keys - 1) / piece + 1; }

}  // namespace seq
