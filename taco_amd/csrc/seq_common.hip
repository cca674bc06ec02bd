// libtaco_sequence.so: version, source hash, errors.
#include <stdarg.h>
#include <stdio.h>
#include "seq_host.hpp"

#ifndef TACO_SOURCE_HASH
#define TACO_SOURCE_HASH "unknown"
#endif
static const char hash_text[] = "taco-src-hash:" TACO_SOURCE_HASH;
static thread_local char error_text[256];

namespace seq {
int fail(int code, const char *fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(error_text, sizeof error_text, fmt, ap);
    va_end(ap);
    return code;
}
}  // namespace seq

SEQ_API int taco_sequence_abi_version(void) { return TACO_SEQUENCE_ABI_VERSION; }
SEQ_API const char *taco_sequence_source_hash(void) { return hash_text + 14; }
SEQ_API const char *taco_sequence_last_error(void) { return error_text; }
