/*
 * taco_sequence.h -- C ABI of libtaco_sequence.so: the sequence memory of a policy on an MI355X (gfx950).
 *
 * The reference's policy remembers through frame stacks and an LSTM (nets_asymmetry.py:128-136); its attention encoder works on the same short
 * stacks.  These entry points hold a memory of any length, in the two forms a policy needs it: over whole episodes packed one behind the other
 * (training), and one token per row and call (acting).
 *
 * Ownership, errors and streams as in taco_env.h: the caller allocates every buffer, the library borrows DEVICE pointers for the call, enqueues on
 * the caller's stream (whose device has to be the current one), never synchronises, allocates or throws.  Every function returns TACO_SEQ_OK or
 * a negative status; taco_sequence_last_error() returns a thread-local message.  Everything may be captured into a HIP graph.  No sum depends on an
 * order that is not fixed: the same call gives the same bits.
 *
 * Tensors: `ptr` 16-byte aligned, the head dimension contiguous, token and head strides in ELEMENTS, multiples of 16 bytes, token strides (and the head
 * stride of taco_attention_step's q) at most 2^21.  All of one dtype
 * unless said otherwise.  dim: a multiple of 8, 8 .. 128.  Sums, softmax statistics and states are float32.
 */
#ifndef TACO_SEQUENCE_H
#define TACO_SEQUENCE_H
#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define TACO_SEQUENCE_ABI_VERSION 2

enum { TACO_SEQ_OK = 0, TACO_SEQ_ERR_INVALID_ARG = -1, TACO_SEQ_ERR_HIP = -2, TACO_SEQ_ERR_WORKSPACE = -3 };
enum { TACO_SEQ_F32 = 0, TACO_SEQ_F16 = 1, TACO_SEQ_BF16 = 2 };

typedef struct taco_seq_tensor {   /* [tokens][heads][dim] */
    void *ptr;
    int64_t token_stride, head_stride;
} taco_seq_tensor;

int taco_sequence_abi_version(void);
const char *taco_sequence_source_hash(void);
const char *taco_sequence_last_error(void);

/* ---- Attention inside packed sequences.  o_i = sum_j P_ij v_j, P_i = softmax over j of scale * q_i . k_j; j runs over the keys of the token's own
 * sequence, up to the token itself if `causal`.  Query head h reads key-value head h / (heads / kv_heads).
 * A hidden key has no influence, whatever its row holds (NaN and infinities included).  lse[token][head] = log sum_j exp(scale * q_i . k_j).
 * The work list: tiles of `tile_rows` = 32 or 128 queries, DEVICE array of {first token of the sequence, its length, first query of the
 * tile (in the sequence), 0}, the longest first.  Rows that no tile names are neither read nor written. */
typedef struct taco_seq_tile { int32_t start, length, first, pad; } taco_seq_tile;

typedef struct taco_attention_args {
    taco_seq_tensor q, k, v, o;         /* q, o: heads; k, v: kv_heads */
    float *lse;                         /* [tokens][heads], contiguous */
    const taco_seq_tile *tiles;
    const taco_seq_tile *key_tiles;     /* backward: the same tiles in the order their keys want (most queries first), or NULL */
    int32_t n_tiles, tile_rows;
    int32_t whole;                      /* backward: not 0: every tile is a whole sequence, of at most tile_rows = 32 tokens (longer ones are cut off there); not
                                           for float32 with dim > 96, which is refused */
    int32_t heads, kv_heads, dim, dtype, causal;
    float scale;                        /* > 0 */
    /* backward only: */
    taco_seq_tensor d_o, d_q, d_k, d_v;
    float *delta;                       /* workspace [tokens][heads]: scale * rowsum(d_o o) */
    int32_t parts;                      /* 128-row tiles: a key-value head's group of query heads in that many parts (a divisor of heads / kv_heads), each a
                                           workgroup of its own; more than 1 needs the workspace [n_tiles][128][kv_heads][parts][2][dim rounded up to a multiple of 32] */
    float *partial;
} taco_attention_args;
int taco_attention(const taco_attention_args *a, void *stream);
/* Gradients by the formulas (P from lse; dS = P (dP - rowsum(d_o o))): two launches, the second reads `delta`, which the first writes; one launch where
 * the tiles are whole sequences (o and delta have to be given then too, but are neither read nor written). */
int taco_attention_backward(const taco_attention_args *a, void *stream);

/* ---- Attention of one new token per row over a paged cache, which the token joins.
 * Token t of row b lies in page table[b][t / page_size], slot t % page_size.  Row b's cache holds lengths[b] tokens before the call.  With k_new and
 * v_new the token becomes number lengths[b] (written into the cache) and is attended too; without (NULL), the cache is read as it is, and a row of
 * length 0 gets zeros.  lengths is not changed.  A page that several rows share may be read by all; the slot a token is written to must be one row's, and named once.
 * A row whose length is negative or leaves no room in its table, or whose table names a page outside [0, num_pages) for a token that is read, gets
 * NaN in its output; nothing outside the buffers is read or written, and the rows beside it are not touched (its own token still joins the cache
 * if that has a page and a slot). */
typedef struct taco_attention_step_args {
    taco_seq_tensor q, o;               /* [rows][heads][dim]: token_stride = the row's */
    taco_seq_tensor k_new, v_new;       /* [rows][kv_heads][dim], or both NULL */
    void *k_pages, *v_pages;            /* [num_pages][page_size][kv_heads][dim], strides in elements below */
    int64_t k_page_stride, k_token_stride, k_head_stride;
    int64_t v_page_stride, v_token_stride, v_head_stride;
    const int32_t *table;               /* [rows][table_width], rows table_stride apart */
    int64_t table_stride;
    const int32_t *lengths;             /* [rows] */
    int32_t rows, table_width, num_pages, page_size;
    int32_t heads, kv_heads, dim, dtype;
    float scale;
    void *workspace;                    /* taco_attention_step_workspace_bytes, 16-byte aligned; may be NULL if that is 0 */
    size_t workspace_bytes;
} taco_attention_step_args;
size_t taco_attention_step_workspace_bytes(const taco_attention_step_args *a);
int taco_attention_step(const taco_attention_step_args *a, void *stream);

/* ---- Linear attention with a decay for each head: S_t = g S_{t-1} + k_t v_t^T, o_t = scale * q_t S_t, g = exp(log_decay[head]).
 * state0, state_last: float32 [sequences][heads][dim][dim] (key dimension first), contiguous; NULL: zeros / not wanted.  They must not overlap.
 * The work list: DEVICE array of segments, those of one sequence behind one another in order.  A sequence of no tokens has one segment of none.
 * n_segments > n_sequences needs the workspace (float32 [n_segments][heads][dim rounded up to a multiple of 32]^2). */
typedef struct taco_seq_segment { int32_t sequence, start, length, first, count, index, pad0, pad1; } taco_seq_segment;
                        /* start, length: the sequence's tokens; first, count: the segment's, counted in the sequence; index: its number in the sequence */
typedef struct taco_linear_attention_args {
    taco_seq_tensor q, k, v, o;
    const float *log_decay;             /* [heads] */
    const float *state0;
    float *state_last;
    const taco_seq_segment *segments;
    const int32_t *first_segment;       /* [n_sequences + 1] */
    int32_t n_segments, n_sequences;
    int32_t heads, dim, dtype;
    float scale;                        /* finite, at least 2^-126 in size (the gradients' states are divided by it) */
    void *workspace;
    size_t workspace_bytes;
    /* backward only: */
    taco_seq_tensor d_o, d_q, d_k, d_v;
    const float *d_state_last;          /* or NULL */
    float *d_state0;                    /* or NULL */
} taco_linear_attention_args;
size_t taco_linear_attention_workspace_bytes(const taco_linear_attention_args *a, int backward);
int taco_linear_attention(const taco_linear_attention_args *a, void *stream);
/* The gradients are the same product with its roles exchanged: dq_t = scale (d_o, v, k), dk and dv run from the last token to the first.
 * log_decay has none. */
int taco_linear_attention_backward(const taco_linear_attention_args *a, void *stream);

/* One token per row: state[row] = g state[row] + k v^T in place (reset[row] != 0: from zeros, whatever it holds), o = scale * q state[row]. */
typedef struct taco_linear_attention_step_args {
    taco_seq_tensor q, k, v, o;         /* [rows][heads][dim] */
    const float *log_decay;
    float *state;                       /* [rows][heads][dim][dim] float32, contiguous */
    const void *reset;                  /* [rows] of reset_bytes each (1, 4 or 8), or NULL */
    int32_t reset_bytes, rows, heads, dim, dtype;
    float scale;
} taco_linear_attention_step_args;
int taco_linear_attention_step(const taco_linear_attention_step_args *a, void *stream);

#ifdef __cplusplus
}
#endif
#endif /* TACO_SEQUENCE_H */
