/*
 * afa_sm100_ops.h -- C ABI of the operators around a 4-bit key/value cache on
 * B200 (sm_100a), in the same library as the attention forward
 * (libafa_sm100.so): rotary positions with several axes, quantising keys and
 * values as they are written to a paged cache, reading them back, and
 * attention over the cache.  None of them has a counterpart in the reference,
 * whose only operation is the dense forward.
 *
 * As in afa_sm100.h: plain C types, device pointers, a cudaStream_t passed as
 * void*; no call allocates, frees or synchronises; every entry point returns
 * an AFA_* code, checks its arguments before any CUDA call and never throws.
 * Every wait for a barrier inside a kernel is bounded, as there; the allocation
 * of tensor memory waits as long as kernels of other streams hold it.
 *
 * The cache.  One uint8 array [n_pages][n_kv_heads][2][page_size][row] (index
 * 2: keys, values), row = head_dim / 2 + head_dim / 16 bytes: 36 at head_dim
 * 64, 72 at 128.  Pages may lie page_stride bytes apart; the rest is dense.  A
 * row is one token of one head: head_dim / 2 bytes of codes (byte j: channel
 * 2j in its low half, 2j + 1 in its high half), then for each group of 64
 * channels a step s and a minimum m, 16 bits each in the call's dtype.  A code
 * c stands for s * c + m.  Token t of sequence b is at place t % page_size of
 * page page_table[b][t / page_size].
 */
#ifndef AFA_SM100_OPS_H_
#define AFA_SM100_OPS_H_

#include <stdint.h>

#include "afa_sm100.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Element types of rotary positions. */
#define AFA_POS_INT32 0
#define AFA_POS_INT64 1
#define AFA_POS_FP32 2
#define AFA_ROTARY_MAX_AXES 8
#define AFA_ROTARY_MAX_HEADS 8192 /* n_heads + n_k_heads */

/* Device status words of the cache operators (AfaCache4.status; plain stores,
 * as for afa_fwd_sm100).  What the faulty entry names is skipped: nothing out
 * of bounds is read or written, and outputs that depend on it are undefined. */
#define AFA_DEV_BAD_PAGE 0x201   /* a page_table entry in use is not in [0, n_pages) */
#define AFA_DEV_BAD_LENGTH 0x202 /* kv_lens or new_lens negative or too large */

/* Rotary positions with several axes.  Pair j of a row (rot_dim / 2 pairs) is
 * turned by the angle  positions[axis(j)][b][n] * inv_freq[j], formed in 64
 * bits; the first sections[0] pairs belong to axis 0, the next sections[1] to
 * axis 1 and so on.  Pair j is channels (j, j + rot_dim / 2), or (2j, 2j + 1)
 * with `interleaved`; (a, b) becomes (a cos - b sin, b cos + a sin).  Channels
 * from rot_dim on are copied.  `inverse` turns back, which is the operator's
 * gradient.  q_out may be q and k_out may be k (the same strides); any other
 * overlap of inputs and outputs is undefined.
 * head_dim and rot_dim: multiples of 16, 16 <= rot_dim <= head_dim <= 512. */
typedef struct AfaRotaryArgs {
  const void* q; /* [batch, seq_len, n_heads, head_dim] */
  const void* k; /* [batch, seq_len, n_k_heads, head_dim], or NULL */
  void* q_out;
  void* k_out;
  int64_t q_strides[3]; /* elements: batch, seq, head; head_dim contiguous */
  int64_t k_strides[3];
  int64_t q_out_strides[3];
  int64_t k_out_strides[3];
  const void* positions;  /* [n_axes, batch, seq_len], AFA_POS_* */
  int64_t pos_strides[3]; /* elements: axis, batch, seq; 0 repeats */
  const float* inv_freq;  /* [rot_dim / 2], contiguous */
  int32_t sections[AFA_ROTARY_MAX_AXES];
  int32_t n_axes;
  int32_t pos_type;
  int32_t batch;
  int32_t seq_len;
  int32_t n_heads;
  int32_t n_k_heads; /* ignored without k */
  int32_t head_dim;
  int32_t rot_dim;
  int32_t dtype; /* AFA_DTYPE_FP16 or AFA_DTYPE_BF16 */
  int32_t interleaved;
  int32_t inverse;
} AfaRotaryArgs;

int afa_rotary_sm100(const AfaRotaryArgs* args, void* stream);

/* A paged 4-bit cache and the sequences in it, as the three cache operators
 * take it. */
typedef struct AfaCache4 {
  void* cache;               /* see the top of this file; 16-byte aligned */
  int64_t page_stride;       /* bytes from page to page, a multiple of 16 */
  const int32_t* page_table; /* [batch][max_pages] */
  int64_t table_stride;      /* elements from one sequence's row to the next */
  const int32_t* kv_lens;    /* [batch] tokens of each sequence, the new ones included */
  const int32_t* new_lens;   /* [batch] how many of the call's rows are new tokens of the
                                sequence (the others are padding), or NULL: all of them.
                                Row i < new_lens[b] is position kv_lens[b] - new_lens[b] + i.
                                With none the sequence's pages are not looked at */
  int32_t* status;           /* optional, as AfaFwdArgs.status */
  int32_t n_pages;
  int32_t page_size; /* 16, 32, 64, 128 or 256 */
  int32_t max_pages;
  int32_t batch;
  int32_t n_kv_heads;
  int32_t head_dim; /* 64 or 128 */
  int32_t dtype;    /* AFA_DTYPE_FP16 or AFA_DTYPE_BF16: of k, v, q, o and the cache's s and m */
} AfaCache4;

/* Quantises k and v [batch, seq_len, n_kv_heads, head_dim] (element strides
 * for batch, seq, head) into the cache's rows at the new positions.  For each
 * group of 64 channels: m = min(x), s = (max(x) - min(x)) / 15 rounded to
 * dtype, code = (x - m) / s rounded to the nearest integer, halves to even, at
 * most 15; 0 where s is 0.  Each rounding is that of the exact quotient.  A
 * group that holds an infinity or a NaN, or whose range passes the largest
 * fp32, gets s = m = NaN and reads back as NaN.  Padding rows are not written
 * anywhere and nothing else of the cache is written.  Two sequences of one call
 * must not write the same row (a page that is in both tables, at the same
 * place): it would be left with parts of either. */
int afa_cache4_write_sm100(const AfaCache4* cache, const void* k, const void* v, const int64_t k_strides[3],
                           const int64_t v_strides[3], int32_t seq_len, void* stream);

/* The reverse: k and v rows at the new positions become s * c + m, rounded to
 * dtype; padding rows become zero.  (A value within half a step of the type's
 * largest may round to an infinity.) */
int afa_cache4_read_sm100(const AfaCache4* cache, void* k, void* v, const int64_t k_strides[3],
                          const int64_t v_strides[3], int32_t seq_len, void* stream);

/* O = softmax(scale * Q K^T) V for queries [batch, seq_len, n_heads, head_dim]
 * over the first kv_lens[b] tokens of each sequence, K and V being s * c + m
 * unrounded.  n_heads is a multiple of n_kv_heads, grouped as in
 * afa_fwd_sm100.  causal: row i sees the tokens up to its own position
 * kv_lens[b] - new_lens[b] + i.  A row that sees no token and a padding row
 * get O = 0 and lse = -inf.  A NaN among a row's visible keys makes the row NaN,
 * one among its visible values the 64 channels of its group; a masked token does
 * nothing, whatever it holds.  Queries are exact where a row's largest element is
 * from 2^-77 to 2^110, elements down to 2^-23 of it, and to 2^-34 of it below.  A
 * token's weight times each of its values' steps is held in fp16, measured by the
 * largest such product of the row: to 2^-11 relative down to 2^-21 of that, and to
 * 2^-32 of it below.  Steps may go up to 2^100; where all of a row's lie below
 * 2^-81 they lose bits.  Calls of more than 64 query rows a key/value head
 * (seq_len * n_heads / n_kv_heads) run on tcgen05, others on mma.sync. */
typedef struct AfaCache4FwdArgs {
  const void* q;
  void* o;
  int64_t q_strides[3]; /* elements: batch, seq, head */
  int64_t o_strides[3];
  float* lse; /* optional fp32 [batch, n_heads, seq_len], contiguous, natural logarithm */
  void* workspace;         /* 16-byte aligned, afa_cache4_fwd_workspace() bytes, not shared by
                              calls that may overlap; its contents need no set-up */
  int64_t workspace_bytes;
  int32_t seq_len;
  int32_t n_heads;
  int32_t causal;
  float scale; /* <= 0 selects 1/sqrt(head_dim); below 1e38, not NaN */
  uint64_t timeout_ns; /* bound of every device-side wait; 0 selects the default (4 s) */
  uint32_t test_flags; /* 0 in normal use; AFA_TEST_PRODUCER_IDLE: in calls of more than 64 query rows a
                          key/value head nothing is loaded, and the bounded waits run out */
} AfaCache4FwdArgs;

/* Bytes of workspace a call with these sizes needs on the current device, or
 * the negative of an AFA_ERR_* code. */
int64_t afa_cache4_fwd_workspace(const AfaCache4* cache, int32_t seq_len, int32_t n_heads);

int afa_cache4_fwd_sm100(const AfaCache4* cache, const AfaCache4FwdArgs* args, void* stream);

/* Bytes of one cache row (one token, one head, keys or values), or -1. */
int32_t afa_cache4_row_bytes(int32_t head_dim);

/* Version of this header's part of the ABI (major * 100 + minor). */
int afa_sm100_ops_version(void);

#ifdef __cplusplus
} /* extern "C" */
#endif

#endif /* AFA_SM100_OPS_H_ */
