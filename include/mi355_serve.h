/*
 * mi355_serve.h — C ABI of the MI355X (gfx950) serving operators: attention over
 * packed sequences, one-token attention over a paged key-value cache, rotary
 * positions with the write into that cache, and the cache's layout.
 *
 * Plain pointers and sizes only; no torch types cross this boundary. The library
 * never allocates device memory and never synchronises: all work is enqueued on
 * the caller's stream. Lengths, offsets, page and slot numbers are device data,
 * which the host does not read: a value outside its range leaves its keys unseen
 * or its rows unwritten, and reaches no memory outside the tensors.
 *
 * These operators have no counterpart in the reference, whose attention takes
 * contiguous K/V and a dense mask (csrc/fa/fa_fwd_op.cu:46-197); names, layouts
 * of a head and the handling of rows that see nothing follow that operator.
 */
#ifndef MI355_SERVE_H
#define MI355_SERVE_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define MI355_SERVE_ABI_VERSION 1

/* Error codes returned by the entry points (0 = success). */
enum {
  MI355_SERVE_OK = 0,
  MI355_SERVE_EINVAL = 1,     /* argument/contract violation (message filled)         */
  MI355_SERVE_EWORKSPACE = 2, /* workspace missing or too small                       */
  MI355_SERVE_ELAUNCH = 3,    /* HIP launch error (message carries hipGetErrorString) */
  MI355_SERVE_EDEVICE = 4     /* current device is not gfx950                         */
};

/* Element type of the 16-bit tensors of a call (they share it). */
enum { MI355_SERVE_FP16 = 0, MI355_SERVE_BF16 = 1 };

/*
 * The scores of both attention operators, of row i and key j of one sequence,
 * i and j its positions (the last row is at the last key):
 *   s = scale·q_i·k_j
 *   s = softcap·tanh(s / softcap)        where softcap > 0
 *   s = s − slopes[head]·|i − j|         where slopes is given
 * Seen keys: j <= i where causal (always, for one token); |i − j| < window where
 * window > 0; and, whatever those say, the first prefix_lens[sequence] keys.
 * O = softmax(s over the seen keys)·V; a row that sees none gives 0. Keys that a
 * row does not see have no influence on it, whatever they hold. (Where one holds a
 * V that is not finite, a column of the row can round differently in the last place.)
 */

/*
 * Attention over packed sequences. Rows cu_q[n] .. cu_q[n+1]-1 of q and o, and
 * cu_k[n] .. cu_k[n+1]-1 of k and v, are sequence n; offsets ascend. Rows of o in
 * no sequence are set to 0. Layouts: q, o [total_q, h, d]; k, v [total_k, h_k, d];
 * innermost stride 1, 16-byte aligned bases, other strides multiples of 8 elements,
 * token strides below 2^24 and, of v and o with more than one token, at least d.
 */
typedef struct mi355_packed_params {
  const void* q;
  const void* k;
  const void* v;
  void* o;
  const int32_t* cu_q;        /* [n_seqs + 1] */
  const int32_t* cu_k;        /* [n_seqs + 1] */
  const int32_t* prefix_lens; /* [n_seqs], or NULL */
  const float* slopes;        /* [h], or NULL */
  int64_t q_token_stride, q_head_stride;
  int64_t k_token_stride, k_head_stride;
  int64_t v_token_stride, v_head_stride;
  int64_t o_token_stride, o_head_stride;
  int32_t total_q, total_k, n_seqs;
  int32_t h, h_k, d;          /* d: 64 or 128; h a multiple of h_k */
  int32_t dtype;
  int32_t causal;             /* 0 or 1 */
  int32_t window;             /* 0 = none */
  float scale;                /* > 0 */
  float softcap;              /* 0 = none */
} mi355_packed_params;

int mi355_packed_fwd(const mi355_packed_params* p, void* stream, char* err, size_t errlen);

/*
 * Attention of one new token per request over a paged cache: request n's key j is
 * row j % page_size of page block_table[n][j / page_size], j < kv_lens[n]; its row
 * is at the last key. Layouts: q, o [b, h, d]; caches [num_pages, h_k, page_size, d]
 * (strides as above); block_table [b, table_cols]. A page number outside the cache
 * hides that page's keys; kv_lens past table_cols·page_size (2^30 at most) count as that.
 */
typedef struct mi355_decode_params {
  const void* q;
  const void* k_cache;
  const void* v_cache;
  void* o;
  const int32_t* block_table;
  const int32_t* kv_lens;
  const float* slopes;        /* [h], or NULL */
  int64_t q_batch_stride, q_head_stride;
  int64_t o_batch_stride, o_head_stride;
  int64_t k_page_stride, k_head_stride, k_row_stride;
  int64_t v_page_stride, v_head_stride, v_row_stride;
  int64_t table_stride;
  int32_t b, h, h_k, d, dtype;
  int32_t num_pages, page_size, table_cols; /* page_size: a power of two, 8 .. 1024 */
  int32_t window;
  float scale, softcap;
  void* workspace;            /* device memory, 16-byte aligned; contents need no clearing */
  size_t workspace_bytes;
} mi355_decode_params;

int mi355_paged_decode(const mi355_decode_params* p, void* stream, char* err, size_t errlen);

/* Bytes of workspace mi355_paged_decode needs for these params (the joined
 * parts of sequences that several workgroups share; 0 when none). */
size_t mi355_paged_decode_workspace_bytes(const mi355_decode_params* p);

/*
 * Rotary positions of q and k, and the write of k and v into a paged cache. Pair i
 * (of rot / 2) of a head turns by positions[t]·inv_freq[i] radians, formed in 64
 * bits, and is scaled by amplitude; pairs are elements (i, i + rot/2), or
 * (2i, 2i + 1) where interleaved; elements from rot on are copied. Slot s is row
 * s % page_size of page s / page_size. A slot outside the cache stores nothing;
 * among equal slots of one call it is not defined whose elements stay.
 * Layouts: q, q_out [t, h, d]; k, v, k_out [t, h_k, d]; caches as above.
 */
typedef struct mi355_rope_params {
  const void* q;
  const void* k;
  const void* v;
  void* q_out;
  void* k_out;
  void* k_cache;
  void* v_cache;
  const int32_t* positions;   /* [t] */
  const double* inv_freq;     /* [rot / 2] */
  const int64_t* slot_map;    /* [t] */
  int64_t q_token_stride, q_head_stride;
  int64_t k_token_stride, k_head_stride;
  int64_t v_token_stride, v_head_stride;
  int64_t qo_token_stride, qo_head_stride;
  int64_t ko_token_stride, ko_head_stride;
  int64_t kc_page_stride, kc_head_stride, kc_row_stride;
  int64_t vc_page_stride, vc_head_stride, vc_row_stride;
  int32_t t, h, h_k, d, dtype;
  int32_t rot;                /* a multiple of 16, 0 .. d */
  int32_t interleaved;        /* 0 or 1 */
  int32_t num_pages, page_size;
  float amplitude;
} mi355_rope_params;

int mi355_rope_paged_store(const mi355_rope_params* p, void* stream, char* err, size_t errlen);

/*
 * Page tables and slots of one step: request r holds seq_lens[r] tokens and gets
 * new_lens[r] more. It holds ceil(seq/page) pages and needs ceil((seq + new)/page),
 * at most table_cols; requests take the difference from free_pages in order of r.
 *   kv_lens[r] = seq + new             cu_new[r] = sum of new before r (n + 1 of them)
 *   table[r]   = the pages held (as in block_table), then those taken; -1 behind
 *                them and where free_pages ran out
 *   positions[t], slot_map[t]: of new token t of all requests in order; 0 and -1
 *                behind the last; slot -1 where the token has no page
 *   counts = {new tokens, pages taken, pages wanted and not had}
 * Negative lengths count as 0. Sums of lengths stay below 2^31.
 */
typedef struct mi355_layout_params {
  const int32_t* seq_lens;
  const int32_t* new_lens;
  const int32_t* block_table; /* [n, table_cols] */
  const int32_t* free_pages;  /* [n_free] */
  int32_t* kv_lens;           /* [n] */
  int32_t* cu_new;            /* [n + 1] */
  int32_t* positions;         /* [max_tokens] */
  int64_t* slot_map;          /* [max_tokens] */
  int32_t* table;             /* [n, table_cols], contiguous */
  int32_t* counts;            /* [3] */
  int64_t table_stride;       /* of block_table */
  int32_t n, table_cols, n_free, page_size, max_tokens; /* page_size >= 1, table_cols <= 2^30 */
} mi355_layout_params;

#define MI355_SERVE_MAX_REQUESTS 8192 /* n of mi355_paged_layout */

int mi355_paged_layout(const mi355_layout_params* p, void* stream, char* err, size_t errlen);

int mi355_serve_abi_version(void);

#ifdef __cplusplus
}
#endif

#endif /* MI355_SERVE_H */
