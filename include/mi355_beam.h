/*
 * mi355_beam.h — C ABI of the MI355X (gfx950) operators for several continuations of a
 * prompt over a paged cache: attention that reads a common prefix once, the selection
 * of beams, and the forking, compacting and copying of pages.
 *
 * Plain pointers and sizes only; no torch types cross this boundary. The library
 * never allocates device memory and never synchronises: all work is enqueued on
 * the caller's stream. Lengths, offsets, rows and page numbers are device data,
 * which the host does not read: a value outside its range hides its keys or leaves
 * its row empty, and reaches no memory outside the tensors.
 *
 * These operators have no counterpart in the reference, whose attention takes
 * contiguous K/V and a dense mask (csrc/fa/fa_fwd_op.cu:46-197); layouts of a head and
 * of the cache are those of mi355_serve.h.
 */
#ifndef MI355_BEAM_H
#define MI355_BEAM_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define MI355_BEAM_ABI_VERSION 1

/* Error codes returned by the entry points (0 = success). */
enum {
  MI355_BEAM_OK = 0,
  MI355_BEAM_EINVAL = 1,     /* argument/contract violation (message filled)         */
  MI355_BEAM_EWORKSPACE = 2, /* workspace missing or too small                       */
  MI355_BEAM_ELAUNCH = 3,    /* HIP launch error (message carries hipGetErrorString) */
  MI355_BEAM_EDEVICE = 4     /* current device is not gfx950                         */
};

/* Element types. The 16-bit tensors of an attention call share theirs. */
enum { MI355_BEAM_FP16 = 0, MI355_BEAM_BF16 = 1, MI355_BEAM_FP32 = 2 };

/*
 * Attention of one new token per request over a paged cache, of which requests share
 * prefixes. Requests cu_groups[g] .. cu_groups[g+1]-1 are group g (offsets ascend); the
 * first prefix_lens[g] keys of each are those that block_table's row of its first request
 * names, its others those of its own row. (First of those that have keys, or a page of the
 * cache in their row's first column: a row that mi355_paged_fork left empty is passed
 * over.) Requests of no group have no prefix. What is read once is the part of the prefix
 * that all requests of the group with keys see: one that is shorter than the prefix, or a
 * window that ends inside it, leaves the rest to each. Key j is row
 * j % page_size of page table[j / page_size], j < kv_lens[n]; a request's row is at its
 * last key, len - 1. Scores of key j:
 *   s = scale·q·k_j
 *   s = softcap·tanh(s / softcap)        where softcap > 0
 *   s = s − slopes[head]·(len − 1 − j)   where slopes is given
 * Seen keys: j >= len − window where window > 0, else all. O = softmax(s)·V over them; a
 * request that sees none gives 0. Keys that are not seen have no influence.
 * Layouts: q, o [b, h, d]; caches [num_pages, h_k, page_size, d]; block_table
 * [b, table_cols]; innermost stride 1, 16-byte aligned bases, other strides multiples of
 * 8 elements, the caches' row strides below 2^24. A page number outside the cache hides
 * that page's keys; kv_lens and prefix_lens past table_cols·page_size (2^30 at most) count
 * as that. Tiles of 32 keys that a table spans, for each KV head and 16 of its heads: at
 * most 2^30 of a request and 2^35 of all. Workgroups are counted: b·h stays below
 * 2^26, and h_k·n_groups + b·h / 32 about below 2^24.
 */
typedef struct mi355_shared_params {
  const void* q;
  const void* k_cache;
  const void* v_cache;
  void* o;
  const int32_t* block_table;
  const int32_t* kv_lens;     /* [b] */
  const int32_t* cu_groups;   /* [n_groups + 1] */
  const int32_t* prefix_lens; /* [n_groups] */
  const float* slopes;        /* [h], or NULL */
  int64_t q_batch_stride, q_head_stride;
  int64_t o_batch_stride, o_head_stride;
  int64_t k_page_stride, k_head_stride, k_row_stride;
  int64_t v_page_stride, v_head_stride, v_row_stride;
  int64_t table_stride;
  int32_t b, n_groups;        /* at most MI355_BEAM_MAX_REQUESTS each */
  int32_t h, h_k, d, dtype;   /* d: 64 or 128; h a multiple of h_k */
  int32_t num_pages, page_size, table_cols; /* page_size: a power of two, 8 .. 1024 */
  int32_t window;             /* 0 = none */
  float scale, softcap;
  void* workspace;            /* device memory, 16-byte aligned; contents need no clearing */
  size_t workspace_bytes;
} mi355_shared_params;

#define MI355_BEAM_MAX_REQUESTS 1024

int mi355_shared_decode(const mi355_shared_params* p, void* stream, char* err, size_t errlen);

/* Bytes of workspace mi355_shared_decode needs for these params (0 for a call that it refuses). */
size_t mi355_shared_decode_workspace_bytes(const mi355_shared_params* p);

/*
 * The selection of a step of beam search. Of n_groups searches of `beams` beams each:
 *   s[w, v] = scores[w] + x[w, v] − log Σ_v exp x[w, v]
 * formed in 64 bits, and of its beams·vocab values the k largest, in descending order; among
 * equals the lowest w first, of one w the largest logit, then the lowest v: their scores
 * (rounded to 32 bits), tokens v and parents g·beams + w. So candidates of one beam are in
 * the order of their logits, also where the score's 64 bits do not tell them apart. A
 * beam that is finished has one candidate, its own score with the token eos. A beam with
 * a score that is not finite, or whose logits hold a NaN or +infinity, has none; nor
 * has a logit of −infinity. Behind the candidates there are, outputs hold −infinity, −1 and −1.
 * Layouts: logits [n_groups, beams, vocab], innermost stride 1; others contiguous.
 */
typedef struct mi355_select_params {
  const void* logits;
  const float* scores;        /* [n_groups, beams] */
  const uint8_t* finished;    /* [n_groups, beams], 0 or 1, or NULL */
  float* out_scores;          /* [n_groups, k] */
  int32_t* out_tokens;
  int32_t* out_parents;
  int64_t group_stride, beam_stride; /* of logits, in elements, not negative */
  int32_t n_groups, beams, vocab, k; /* beams 1 .. 256, k 1 .. 64; beams·vocab < 2^31, n_groups·beams < 2^24 */
  int32_t eos;                /* 0 .. vocab − 1 where finished is given */
  int32_t dtype;
  void* workspace;            /* device memory, 16-byte aligned; contents need no clearing */
  size_t workspace_bytes;
} mi355_select_params;

int mi355_beam_select(const mi355_select_params* p, void* stream, char* err, size_t errlen);
size_t mi355_beam_select_workspace_bytes(const mi355_select_params* p);

/*
 * Rows of a page table for the children of requests. Row i of the new table continues
 * row parents[i] of the old one, with its length; a parent outside 0 .. n-1 leaves the
 * row empty (length 0), and a row without children is freed. A row holds
 * ceil(len / page_size) pages; entries outside 0 .. num_pages-1 become -1. Whole pages
 * are shared. A last page that is partly filled, into which the next token will be
 * written, stays with the lowest new row that has it so, if no row has it as a whole one
 * and it is not held; the other rows get a free page each, in order, and (src, dst) says
 * what has to be copied. Free: pages that no new row has and that are not in `held`.
 *   table [r, table_cols], lens [r], src, dst [r] (-1 where there is nothing to copy)
 *   free_pages [num_pages]: the pages left, ascending, -1 behind them
 *   counts = {free pages left, pages copied, pages wanted and not had}
 * A row without a page for its last tokens has -1 there.
 */
typedef struct mi355_fork_params {
  const int32_t* block_table; /* [n, table_cols] */
  const int32_t* seq_lens;    /* [n]; counted as 0 .. table_cols·page_size */
  const int32_t* parents;     /* [r] */
  const int32_t* held;        /* [n_held] page numbers, or NULL */
  int32_t* table;             /* [r, table_cols], contiguous */
  int32_t* lens;
  int32_t* src;
  int32_t* dst;
  int32_t* free_pages;        /* [num_pages] */
  int32_t* counts;            /* [3] */
  int64_t table_stride;       /* of block_table */
  int32_t n, r, table_cols, num_pages, page_size, n_held; /* r at most MI355_BEAM_MAX_ROWS, num_pages at most
                                                             MI355_BEAM_MAX_PAGES, page_size >= 1, table_cols <= 2^30 */
  void* workspace;            /* device memory, 16-byte aligned; contents need no clearing */
  size_t workspace_bytes;
} mi355_fork_params;

#define MI355_BEAM_MAX_ROWS 4096
#define MI355_BEAM_MAX_PAGES (1 << 19)

int mi355_paged_fork(const mi355_fork_params* p, void* stream, char* err, size_t errlen);
size_t mi355_paged_fork_workspace_bytes(const mi355_fork_params* p);

/*
 * Moves the pages in use to the front of a cache: of u pages that rows have or that are
 * in `held`, the j-th numbered u or more moves to the j-th free one below u.
 *   table [n, table_cols]: the rows' pages by their new numbers, -1 elsewhere
 *   src, dst [num_pages / 2]: the moves, -1 behind them
 *   remap [num_pages]: the new number of each page in use, -1 of the others
 *   free_pages [num_pages]: u, u + 1, ..; -1 behind them
 *   counts = {pages in use, pages moved}
 */
typedef struct mi355_compact_params {
  const int32_t* block_table; /* [n, table_cols] */
  const int32_t* seq_lens;    /* [n] */
  const int32_t* held;        /* [n_held], or NULL */
  int32_t* table;             /* [n, table_cols], contiguous */
  int32_t* src;
  int32_t* dst;
  int32_t* remap;
  int32_t* free_pages;
  int32_t* counts;            /* [2] */
  int64_t table_stride;
  int32_t n, table_cols, num_pages, page_size, n_held; /* as above; n at most MI355_BEAM_MAX_ROWS */
  void* workspace;
  size_t workspace_bytes;
} mi355_compact_params;

int mi355_paged_compact(const mi355_compact_params* p, void* stream, char* err, size_t errlen);
size_t mi355_paged_compact_workspace_bytes(const mi355_compact_params* p);

/*
 * Copies pages src[i] to dst[i] of both caches [num_pages, h_k, page_size, d] (strides as
 * above). A pair with a number outside the cache copies nothing. The dst of a call are
 * distinct and none of them is a src of it, or it is not defined what their pages hold.
 */
typedef struct mi355_copy_params {
  void* k_cache;
  void* v_cache;
  const int32_t* src;         /* [n] */
  const int32_t* dst;         /* [n] */
  int64_t k_page_stride, k_head_stride, k_row_stride;
  int64_t v_page_stride, v_head_stride, v_row_stride;
  int32_t n, num_pages, h_k, page_size, d; /* d: 64 or 128; 16-bit elements; a page of 2^27 elements at most */
} mi355_copy_params;

int mi355_paged_copy(const mi355_copy_params* p, void* stream, char* err, size_t errlen);

int mi355_beam_abi_version(void);

#ifdef __cplusplus
}
#endif

#endif /* MI355_BEAM_H */
