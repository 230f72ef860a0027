// serve.hip — the serving operators for MI355X (gfx950 / CDNA4): attention over
// packed sequences, one-token attention over a paged key-value cache, rotary
// positions with the write into that cache, and the cache's layout. C ABI in
// include/mi355_serve.h; each operator's kernels and their reasons in its header.

#include <hip/hip_runtime.h>

#include <limits.h>
#include <math.h>
#include <stdarg.h>
#include <stdint.h>
#include <stdio.h>
#include <string.h>

#include <algorithm>
#include <mutex>
#include <type_traits>

#include "mi355_serve.h"
#include "gfx950.h"
#include "serve_sched.h"

namespace mi355fa {
namespace {

#include "packed_fwd.h"
#include "paged_decode.h"
#include "rope_store.h"
#include "paged_layout.h"

// ── host side ─────────────────────────────────────────────────────────────────

#include "launch.h"

// f(integral_constant...) for the runtime values of (cap, bias)
template <class F> void by_scores(bool cap, bool bias, F f) {
  if (cap) bias ? f(std::true_type{}, std::true_type{}) : f(std::true_type{}, std::false_type{});
  else bias ? f(std::false_type{}, std::true_type{}) : f(std::false_type{}, std::false_type{});
}

constexpr int kMaxRows = 1 << 30;
constexpr int64_t kMaxRowStride = 1 << 24;   // 64 rows of it stay below 2^31 bytes

int packed_fwd(const mi355_packed_params* p, hipStream_t st, const Err& err) {
  if (!p) return err.fail(MI355_SERVE_EINVAL, "params must not be NULL");
  if (int rc = check_heads(err, p->h, p->h_k, p->d, p->dtype)) return rc;
  if (p->total_q < 0 || p->total_k < 0 || p->n_seqs < 0 || p->total_q > kMaxRows || p->total_k > kMaxRows || p->n_seqs > kMaxRows)
    return err.fail(MI355_SERVE_EINVAL, "total_q, total_k and n_seqs must be in 0 .. 2^30");
  if (!window_ok(p->window)) return err.fail(MI355_SERVE_EINVAL, "window must be 0 (none) or positive");
  PackedArgs a{};
  if (!score_factors(a, p->scale, p->softcap)) return err.fail(MI355_SERVE_EINVAL, "%s", kScoresText);
  if (p->total_q == 0 || p->h == 0) return MI355_SERVE_OK;
  if (!p->q || !p->o || !p->cu_q || !p->cu_k || (p->total_k > 0 && (!p->k || !p->v)))
    return err.fail(MI355_SERVE_EINVAL, "tensor pointer is NULL");
  if (!rows_ok(p->q, {p->q_token_stride, p->q_head_stride}) || !rows_ok(p->k, {p->k_token_stride, p->k_head_stride}) ||
      !rows_ok(p->v, {p->v_token_stride, p->v_head_stride}) || !rows_ok(p->o, {p->o_token_stride, p->o_head_stride}))
    return err.fail(MI355_SERVE_EINVAL, "q/k/v/o must be 16-byte aligned with strides that are multiples of 8 elements");
  for (int64_t s : {p->q_token_stride, p->k_token_stride, p->v_token_stride, p->o_token_stride})
    if (s < 0 || s >= kMaxRowStride) return err.fail(MI355_SERVE_EINVAL, "token strides must be in 0 .. 2^24 elements");
  // (a tile's rows behind the last key must lie behind the last row's end)
  if (p->total_k > 1 && p->v_token_stride < p->d) return err.fail(MI355_SERVE_EINVAL, "v's rows must not overlap: its token stride must be at least d");
  // (a wave stores 32 rows: those behind a sequence's last must lie behind that row's end)
  if (p->total_q > 1 && p->o_token_stride < p->d) return err.fail(MI355_SERVE_EINVAL, "o's rows must not overlap: its token stride must be at least d");
  const Device dev = device_info();
  if (!dev.gfx950) return err.fail(MI355_SERVE_EDEVICE, "mi355_serve: current HIP device is not gfx950 (MI355X)");

  a.q = (const uint16_t*)p->q; a.k = (const uint16_t*)p->k; a.v = (const uint16_t*)p->v; a.o = (uint16_t*)p->o;
  if (p->softcap > 0.f) {
    // (tanh z) / 2 = k·u·(c0 + c1·z² + ..) / 2 with z = k·u; powers of a k below 10^-5 would underflow
    const double c[4] = {0.999999464, -0.3332637607, 0.1319091244, -0.04441858165}, k = (double)p->scale / p->softcap;
    for (int i = 0; i < 4; ++i) a.tanh_p[i] = (float)(0.5 * c[i] * pow(k, 2 * i + 1));
    a.tanh_lim = k >= 1e-5 && k <= 1e5 ? (float)(0.5 / k) : -1.f;
  }
  a.cu_q = p->cu_q; a.cu_k = p->cu_k; a.prefix = p->prefix_lens; a.slopes = p->slopes;
  a.q_ts = p->q_token_stride; a.q_hs = p->q_head_stride; a.k_ts = p->k_token_stride; a.k_hs = p->k_head_stride;
  a.v_ts = p->total_k > 1 ? p->v_token_stride : p->d;   // (never stepped over)
  a.v_hs = p->v_head_stride;
  a.o_ts = p->total_q > 1 ? p->o_token_stride : p->d;
  a.o_hs = p->o_head_stride;
  a.tq = p->total_q; a.tk = p->total_k; a.n = p->n_seqs; a.h = p->h; a.ratio = p->h / p->h_k;
  a.causal = p->causal != 0; a.window = window_of(p->window);
  // A workgroup's shape: 4 waves of 32 rows (two workgroups on a CU); 8 waves, 4 of rows
  // by 2 groups that take every other key tile; 2 by 4; or 2 by 2. More groups make
  // shorter chains of tiles, fewer rows more workgroups, which read K and V more often.
  // By the workgroups that 256 rows each would make (us for the four shapes, bf16, 16/4
  // heads, d = 128; * chosen):
  //   more than CUs: 8192 tokens 266* / 290 / 419 / 457; 24 documents, 8000 tokens
  //     42* / 63 / 107 / 102; 8 documents, 4000 tokens 35* / 42 / 68 / 66
  //   up to CUs: 4000 tokens 95 / 82* / 121 / 127; 2000 tokens 46 / 38* / 45 / 44
  //   a quarter: 4000 tokens, 4 heads 79 / 61 / 52* / 55; 500 tokens 16 / 16 / 14 / 14*;
  //     100 tokens, 8 heads 9.0 / 9.9 / 9.9 / 8.9*
  // d = 64 keeps two 8-wave workgroups on a CU: 8000 tokens 162 / 163* / 248 / 198, 24
  // documents of 8 heads 28 / 24* / 44 / 27.
  const int64_t full = (((int64_t)p->total_q + 255) / 256 + p->n_seqs / 2) * p->h;
  enum { k4x1, k4x2, k2x4, k2x2 };
  const int shape = full <= dev.cus / 4 ? (p->total_k / std::max(p->n_seqs, 1) > 512 ? k2x4 : k2x2)
                    : p->d == 64 || full <= dev.cus ? k4x2 : k4x1;
  const int rows = shape == k4x1 || shape == k4x2 ? 128 : 64;
  // Heads that share a KV head share a workgroup: the same keys for fewer rows of a
  // sequence, so short ones waste less (100 documents, 8000 tokens: 68 us, together 32).
  a.pack = std::min(a.ratio % 4 == 0 ? 4 : a.ratio % 2 == 0 ? 2 : 1, rows / 32);
  a.bm_shift = __builtin_ctz((unsigned)(rows / a.pack));
  const int64_t blocks = ((int64_t)p->total_q >> a.bm_shift) + p->n_seqs + 2, total = blocks * (p->h / a.pack);
  a.levels = total > 2 * dev.cus ? 4 : 1;   // the order matters once workgroups wait for others
  // Two workgroups on a CU: the second ones in reverse order, so that the longest block
  // shares its CU with the shortest (24 documents, 16/4 heads, d = 128: 43.6 -> 41.2 us;
  // 4000 tokens, d = 64: 54.6 -> 50.6).
  const int heads = p->h / a.pack;
  if (shape == k4x1 || (shape == k4x2 && p->d == 64)) {
    a.fold = dev.cus % heads == 0 && total > dev.cus ? dev.cus / heads : 0;
    if (a.fold) a.levels = 4;
  }
  int rc = MI355_SERVE_OK;
  by_type(p->d, p->dtype == MI355_SERVE_BF16, [&](auto d, auto bf) {
    by_scores(p->softcap > 0.f, p->slopes != nullptr, [&](auto cap, auto bias) {
      constexpr int D = decltype(d)::value;
      constexpr bool BF = decltype(bf)::value, CAP = decltype(cap)::value, BIAS = decltype(bias)::value;
      auto go = [&](void (*kernel)(const PackedArgs), int waves) { rc = run(err, "mha_packed_fwd", kernel, total, 64 * waves, 0, st, a); };
      if (shape == k4x2) go(packed_fwd_kernel<D, BF, CAP, BIAS, 4, 2>, 8);
      else if (shape == k2x4) go(packed_fwd_kernel<D, BF, CAP, BIAS, 2, 4>, 8);
      else if (shape == k2x2) go(packed_fwd_kernel<D, BF, CAP, BIAS, 2, 2>, 4);
      else if constexpr (D == 128) go(packed_fwd_kernel<D, BF, CAP, BIAS, 4, 1>, 4);
    });
  });
  return rc;
}

struct DecodePlan {
  int groups, split, target, least;
  int64_t grid;   // workgroups, and parts at most
  size_t ml, o, bytes;   // offsets of the parts' statistics and sums in the workspace
};

DecodePlan decode_plan(const mi355_decode_params* p, int cus) {
  DecodePlan pl{};
  const int ratio = p->h / p->h_k;
  pl.groups = (ratio + kDecHeads - 1) / kDecHeads;
  const int64_t units = (int64_t)p->b * p->h_k * pl.groups;
  const int64_t tiles = ((int64_t)p->table_cols * p->page_size + kDecTile - 1) / kDecTile;
  // Parts to make, beside a remainder for each unit. Two workgroups of 4 waves are
  // resident on a CU. Few units: all parts at once, one a CU or two (any count between
  // leaves CUs unequal: [131072 keys, 32/4, 128] 256 parts 57.6 us, 320 72.4, 512 59.4;
  // [6 x <= 39725, 16/8] 464 + 48 parts 124 us, 512 + 48 146). More: several rounds of
  // small parts ([32 x <= 8192, 16/4] 384 + 128: 56.6 us, 1024 + 128: 55.0).
  pl.target = (int)(units <= 16 ? cus - units : units <= cus / 4 ? 2 * cus - units : 4 * cus);
  // A CU alone reads about 40 GB/s, so even short sequences are shared once that pays
  // for the join's launch, about 5 us: [1000 keys, 16/4, 128] 18.3 us whole, 10.3 in
  // parts of 4 tiles; [500, 8/8, 64] (16 tiles) 7.1 whole, 8.9 in parts.
  pl.least = p->d == 128 ? 4 : 8;
  // (beyond kDecMaxScan requests the scan of their lengths is no longer small)
  pl.split = tiles > 3 * pl.least && p->b <= kDecMaxScan;
  pl.grid = units;
  if (pl.split) {
    pl.grid += pl.target;
    auto up = [](size_t x) { return (x + 255) & ~(size_t)255; };
    pl.ml = up((size_t)units * 8);
    pl.o = pl.ml + up((size_t)pl.grid * kDecHeads * 8);
    pl.bytes = pl.o + (size_t)pl.grid * kDecHeads * p->d * 4;
  }
  return pl;
}

int decode_check(const mi355_decode_params* p, const Err& err) {
  if (!p) return err.fail(MI355_SERVE_EINVAL, "params must not be NULL");
  if (int rc = check_heads(err, p->h, p->h_k, p->d, p->dtype)) return rc;
  if (p->b < 0 || p->num_pages < 0 || p->table_cols < 0) return err.fail(MI355_SERVE_EINVAL, "negative dimension");
  if (p->page_size < 8 || p->page_size > 1024 || (p->page_size & (p->page_size - 1)))
    return err.fail(MI355_SERVE_EINVAL, "page_size must be a power of two in 8 .. 1024");
  if ((int64_t)p->table_cols * p->page_size > kMaxRows) return err.fail(MI355_SERVE_EINVAL, "block_table must span at most 2^30 keys");
  if (!window_ok(p->window)) return err.fail(MI355_SERVE_EINVAL, "window must be 0 (none) or positive");
  return MI355_SERVE_OK;
}

int paged_decode(const mi355_decode_params* p, hipStream_t st, const Err& err) {
  if (int rc = decode_check(p, err)) return rc;
  DecodeArgs a{};
  if (!score_factors(a, p->scale, p->softcap)) return err.fail(MI355_SERVE_EINVAL, "%s", kScoresText);
  if (p->b == 0 || p->h == 0) return MI355_SERVE_OK;
  if (!p->q || !p->o || !p->kv_lens || (p->table_cols > 0 && !p->block_table) || (p->num_pages > 0 && (!p->k_cache || !p->v_cache)))
    return err.fail(MI355_SERVE_EINVAL, "tensor pointer is NULL");
  if (!rows_ok(p->q, {p->q_batch_stride, p->q_head_stride}) || !rows_ok(p->o, {}) ||
      !rows_ok(p->k_cache, {p->k_page_stride, p->k_head_stride, p->k_row_stride}) ||
      !rows_ok(p->v_cache, {p->v_page_stride, p->v_head_stride, p->v_row_stride}))
    return err.fail(MI355_SERVE_EINVAL, "q and the caches must be 16-byte aligned with strides that are multiples of 8 elements");
  const Device dev = device_info();
  if (!dev.gfx950) return err.fail(MI355_SERVE_EDEVICE, "mi355_serve: current HIP device is not gfx950 (MI355X)");
  const DecodePlan pl = decode_plan(p, dev.cus);
  if (pl.bytes && (!p->workspace || p->workspace_bytes < pl.bytes || ((uintptr_t)p->workspace & 15)))
    return err.fail(MI355_SERVE_EWORKSPACE, "workspace of %zu bytes needed (16-byte aligned), got %zu", pl.bytes, p->workspace_bytes);
  a.q = (const uint16_t*)p->q; a.k = (const uint16_t*)p->k_cache; a.v = (const uint16_t*)p->v_cache; a.o = (uint16_t*)p->o;
  a.table = p->block_table; a.lens = p->kv_lens; a.slopes = p->slopes;
  a.q_bs = p->q_batch_stride; a.q_hs = p->q_head_stride; a.o_bs = p->o_batch_stride; a.o_hs = p->o_head_stride;
  a.kp = p->k_page_stride; a.kh = p->k_head_stride; a.kr = p->k_row_stride;
  a.vp = p->v_page_stride; a.vh = p->v_head_stride; a.vr = p->v_row_stride; a.ts = p->table_stride;
  a.b = p->b; a.h = p->h; a.hk = p->h_k; a.ratio = p->h / p->h_k; a.groups = pl.groups;
  a.pages = p->num_pages; a.shift = __builtin_ctz((unsigned)p->page_size);
  a.cols = p->num_pages > 0 ? p->table_cols : 0;   // no pages: nothing is seen
  a.window = window_of(p->window);
  a.split = pl.split; a.target = pl.target; a.least = pl.least;
  a.rec = (int*)p->workspace;
  a.part_ml = (float*)((char*)p->workspace + pl.ml);
  a.part_o = (float*)((char*)p->workspace + pl.o);
  const int64_t total = pl.grid;
  int rc = MI355_SERVE_OK;
  by_type(p->d, p->dtype == MI355_SERVE_BF16, [&](auto d, auto bf) {
    constexpr int D = decltype(d)::value;
    constexpr bool BF = decltype(bf)::value;
    by_scores(p->softcap > 0.f, p->slopes != nullptr, [&](auto cap, auto bias) {
      rc = run(err, "mha_paged_decode", paged_decode_kernel<D, BF, decltype(cap)::value, decltype(bias)::value, kDecWaves>, total, 64 * kDecWaves, 0, st, a);
    });
    if (rc == MI355_SERVE_OK && pl.split) rc = run(err, "mha_paged_decode (join)", paged_join_kernel<D, BF>, (int64_t)p->b * p->h, 256, 0, st, a);
  });
  return rc;
}

int rope_store(const mi355_rope_params* p, hipStream_t st, const Err& err) {
  if (!p) return err.fail(MI355_SERVE_EINVAL, "params must not be NULL");
  if (int rc = check_heads(err, p->h, p->h_k, p->d, p->dtype)) return rc;
  // (a workgroup counts its token's 16-element units in 32 bits)
  if ((int64_t)p->h + 2 * (int64_t)p->h_k > (1 << 27)) return err.fail(MI355_SERVE_EINVAL, "at most 2^27 heads of q, k and v together");
  if (p->t < 0 || p->num_pages < 0 || p->t > kMaxRows) return err.fail(MI355_SERVE_EINVAL, "t and num_pages must be in 0 .. 2^30");
  if (p->rot < 0 || p->rot > p->d || p->rot % 16) return err.fail(MI355_SERVE_EINVAL, "rot must be a multiple of 16 in 0 .. head_dim");
  if (p->page_size < 1) return err.fail(MI355_SERVE_EINVAL, "page_size must be positive");
  if (!std::isfinite(p->amplitude)) return err.fail(MI355_SERVE_EINVAL, "amplitude must be finite");
  if (p->t == 0) return MI355_SERVE_OK;
  if (!p->q || !p->k || !p->v || !p->q_out || !p->k_out || !p->positions || !p->slot_map || (p->rot > 0 && !p->inv_freq) ||
      (p->num_pages > 0 && (!p->k_cache || !p->v_cache)))
    return err.fail(MI355_SERVE_EINVAL, "tensor pointer is NULL");
  if (!rows_ok(p->q, {p->q_token_stride, p->q_head_stride}) || !rows_ok(p->k, {p->k_token_stride, p->k_head_stride}) ||
      !rows_ok(p->v, {p->v_token_stride, p->v_head_stride}) || !rows_ok(p->q_out, {p->qo_token_stride, p->qo_head_stride}) ||
      !rows_ok(p->k_out, {p->ko_token_stride, p->ko_head_stride}) ||
      !rows_ok(p->k_cache, {p->kc_page_stride, p->kc_head_stride, p->kc_row_stride}) ||
      !rows_ok(p->v_cache, {p->vc_page_stride, p->vc_head_stride, p->vc_row_stride}))
    return err.fail(MI355_SERVE_EINVAL, "q/k/v, outputs and caches must be 16-byte aligned with strides that are multiples of 8 elements");
  if (!device_info().gfx950) return err.fail(MI355_SERVE_EDEVICE, "mi355_serve: current HIP device is not gfx950 (MI355X)");
  RopeArgs a{};
  a.q = (const uint16_t*)p->q; a.k = (const uint16_t*)p->k; a.v = (const uint16_t*)p->v;
  a.qo = (uint16_t*)p->q_out; a.ko = (uint16_t*)p->k_out; a.kc = (uint16_t*)p->k_cache; a.vc = (uint16_t*)p->v_cache;
  a.positions = p->positions; a.inv_freq = p->inv_freq; a.slots = p->slot_map;
  a.q_ts = p->q_token_stride; a.q_hs = p->q_head_stride; a.k_ts = p->k_token_stride; a.k_hs = p->k_head_stride;
  a.v_ts = p->v_token_stride; a.v_hs = p->v_head_stride; a.qo_ts = p->qo_token_stride; a.qo_hs = p->qo_head_stride;
  a.ko_ts = p->ko_token_stride; a.ko_hs = p->ko_head_stride;
  a.kc_ps = p->kc_page_stride; a.kc_hs = p->kc_head_stride; a.kc_rs = p->kc_row_stride;
  a.vc_ps = p->vc_page_stride; a.vc_hs = p->vc_head_stride; a.vc_rs = p->vc_row_stride;
  a.num_slots = (int64_t)p->num_pages * p->page_size;
  a.t = p->t; a.h = p->h; a.hk = p->h_k; a.rot = p->rot; a.page = p->page_size; a.amplitude = p->amplitude;
  int rc = MI355_SERVE_OK;
  by_type(p->d, p->dtype == MI355_SERVE_BF16, [&](auto d, auto bf) {
    constexpr int D = decltype(d)::value;
    constexpr bool BF = decltype(bf)::value;
    rc = run(err, "rope_paged_store", p->interleaved ? rope_store_kernel<D, BF, true> : rope_store_kernel<D, BF, false>, p->t, 256, 0, st, a);
  });
  return rc;
}

int paged_layout(const mi355_layout_params* p, hipStream_t st, const Err& err) {
  if (!p) return err.fail(MI355_SERVE_EINVAL, "params must not be NULL");
  if (p->n < 0 || p->n > MI355_SERVE_MAX_REQUESTS) return err.fail(MI355_SERVE_EINVAL, "at most %d requests", MI355_SERVE_MAX_REQUESTS);
  if (p->table_cols < 0 || p->n_free < 0 || p->max_tokens < 0) return err.fail(MI355_SERVE_EINVAL, "negative dimension");
  // (a wave steps over a row of the table with 32-bit columns)
  if (p->table_cols > kMaxRows) return err.fail(MI355_SERVE_EINVAL, "block_table must have at most 2^30 columns");
  if (p->page_size < 1) return err.fail(MI355_SERVE_EINVAL, "page_size must be positive");
  if (!p->cu_new || !p->counts || (p->n > 0 && (!p->seq_lens || !p->new_lens || !p->kv_lens)) ||
      (p->n > 0 && p->table_cols > 0 && (!p->block_table || !p->table)) || (p->n_free > 0 && !p->free_pages) ||
      (p->max_tokens > 0 && (!p->positions || !p->slot_map)))
    return err.fail(MI355_SERVE_EINVAL, "tensor pointer is NULL");
  const Device dev = device_info();
  if (!dev.gfx950) return err.fail(MI355_SERVE_EDEVICE, "mi355_serve: current HIP device is not gfx950 (MI355X)");
  LayoutArgs a{};
  a.seq = p->seq_lens; a.fresh = p->new_lens; a.table_in = p->block_table; a.free_pages = p->free_pages;
  a.kv_lens = p->kv_lens; a.cu = p->cu_new; a.positions = p->positions; a.slots = p->slot_map; a.table = p->table; a.counts = p->counts;
  a.ts = p->table_stride; a.n = p->n; a.cols = p->table_cols; a.n_free = p->n_free; a.page = p->page_size; a.max_tokens = p->max_tokens;
  // a wave for each row of the table, a thread for each token
  const int64_t items = std::max((int64_t)p->n * 64, (int64_t)p->max_tokens);
  const int64_t wgs = std::max<int64_t>(1, std::min<int64_t>((items + kLayoutThreads - 1) / kLayoutThreads, dev.cus));
  return run(err, "paged_layout", paged_layout_kernel, wgs, kLayoutThreads, (size_t)(2 * p->n + 1) * 4, st, a);
}

}  // namespace
}  // namespace mi355fa

extern "C" {

int mi355_serve_abi_version(void) { return MI355_SERVE_ABI_VERSION; }

int mi355_packed_fwd(const mi355_packed_params* p, void* stream, char* err, size_t errlen) {
  return mi355fa::packed_fwd(p, (hipStream_t)stream, {err, errlen});
}

size_t mi355_paged_decode_workspace_bytes(const mi355_decode_params* p) {
  if (mi355fa::decode_check(p, {nullptr, 0}) || p->b == 0 || p->h == 0) return 0;
  return mi355fa::decode_plan(p, mi355fa::device_info().cus).bytes;
}

int mi355_paged_decode(const mi355_decode_params* p, void* stream, char* err, size_t errlen) {
  return mi355fa::paged_decode(p, (hipStream_t)stream, {err, errlen});
}

int mi355_rope_paged_store(const mi355_rope_params* p, void* stream, char* err, size_t errlen) {
  return mi355fa::rope_store(p, (hipStream_t)stream, {err, errlen});
}

int mi355_paged_layout(const mi355_layout_params* p, void* stream, char* err, size_t errlen) {
  return mi355fa::paged_layout(p, (hipStream_t)stream, {err, errlen});
}

}  // extern "C"
