// beam.hip — the operators for several continuations of a prompt over a paged cache, for
// MI355X (gfx950 / CDNA4): attention that reads a common prefix once, the selection of
// beams, forking, compacting and copying of pages. C ABI in include/mi355_beam.h; each
// operator's kernels and their reasons in its header.

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

#include "mi355_beam.h"
#include "gfx950.h"
#include "beam_sched.h"

namespace mi355fa {
namespace {

#include "shared_decode.h"
#include "beam_select.h"
#include "page_ops.h"

// ── host side ─────────────────────────────────────────────────────────────────

#include "launch.h"

static_assert(kShMax == MI355_BEAM_MAX_REQUESTS && kPgRows == MI355_BEAM_MAX_ROWS, "limits of the C ABI");
constexpr int kMaxKeys = 1 << 30;
constexpr int64_t kMaxRowStride = 1 << 24;
constexpr int64_t kMaxGrid = 1 << 24;   // workgroups of 256 threads

int device_ok(const Err& err, Device* dev) {
  *dev = device_info();
  return dev->gfx950 ? kOk : err.fail(kEdevice, "mi355_beam: current HIP device is not gfx950 (MI355X)");
}
int workspace_ok(const Err& err, const void* ws, size_t have, size_t need) {
  if (need && (!ws || have < need || ((uintptr_t)ws & 15)))
    return err.fail(kEworkspace, "workspace of %zu bytes needed (16-byte aligned), got %zu", need, have);
  return kOk;
}
size_t up(size_t x) { return (x + 255) & ~(size_t)255; }

struct SharedPlan {
  int columns, groups, target;
  int64_t common, grid;   // parts of groups that are not whole, workgroups: at most
  int64_t own_rows, rows; // rows of partial sums: of groups' parts, and all
  size_t ml, o, bytes;    // offsets of the parts' statistics and sums in the workspace
};

SharedPlan shared_plan(const mi355_shared_params* p, int cus) {
  SharedPlan pl{};
  const int64_t ratio = p->h / p->h_k;
  pl.groups = (int)((ratio + 15) / 16);
  // Columns of a workgroup, from those that a group has of a KV head on average. Measured (d 128, 4 KV
  // heads, prefixes of 4099 keys), us a call with 32, 64, 128: 29 columns 27.9, 28.0, 29.4; 40 columns
  // 33.0, 29.8, 30.2 (120 requests) and 23.3, 23.0, 23.3 (40); 186 columns 39.9, 31.0, 31.0; 1020 of one
  // group 136.9, 55.8, 47.4.
  const int64_t mean = p->n_groups > 0 ? p->b * ratio / p->n_groups : 0;
  pl.columns = mean > 64 ? 128 : mean > 32 ? 64 : 32;
  auto per_cu = [&](auto d) {
    constexpr int D = decltype(d)::value;
    return pl.columns == 128 ? kShPerCu<D, 4, 1>() : pl.columns == 64 ? kShPerCu<D, 2, 2>() : kShPerCu<D, 1, 4>();
  };
  const int slots = cus * (p->d == 64 ? per_cu(std::integral_constant<int, 64>{}) : per_cu(std::integral_constant<int, 128>{}));
  const int64_t own = (int64_t)p->b * p->h_k * pl.groups;
  const int64_t common = pl.common = p->h_k * ((p->b * ratio + pl.columns - 1) / pl.columns + p->n_groups);
  // Workgroups that run at once, less what groups' units give in parts that are not whole: half of the most
  // (a quarter, half, all: one group of 1020 columns 54.1, 48, 49.9 us; 9 of 29 28.1, 27.9, 30.1)
  pl.target = slots - (int)(common < slots ? common / 2 : slots / 2);
  // (no more than the tables' tiles keep busy: a workgroup without any still plans)
  const int64_t most = (own + common * (pl.columns / 32)) * ((int64_t)p->table_cols * p->page_size / kDecTile + 1);
  if (most < 4 * (int64_t)pl.target) pl.target = (int)((most + 3) / 4);
  pl.grid = pl.target + common + 1;
  pl.own_rows = (common + pl.target) * pl.columns;
  pl.rows = pl.own_rows + (4 * (int64_t)(pl.target + 1) + own) * 16;
  pl.ml = up((size_t)(p->n_groups + p->b + 1) * 16);
  pl.o = pl.ml + up((size_t)pl.rows * 8);
  pl.bytes = pl.o + (size_t)pl.rows * p->d * 4;
  return pl;
}

// Whether the launches take it (they count their threads in 32 bits), and rows of sums fit theirs.
bool shared_fits(const mi355_shared_params* p, const SharedPlan& pl) {
  return pl.rows <= INT_MAX && pl.grid < kMaxGrid && (int64_t)p->b * p->h < 4 * (kMaxGrid - 1);
}

int shared_check(const mi355_shared_params* p, const Err& err) {
  if (!p) return err.fail(kEinval, "params must not be NULL");
  if (int rc = check_heads(err, p->h, p->h_k, p->d, p->dtype)) return rc;
  if (p->b < 0 || p->n_groups < 0 || p->b > kShMax || p->n_groups > kShMax) return err.fail(kEinval, "at most %d requests and groups", kShMax);
  if (p->h > (1 << 16)) return err.fail(kEinval, "at most 2^16 heads");
  if (p->num_pages < 0 || p->table_cols < 0) return err.fail(kEinval, "negative dimension");
  if (p->page_size < 8 || p->page_size > 1024 || (p->page_size & (p->page_size - 1)))
    return err.fail(kEinval, "page_size must be a power of two in 8 .. 1024");
  if ((int64_t)p->table_cols * p->page_size > kMaxKeys) return err.fail(kEinval, "block_table must span at most 2^30 keys");
  if (!window_ok(p->window)) return err.fail(kEinval, "window must be 0 (none) or positive");
  // (places of tiles among a request's are of 32 bits, and so is a workgroup's share of all)
  const int64_t tiles = (int64_t)p->table_cols * p->page_size / kDecTile + 1;
  const int64_t own = p->h > 0 ? p->h_k * (int64_t)((p->h / p->h_k + 15) / 16) * tiles : 0;
  if (own > 1 << 30 || own * p->b > (int64_t)1 << 35) return err.fail(kEinval, "too many requests, heads and keys");
  return kOk;
}

int shared_decode(const mi355_shared_params* p, hipStream_t st, const Err& err) {
  if (int rc = shared_check(p, err)) return rc;
  SharedArgs a{};
  if (!score_factors(a, p->scale, p->softcap)) return err.fail(kEinval, "%s", kScoresText);
  if (p->b == 0 || p->h == 0) return kOk;
  if (!p->q || !p->o || !p->kv_lens || !p->cu_groups || (p->n_groups > 0 && !p->prefix_lens) || (p->table_cols > 0 && !p->block_table) ||
      (p->num_pages > 0 && (!p->k_cache || !p->v_cache)))
    return err.fail(kEinval, "tensor pointer is NULL");
  if (!rows_ok(p->q, {p->q_batch_stride, p->q_head_stride}) || !rows_ok(p->o, {p->o_batch_stride, p->o_head_stride}) ||
      !rows_ok(p->k_cache, {p->k_page_stride, p->k_head_stride, p->k_row_stride}) ||
      !rows_ok(p->v_cache, {p->v_page_stride, p->v_head_stride, p->v_row_stride}))
    return err.fail(kEinval, "q, o and the caches must be 16-byte aligned with strides that are multiples of 8 elements");
  // (a lane's offset from its tile's rows is of 32 bits)
  if (p->k_row_stride < 0 || p->v_row_stride < 0 || p->k_row_stride >= kMaxRowStride || p->v_row_stride >= kMaxRowStride)
    return err.fail(kEinval, "the caches' row strides must be in 0 .. 2^24 elements");
  Device dev;
  if (int rc = device_ok(err, &dev)) return rc;
  const SharedPlan pl = shared_plan(p, dev.cus);
  if (!shared_fits(p, pl)) return err.fail(kEinval, "too many requests, groups and heads");
  if (int rc = workspace_ok(err, p->workspace, p->workspace_bytes, pl.bytes)) return rc;
  a.q = (const uint16_t*)p->q; a.k = (const uint16_t*)p->k_cache; a.v = (const uint16_t*)p->v_cache; a.o = (uint16_t*)p->o;
  a.table = p->block_table; a.lens = p->kv_lens; a.cu = p->cu_groups; a.prefix = p->prefix_lens; a.slopes = p->slopes;
  a.rec = (int*)p->workspace;
  a.part_ml = (float*)((char*)p->workspace + pl.ml);
  a.part_o = (float*)((char*)p->workspace + pl.o);
  a.q_bs = p->q_batch_stride; a.q_hs = p->q_head_stride; a.o_bs = p->o_batch_stride; a.o_hs = p->o_head_stride;
  a.kp = p->k_page_stride; a.kh = p->k_head_stride; a.kr = p->k_row_stride;
  a.vp = p->v_page_stride; a.vh = p->v_head_stride; a.vr = p->v_row_stride; a.ts = p->table_stride;
  a.b = p->b; a.n_groups = p->n_groups; a.h = p->h; a.hk = p->h_k; a.ratio = p->h / p->h_k; a.groups = pl.groups; a.columns = pl.columns; a.own_rows = (int)pl.own_rows;
  a.pages = p->num_pages; a.shift = __builtin_ctz((unsigned)p->page_size);
  a.cols = p->num_pages > 0 ? p->table_cols : 0;   // no pages: nothing is seen
  a.window = window_of(p->window);
  a.target = pl.target; a.col_shift = __builtin_ctz((unsigned)pl.columns);
  a.cap = p->softcap > 0.f;
  int rc = kOk;
  by_type(p->d, p->dtype == MI355_BEAM_BF16, [&](auto d, auto bf) {
    constexpr int D = decltype(d)::value;
    constexpr bool BF = decltype(bf)::value;
    auto go = [&](void (*kernel)(const SharedArgs)) { rc = run(err, "mha_shared_decode", kernel, pl.grid, kShThreads, 0, st, a); };
    if (pl.columns == 128) go(shared_decode_kernel<D, BF, 4, 1>);
    else if (pl.columns == 64) go(shared_decode_kernel<D, BF, 2, 2>);
    else go(shared_decode_kernel<D, BF, 1, 4>);
    if (rc != kOk) return;
    // A wave joins a row, or a workgroup where that leaves the card idle and a row has many parts (about
    // target / common). Measured, us a call by waves and by workgroups: 32 rows of 8 parts 11.7, 13.0; 640 of
    // 18 22.4, 23.0; 512 of 31 21.5, 20.3; 336 of 63 20.7, 19.9; 1072 of 3 27.8, 29.4; 4096 of 14 47.3, 55.3.
    const int64_t bh = (int64_t)p->b * p->h;
    if (bh >= 1024 || pl.target <= 24 * pl.common) rc = run(err, "mha_shared_decode (join)", shared_join_kernel<D, BF, true>, (bh + 3) / 4, 256, 0, st, a);
    else rc = run(err, "mha_shared_decode (join)", shared_join_kernel<D, BF, false>, bh, 256, 0, st, a);
  });
  return rc;
}

struct SelectPlan {
  SelectSplit split;
  size_t lists, bytes;
};

SelectPlan select_plan(const mi355_select_params* p, int cus) {
  SelectPlan pl{};
  const int64_t rows = (int64_t)p->n_groups * p->beams;
  pl.split = select_split(rows, p->beams, p->vocab, p->k, p->dtype == MI355_BEAM_FP32 ? kSelWide<float> : kSelWide<__bf16>, cus);
  pl.lists = up((size_t)rows * pl.split.parts * sizeof(SelectHead));
  pl.bytes = pl.lists + (size_t)rows * pl.split.parts * p->k * 8;
  return pl;
}

int select_check(const mi355_select_params* p, const Err& err) {
  if (!p) return err.fail(kEinval, "params must not be NULL");
  if (p->dtype != MI355_BEAM_FP16 && p->dtype != MI355_BEAM_BF16 && p->dtype != MI355_BEAM_FP32)
    return err.fail(kEinval, "logits must be float16, bfloat16 or float32");
  if (p->n_groups < 0 || p->beams < 1 || p->beams > kSelMaxBeams) return err.fail(kEinval, "beams must be in 1 .. %d", kSelMaxBeams);
  if (p->vocab < 1 || (int64_t)p->vocab * p->beams > INT_MAX || (int64_t)p->n_groups * p->beams >= kMaxGrid)
    return err.fail(kEinval, "vocab must be positive, beams·vocab below 2^31 and n_groups·beams below 2^24");
  if (p->k < 1 || p->k > kSelMaxK) return err.fail(kEinval, "k must be in 1 .. %d", kSelMaxK);
  if (p->finished && (p->eos < 0 || p->eos >= p->vocab)) return err.fail(kEinval, "eos must be a token of the vocabulary");
  if (p->group_stride < 0 || p->beam_stride < 0) return err.fail(kEinval, "logits' strides must not be negative");
  return kOk;
}

int beam_select(const mi355_select_params* p, hipStream_t st, const Err& err) {
  if (int rc = select_check(p, err)) return rc;
  if (p->n_groups == 0) return kOk;
  if (!p->logits || !p->scores || !p->out_scores || !p->out_tokens || !p->out_parents) return err.fail(kEinval, "tensor pointer is NULL");
  if ((uintptr_t)p->logits % (p->dtype == MI355_BEAM_FP32 ? 4 : 2)) return err.fail(kEinval, "logits must be aligned to their elements");
  Device dev;
  if (int rc = device_ok(err, &dev)) return rc;
  const SelectPlan pl = select_plan(p, dev.cus);
  if (int rc = workspace_ok(err, p->workspace, p->workspace_bytes, pl.bytes)) return rc;
  SelectArgs a{};
  a.x = p->logits; a.scores = p->scores; a.done = p->finished;
  a.out_s = p->out_scores; a.out_t = p->out_tokens; a.out_p = p->out_parents;
  a.heads = (SelectHead*)p->workspace;
  a.lists = (u32x2*)((char*)p->workspace + pl.lists);
  a.gs = p->group_stride; a.bs = p->beam_stride;
  a.groups = p->n_groups; a.beams = p->beams; a.vocab = p->vocab; a.k = p->k; a.eos = p->eos;
  a.parts = pl.split.parts; a.per = pl.split.per;
  const uint64_t each = (uint64_t)pl.split.parts * p->k;
  a.row_magic = each == 1 ? 0 : (uint32_t)(((1ull << 32) + each - 1) / each);
  const int64_t grid = (int64_t)p->n_groups * p->beams * pl.split.parts;
  auto go = [&](auto type) {
    typedef decltype(type) T;
    return run(err, "beam_select", pl.split.wide ? select_scan_kernel<T, kSelWide<T>> : select_scan_kernel<T, 1>, grid, kSelThreads, 0, st, a);
  };
  if (int rc = p->dtype == MI355_BEAM_FP32 ? go(float{}) : p->dtype == MI355_BEAM_BF16 ? go(__bf16{}) : go(_Float16{})) return rc;
  if (p->beams * each <= 256) return run(err, "beam_select (join)", select_join_kernel<256, 1>, p->n_groups, 256, 0, st, a);
  return run(err, "beam_select (join)", select_join_kernel<kSelJoin, kSelEach>, p->n_groups, kSelJoin, 0, st, a);
}

// What the page operators have in common.
template <class P> int pages_check(const P* p, int rows, const Err& err) {
  if (p->n < 0 || rows < 0 || rows > kPgRows) return err.fail(kEinval, "at most %d rows", kPgRows);
  if (p->table_cols < 0 || p->table_cols > kMaxKeys) return err.fail(kEinval, "block_table must have at most 2^30 columns");
  if (p->num_pages < 0 || p->num_pages > MI355_BEAM_MAX_PAGES) return err.fail(kEinval, "num_pages must be in 0 .. %d", MI355_BEAM_MAX_PAGES);
  if (p->page_size < 1) return err.fail(kEinval, "page_size must be positive");
  if (p->n_held < 0) return err.fail(kEinval, "negative dimension");
  return kOk;
}
struct PagePlan {
  int words, marks, wgs;
  bool one;   // a workgroup does it all
  size_t lds_mark, lds, bytes;
};
PagePlan page_plan(int rows, int cols, int pages, bool fork, int cus) {
  PagePlan pl{};
  pl.words = std::max(4, (pages + 127) / 128 * 4);
  // A wave a row, until the second kernel would have too many bitmaps to read (512 rows of 84000
  // pages, 32 or 16 of them: a fork, which writes its rows here, 14.9 or 16.2 us; compacting 16.8 or 15.5)
  pl.marks = std::min(std::max(1, (rows + 15) / 16), fork ? 32 : 16);
  // (each reads all bitmaps: 64 at most)
  const int64_t chunks = (int64_t)rows * ((cols + kPgColumns - 1) / kPgColumns);
  pl.wgs = (int)std::min<int64_t>(std::max<int64_t>((pages + kPgThreads * 2 - 1) / (kPgThreads * 2), fork ? 1 : (chunks + 15) / 16), std::min(64, cus));
  pl.wgs = std::max(1, pl.wgs);
  pl.one = pl.marks == 1 && pl.wgs == 1;
  pl.lds_mark = (size_t)2 * pl.words * 4;
  const size_t ranks = (size_t)pl.words * 5 + 16;
  pl.lds = (size_t)pl.words * 4 + (fork ? std::max((size_t)2 * kPgHash * 4, ranks) : ranks);
  if (pl.one && fork) pl.lds += (size_t)pl.words * 4;
  pl.bytes = pl.one ? 0 : (size_t)pl.marks * 2 * pl.words * 4;
  return pl;
}
template <class P> PageArgs page_args(const P* p, const PagePlan& pl) {
  PageArgs a{};
  a.table_in = p->block_table; a.seq = p->seq_lens; a.held = p->n_held > 0 ? p->held : nullptr;
  a.table = p->table; a.src = p->src; a.dst = p->dst; a.free_pages = p->free_pages; a.counts = p->counts;
  a.maps = (uint32_t*)p->workspace;
  a.ts = p->table_stride;
  a.n = p->n; a.r = p->n; a.cols = p->table_cols; a.pages = p->num_pages; a.page = p->page_size; a.n_held = p->held ? p->n_held : 0;
  a.words = pl.words; a.marks = pl.marks;
  return a;
}

int fork_check(const mi355_fork_params* p, const Err& err) {
  if (!p) return err.fail(kEinval, "params must not be NULL");
  return pages_check(p, p->r, err);
}
int paged_fork(const mi355_fork_params* p, hipStream_t st, const Err& err) {
  if (int rc = fork_check(p, err)) return rc;
  if (!p->counts || (p->n > 0 && !p->seq_lens) || (p->r > 0 && (!p->parents || !p->lens || !p->src || !p->dst)) ||
      (p->table_cols > 0 && ((p->n > 0 && !p->block_table) || (p->r > 0 && !p->table))) || (p->num_pages > 0 && !p->free_pages) || (p->n_held > 0 && !p->held))
    return err.fail(kEinval, "tensor pointer is NULL");
  Device dev;
  if (int rc = device_ok(err, &dev)) return rc;
  const PagePlan pl = page_plan(p->r, p->table_cols, p->num_pages, true, dev.cus);
  if (int rc = workspace_ok(err, p->workspace, p->workspace_bytes, pl.bytes)) return rc;
  PageArgs a = page_args(p, pl);
  a.parents = p->parents; a.lens = p->lens; a.r = p->r;
  if (pl.one) return run(err, "paged_fork", page_fork_kernel<true>, 1, kPgThreads, pl.lds, st, a);
  if (int rc = run(err, "paged_fork (marks)", page_mark_kernel<true>, pl.marks, kPgThreads, pl.lds_mark, st, a)) return rc;
  return run(err, "paged_fork", page_fork_kernel<false>, pl.wgs, kPgThreads, pl.lds, st, a);
}

int compact_check(const mi355_compact_params* p, const Err& err) {
  if (!p) return err.fail(kEinval, "params must not be NULL");
  return pages_check(p, p->n, err);
}
int paged_compact(const mi355_compact_params* p, hipStream_t st, const Err& err) {
  if (int rc = compact_check(p, err)) return rc;
  if (!p->counts || (p->n > 0 && !p->seq_lens) || (p->n > 0 && p->table_cols > 0 && (!p->block_table || !p->table)) ||
      (p->num_pages > 0 && (!p->remap || !p->free_pages)) || (p->num_pages > 1 && (!p->src || !p->dst)) || (p->n_held > 0 && !p->held))
    return err.fail(kEinval, "tensor pointer is NULL");
  Device dev;
  if (int rc = device_ok(err, &dev)) return rc;
  const PagePlan pl = page_plan(p->n, p->table_cols, p->num_pages, false, dev.cus);
  if (int rc = workspace_ok(err, p->workspace, p->workspace_bytes, pl.bytes)) return rc;
  PageArgs a = page_args(p, pl);
  a.remap = p->remap;
  if (pl.one) return run(err, "paged_compact", page_compact_kernel<true>, 1, kPgThreads, pl.lds, st, a);
  if (int rc = run(err, "paged_compact (marks)", page_mark_kernel<false>, pl.marks, kPgThreads, pl.lds_mark, st, a)) return rc;
  return run(err, "paged_compact", page_compact_kernel<false>, pl.wgs, kPgThreads, pl.lds, st, a);
}

int paged_copy(const mi355_copy_params* p, hipStream_t st, const Err& err) {
  if (!p) return err.fail(kEinval, "params must not be NULL");
  if (p->d != 64 && p->d != 128) return err.fail(kEinval, "Only head_dim=64 or head_dim=128 is supported");
  if (p->n < 0 || p->num_pages < 0 || p->h_k < 0 || p->page_size < 0) return err.fail(kEinval, "negative dimension");
  const int64_t units = (int64_t)p->h_k * p->page_size * (p->d / 8);
  if ((int64_t)p->h_k * p->page_size > (1 << 27) / p->d) return err.fail(kEinval, "a page must have at most 2^27 elements");
  const int64_t pieces = (units + kCopyUnits - 1) / kCopyUnits;
  if (2 * pieces * p->n > INT_MAX) return err.fail(kEinval, "too many pages to copy in one call");
  if (p->n == 0 || p->num_pages == 0 || units == 0) return kOk;
  if (!p->k_cache || !p->v_cache || !p->src || !p->dst) return err.fail(kEinval, "tensor pointer is NULL");
  if (!rows_ok(p->k_cache, {p->k_page_stride, p->k_head_stride, p->k_row_stride}) ||
      !rows_ok(p->v_cache, {p->v_page_stride, p->v_head_stride, p->v_row_stride}))
    return err.fail(kEinval, "caches must be 16-byte aligned with strides that are multiples of 8 elements");
  Device dev;
  if (int rc = device_ok(err, &dev)) return rc;
  CopyArgs a{};
  a.k = (uint16_t*)p->k_cache; a.v = (uint16_t*)p->v_cache; a.src = p->src; a.dst = p->dst;
  a.kp = p->k_page_stride; a.kh = p->k_head_stride; a.kr = p->k_row_stride;
  a.vp = p->v_page_stride; a.vh = p->v_head_stride; a.vr = p->v_row_stride;
  a.n = p->n; a.pages = p->num_pages; a.hk = p->h_k; a.page = p->page_size; a.chunks = p->d / 8;
  a.pieces = (int)pieces; a.units = (int)units;
  auto dense = [&](int64_t head, int64_t row) {
    return (p->page_size == 1 || row == p->d) && (p->h_k == 1 || head == (int64_t)p->page_size * p->d);
  };
  a.dense = dense(a.kh, a.kr) && dense(a.vh, a.vr);
  const int64_t waves = 2 * pieces * p->n, per = kCopyThreads / 64;
  return run(err, "paged_copy", page_copy_kernel, std::min<int64_t>((waves + per - 1) / per, (int64_t)dev.cus * 8), kCopyThreads, 0, st, a);
}

}  // namespace
}  // namespace mi355fa

extern "C" {

int mi355_beam_abi_version(void) { return MI355_BEAM_ABI_VERSION; }

int mi355_shared_decode(const mi355_shared_params* p, void* stream, char* err, size_t errlen) {
  return mi355fa::shared_decode(p, (hipStream_t)stream, {err, errlen});
}
size_t mi355_shared_decode_workspace_bytes(const mi355_shared_params* p) {
  if (mi355fa::shared_check(p, {nullptr, 0}) || p->b == 0 || p->h == 0) return 0;
  const mi355fa::SharedPlan pl = mi355fa::shared_plan(p, mi355fa::device_info().cus);
  return mi355fa::shared_fits(p, pl) ? pl.bytes : 0;
}

int mi355_beam_select(const mi355_select_params* p, void* stream, char* err, size_t errlen) {
  return mi355fa::beam_select(p, (hipStream_t)stream, {err, errlen});
}
size_t mi355_beam_select_workspace_bytes(const mi355_select_params* p) {
  if (mi355fa::select_check(p, {nullptr, 0}) || p->n_groups == 0) return 0;
  return mi355fa::select_plan(p, mi355fa::device_info().cus).bytes;
}

int mi355_paged_fork(const mi355_fork_params* p, void* stream, char* err, size_t errlen) {
  return mi355fa::paged_fork(p, (hipStream_t)stream, {err, errlen});
}
size_t mi355_paged_fork_workspace_bytes(const mi355_fork_params* p) {
  if (mi355fa::fork_check(p, {nullptr, 0})) return 0;
  return mi355fa::page_plan(p->r, p->table_cols, p->num_pages, true, mi355fa::device_info().cus).bytes;
}

int mi355_paged_compact(const mi355_compact_params* p, void* stream, char* err, size_t errlen) {
  return mi355fa::paged_compact(p, (hipStream_t)stream, {err, errlen});
}
size_t mi355_paged_compact_workspace_bytes(const mi355_compact_params* p) {
  if (mi355fa::compact_check(p, {nullptr, 0})) return 0;
  return mi355fa::page_plan(p->n, p->table_cols, p->num_pages, false, mi355fa::device_info().cus).bytes;
}

int mi355_paged_copy(const mi355_copy_params* p, void* stream, char* err, size_t errlen) {
  return mi355fa::paged_copy(p, (hipStream_t)stream, {err, errlen});
}

}  // extern "C"
