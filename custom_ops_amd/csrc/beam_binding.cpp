// The CUDA-key implementation of the operators for several continuations of a prompt over
// the C ABI of libmi355_beam.so, for PyTorch-ROCm. beam.py defines the operators
// (schemas, CPU and Meta keys); this file (libmi355_beam_ops.so) checks the arguments,
// allocates outputs and workspaces from the caching allocator and launches on the
// current stream of the inputs' GPU. It reaches the library that the loader opened through
// mi355_beam_connect, so that opening the file changes nothing in the dispatcher,
// and it names the sources and the PyTorch it was built from (mi355_ops_stamp),
// which are read before it is opened.
//
// Every check is of shapes, types and strides, on the host; lengths, offsets, rows and
// page numbers stay on the device, where the kernels hold them to their ranges.
#include "binding.h"

#include "mi355_beam.h"

namespace {

using namespace mi355ops;

decltype(&mi355_shared_decode) g_shared = nullptr;
decltype(&mi355_shared_decode_workspace_bytes) g_shared_bytes = nullptr;
decltype(&mi355_beam_select) g_select = nullptr;
decltype(&mi355_beam_select_workspace_bytes) g_select_bytes = nullptr;
decltype(&mi355_paged_fork) g_fork = nullptr;
decltype(&mi355_paged_fork_workspace_bytes) g_fork_bytes = nullptr;
decltype(&mi355_paged_compact) g_compact = nullptr;
decltype(&mi355_paged_compact_workspace_bytes) g_compact_bytes = nullptr;
decltype(&mi355_paged_copy) g_copy = nullptr;

typedef std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor> Six;

// Workspace of n bytes for p (held by ws until the call is enqueued)
template <class P> void work(P& p, Tensor& ws, size_t n, const Tensor& x) {
  if (n == 0) return;
  ws = fresh(x, {(int64_t)n}, at::kByte);
  p.workspace = ws.data_ptr();
  p.workspace_bytes = n;
}

int* ints(const Tensor& x) { return x.numel() ? x.data_ptr<int>() : nullptr; }

Tensor mha_shared_decode(const Tensor& q, const Tensor& k_cache, const Tensor& v_cache, const Tensor& block_table, const Tensor& kv_lens,
                         const Tensor& cu_groups, const Tensor& prefix_lens, std::optional<double> scale, double softcap, int64_t window,
                         const Maybe& slopes) {
  check_half(q);
  check_rows(q, q, "q", 3);
  check_rows(k_cache, q, "k_cache", 4);
  check_rows(v_cache, q, "v_cache", 4);
  const int64_t B = q.size(0), H = q.size(1), d = q.size(2), P = k_cache.size(0), Hk = k_cache.size(1), page = k_cache.size(2);
  TORCH_CHECK(k_cache.size(3) == d && v_cache.size(3) == d, "head_dim mismatch between q and the caches");
  TORCH_CHECK(v_cache.size(0) == P && v_cache.size(1) == Hk && v_cache.size(2) == page, "k_cache and v_cache must have the same shape");
  check_groups(H, Hk);
  check_head_dim(d);
  TORCH_CHECK(page >= 8 && page <= 1024 && (page & (page - 1)) == 0, "page_size must be a power of two in 8 .. 1024");
  TORCH_CHECK(P <= INT_MAX && H <= (1 << 16), "too many pages or heads");
  TORCH_CHECK(B <= MI355_BEAM_MAX_REQUESTS, "at most ", MI355_BEAM_MAX_REQUESTS, " requests");
  check_gpu(block_table, q, "block_table");
  TORCH_CHECK(block_table.scalar_type() == at::kInt && block_table.dim() == 2 && block_table.size(0) == B,
              "block_table must be int32 of shape (batch, pages)");
  TORCH_CHECK(block_table.size(1) <= 1 || block_table.stride(1) == 1, "block_table must have an innermost stride of 1");
  TORCH_CHECK(block_table.size(1) <= (1 << 30) / page, "block_table must span at most 2^30 keys");
  check_ints(kv_lens, q, "kv_lens", at::kInt, B);
  TORCH_CHECK(prefix_lens.dim() == 1, "prefix_lens must be 1D");
  const int64_t G = prefix_lens.size(0);
  TORCH_CHECK(G <= MI355_BEAM_MAX_REQUESTS, "at most ", MI355_BEAM_MAX_REQUESTS, " groups");
  check_ints(prefix_lens, q, "prefix_lens", at::kInt, G);
  check_ints(cu_groups, q, "cu_groups", at::kInt, G + 1);
  check_scores(scale, softcap, window);
  mi355_shared_params p{};
  p.slopes = slopes_of(slopes, q, H);

  c10::hip::HIPGuardMasqueradingAsCUDA guard(q.device());
  Tensor out = fresh(q, {B, H, d}, q.scalar_type());
  if (out.numel() == 0) return out;
  p.q = q.data_ptr(); p.k_cache = k_cache.data_ptr(); p.v_cache = v_cache.data_ptr(); p.o = out.data_ptr();
  p.block_table = ints(block_table); p.kv_lens = ints(kv_lens); p.cu_groups = ints(cu_groups); p.prefix_lens = ints(prefix_lens);
  p.q_batch_stride = step(q, 0); p.q_head_stride = step(q, 1);
  p.o_batch_stride = H * d; p.o_head_stride = d;
  p.k_page_stride = step(k_cache, 0); p.k_head_stride = step(k_cache, 1); p.k_row_stride = step(k_cache, 2);
  p.v_page_stride = step(v_cache, 0); p.v_head_stride = step(v_cache, 1); p.v_row_stride = step(v_cache, 2);
  p.table_stride = block_table.size(0) <= 1 ? 0 : block_table.stride(0);
  p.b = (int)B; p.n_groups = (int)G; p.h = (int)H; p.h_k = (int)Hk; p.d = (int)d; p.dtype = type_of(q);
  p.num_pages = (int)P; p.page_size = (int)page; p.table_cols = (int)block_table.size(1);
  p.window = (int)window;
  p.scale = scale.has_value() ? (float)*scale : 1.0f / std::sqrt((float)d);
  p.softcap = (float)softcap;
  Tensor ws;
  work(p, ws, g_shared_bytes(&p), q);
  char err[512] = {0};
  finish(g_shared(&p, stream_of(q), err, sizeof err), err);
  return out;
}

std::tuple<Tensor, Tensor, Tensor> beam_select(const Tensor& logits, const Tensor& scores, int64_t k, const Maybe& finished, int64_t eos) {
  TORCH_CHECK(logits.is_cuda(), "logits must be a CUDA tensor");
  const auto type = logits.scalar_type();
  TORCH_CHECK(type == at::kHalf || type == at::kBFloat16 || type == at::kFloat, "logits must be float16, bfloat16 or float32");
  TORCH_CHECK(logits.dim() == 3, "logits must be 3D (searches, beams, vocabulary)");
  const int64_t G = logits.size(0), W = logits.size(1), V = logits.size(2);
  TORCH_CHECK(W >= 1 && W <= 256, "beams must be in 1 .. 256");
  TORCH_CHECK(V >= 1 && V <= INT_MAX / W && G < ((1 << 24) + W - 1) / W, "the vocabulary must not be empty, beams·vocabulary below 2^31 and searches·beams below 2^24");
  TORCH_CHECK(V == 1 || logits.stride(2) == 1, "logits must have an innermost stride of 1");
  check_gpu(scores, logits, "scores");
  TORCH_CHECK(scores.scalar_type() == at::kFloat, "scores must be float32");
  TORCH_CHECK(scores.dim() == 2 && scores.size(0) == G && scores.size(1) == W && scores.is_contiguous(),
              "scores must be contiguous of shape (searches, beams)");
  TORCH_CHECK(k >= 1 && k <= 64, "k must be in 1 .. 64");
  if (finished.has_value()) {
    check_gpu(*finished, logits, "finished");
    TORCH_CHECK(finished->scalar_type() == at::kBool, "finished must be bool");
    TORCH_CHECK(finished->dim() == 2 && finished->size(0) == G && finished->size(1) == W && finished->is_contiguous(),
                "finished must be contiguous of shape (searches, beams)");
    TORCH_CHECK(eos >= 0 && eos < V, "eos must be a token of the vocabulary where finished is given");
  }

  c10::hip::HIPGuardMasqueradingAsCUDA guard(logits.device());
  Tensor out_s = fresh(logits, {G, k}, at::kFloat), out_t = fresh(logits, {G, k}, at::kInt), out_p = fresh(logits, {G, k}, at::kInt);
  if (G == 0) return {out_s, out_t, out_p};
  mi355_select_params p{};
  p.logits = logits.data_ptr(); p.scores = scores.data_ptr<float>();
  p.finished = finished.has_value() ? reinterpret_cast<const uint8_t*>(finished->data_ptr<bool>()) : nullptr;
  p.out_scores = out_s.data_ptr<float>(); p.out_tokens = ints(out_t); p.out_parents = ints(out_p);
  p.group_stride = step(logits, 0); p.beam_stride = step(logits, 1);
  p.n_groups = (int)G; p.beams = (int)W; p.vocab = (int)V; p.k = (int)k;
  p.eos = finished.has_value() ? (int)eos : 0;
  p.dtype = type == at::kFloat ? MI355_BEAM_FP32 : type_of(logits);
  Tensor ws;
  work(p, ws, g_select_bytes(&p), logits);
  char err[512] = {0};
  finish(g_select(&p, stream_of(logits), err, sizeof err), err);
  return {out_s, out_t, out_p};
}

// A page table of requests and their lengths; the pages of a cache; pages that stay.
void check_table(const Tensor& block_table, const Tensor& seq_lens, int64_t page_size, int64_t num_pages, const Maybe& held) {
  TORCH_CHECK(block_table.is_cuda(), "block_table must be a CUDA tensor");
  TORCH_CHECK(block_table.scalar_type() == at::kInt && block_table.dim() == 2, "block_table must be int32 of shape (requests, pages)");
  TORCH_CHECK(block_table.size(1) <= 1 || block_table.stride(1) == 1, "block_table must have an innermost stride of 1");
  TORCH_CHECK(block_table.size(0) <= INT_MAX && block_table.size(1) <= (1 << 30), "block_table must have at most 2^30 columns");
  check_ints(seq_lens, block_table, "seq_lens", at::kInt, block_table.size(0));
  TORCH_CHECK(page_size >= 1 && page_size <= INT_MAX, "page_size must be positive");
  TORCH_CHECK(num_pages >= 0 && num_pages <= MI355_BEAM_MAX_PAGES, "num_pages must be in 0 .. ", MI355_BEAM_MAX_PAGES);
  if (held.has_value()) {
    TORCH_CHECK(held->dim() == 1 && held->size(0) <= INT_MAX, "held must be 1D");
    check_ints(*held, block_table, "held", at::kInt, held->size(0));
  }
}
template <class P> void fill_table(P& p, const Tensor& block_table, const Tensor& seq_lens, int64_t page_size, int64_t num_pages, const Maybe& held) {
  p.block_table = ints(block_table); p.seq_lens = ints(seq_lens);
  p.table_stride = block_table.size(0) <= 1 ? 0 : block_table.stride(0);
  p.n = (int)block_table.size(0); p.table_cols = (int)block_table.size(1);
  p.num_pages = (int)num_pages; p.page_size = (int)page_size;
  p.held = held.has_value() ? ints(*held) : nullptr;
  p.n_held = held.has_value() ? (int)held->size(0) : 0;
}

Six paged_fork(const Tensor& block_table, const Tensor& seq_lens, const Tensor& parents, int64_t page_size, int64_t num_pages, const Maybe& held) {
  check_table(block_table, seq_lens, page_size, num_pages, held);
  TORCH_CHECK(parents.dim() == 1, "parents must be 1D");
  const int64_t R = parents.size(0), M = block_table.size(1);
  TORCH_CHECK(R <= MI355_BEAM_MAX_ROWS, "at most ", MI355_BEAM_MAX_ROWS, " rows");
  check_ints(parents, block_table, "parents", at::kInt, R);

  c10::hip::HIPGuardMasqueradingAsCUDA guard(block_table.device());
  auto make = [&](at::IntArrayRef sizes) { return fresh(block_table, sizes, at::kInt); };
  Tensor table = make({R, M}), lens = make({R}), src = make({R}), dst = make({R}), free_pages = make({num_pages}), counts = make({3});
  mi355_fork_params p{};
  fill_table(p, block_table, seq_lens, page_size, num_pages, held);
  p.parents = ints(parents); p.table = ints(table); p.lens = ints(lens); p.src = ints(src); p.dst = ints(dst);
  p.free_pages = ints(free_pages); p.counts = ints(counts);
  p.r = (int)R;
  Tensor ws;
  work(p, ws, g_fork_bytes(&p), block_table);
  char err[512] = {0};
  finish(g_fork(&p, stream_of(block_table), err, sizeof err), err);
  return {table, lens, src, dst, free_pages, counts};
}

Six paged_compact(const Tensor& block_table, const Tensor& seq_lens, int64_t page_size, int64_t num_pages, const Maybe& held) {
  check_table(block_table, seq_lens, page_size, num_pages, held);
  const int64_t N = block_table.size(0), M = block_table.size(1);
  TORCH_CHECK(N <= MI355_BEAM_MAX_ROWS, "at most ", MI355_BEAM_MAX_ROWS, " rows");

  c10::hip::HIPGuardMasqueradingAsCUDA guard(block_table.device());
  auto make = [&](at::IntArrayRef sizes) { return fresh(block_table, sizes, at::kInt); };
  Tensor table = make({N, M}), src = make({num_pages / 2}), dst = make({num_pages / 2}), remap = make({num_pages}), free_pages = make({num_pages}),
         counts = make({2});
  mi355_compact_params p{};
  fill_table(p, block_table, seq_lens, page_size, num_pages, held);
  p.table = ints(table); p.src = ints(src); p.dst = ints(dst); p.remap = ints(remap); p.free_pages = ints(free_pages); p.counts = ints(counts);
  Tensor ws;
  work(p, ws, g_compact_bytes(&p), block_table);
  char err[512] = {0};
  finish(g_compact(&p, stream_of(block_table), err, sizeof err), err);
  return {table, src, dst, remap, free_pages, counts};
}

void paged_copy(const Tensor& k_cache, const Tensor& v_cache, const Tensor& src, const Tensor& dst) {
  TORCH_CHECK(k_cache.is_cuda(), "k_cache must be a CUDA tensor");
  TORCH_CHECK(k_cache.scalar_type() == at::kHalf || k_cache.scalar_type() == at::kBFloat16, "k_cache must be float16 or bfloat16");
  check_rows(k_cache, k_cache, "k_cache", 4);
  check_rows(v_cache, k_cache, "v_cache", 4);
  TORCH_CHECK(v_cache.sizes() == k_cache.sizes(), "k_cache and v_cache must have the same shape");
  check_head_dim(k_cache.size(3));
  at::assert_no_internal_overlap(k_cache);   // written in place
  at::assert_no_internal_overlap(v_cache);
  at::assert_no_overlap(k_cache, v_cache);
  TORCH_CHECK(!share(k_cache, v_cache), "k_cache and v_cache must not overlap");
  TORCH_CHECK(src.dim() == 1 && src.size(0) <= INT_MAX, "src must be 1D");
  check_ints(src, k_cache, "src", at::kInt, src.size(0));
  check_ints(dst, k_cache, "dst", at::kInt, src.size(0));
  const int64_t P = k_cache.size(0), Hk = k_cache.size(1), page = k_cache.size(2), d = k_cache.size(3);
  TORCH_CHECK(P <= INT_MAX && Hk <= (1 << 27) && page <= (1 << 27), "too many pages, heads or rows");
  if (k_cache.numel() == 0 || src.size(0) == 0) return;

  c10::hip::HIPGuardMasqueradingAsCUDA guard(k_cache.device());
  mi355_copy_params p{};
  p.k_cache = k_cache.data_ptr(); p.v_cache = v_cache.data_ptr(); p.src = ints(src); p.dst = ints(dst);
  p.k_page_stride = step(k_cache, 0); p.k_head_stride = step(k_cache, 1); p.k_row_stride = step(k_cache, 2);
  p.v_page_stride = step(v_cache, 0); p.v_head_stride = step(v_cache, 1); p.v_row_stride = step(v_cache, 2);
  p.n = (int)src.size(0); p.num_pages = (int)P; p.h_k = (int)Hk; p.page_size = (int)page; p.d = (int)d;
  char err[512] = {0};
  finish(g_copy(&p, stream_of(k_cache), err, sizeof err), err);
}

constexpr char kSharedName[] = "recsys_ops::mha_shared_decode", kSelectName[] = "recsys_ops::beam_select", kCopyName[] = "recsys_ops::paged_copy";

// The caches' version counters move, so that autograd notices a cache that it saved for
// another operator. (Inference tensors have none.)
void paged_copy_inplace(c10::DispatchKeySet keys, const Tensor& k_cache, const Tensor& v_cache, const Tensor& src, const Tensor& dst) {
  {
    at::AutoDispatchBelowADInplaceOrView below;
    Gate<kCopyName, decltype(paged_copy)>::op().redispatch(keys & c10::after_ADInplaceOrView_keyset, k_cache, v_cache, src, dst);
  }
  for (const Tensor* x : {&k_cache, &v_cache})
    if (!x->is_inference()) x->unsafeGetTensorImpl()->bump_version();
}

template <class F> bool find(void* handle, const char* name, F& f) {
  f = reinterpret_cast<F>(dlsym(handle, name));
  return f != nullptr;
}

}  // namespace

extern "C" __attribute__((used, visibility("default"))) const char mi355_ops_stamp[] = MI355_OPS_STAMP;

// Takes the entry points of the library opened at `handle` (a dlopen handle) and
// registers the implementations, once. 1, and nothing registered, where the library
// is of another ABI than this file was compiled for.
extern "C" int mi355_beam_connect(void* handle) {
  decltype(&mi355_beam_abi_version) version = nullptr;
  if (!find(handle, "mi355_beam_abi_version", version) || version() != MI355_BEAM_ABI_VERSION) return 1;
  if (!find(handle, "mi355_shared_decode", g_shared) || !find(handle, "mi355_shared_decode_workspace_bytes", g_shared_bytes) ||
      !find(handle, "mi355_beam_select", g_select) || !find(handle, "mi355_beam_select_workspace_bytes", g_select_bytes) ||
      !find(handle, "mi355_paged_fork", g_fork) || !find(handle, "mi355_paged_fork_workspace_bytes", g_fork_bytes) ||
      !find(handle, "mi355_paged_compact", g_compact) || !find(handle, "mi355_paged_compact_workspace_bytes", g_compact_bytes) ||
      !find(handle, "mi355_paged_copy", g_copy))
    return 1;
  try {
    static torch::Library lib(torch::Library::IMPL, "recsys_ops", c10::DispatchKey::CUDA, __FILE__, __LINE__);
    static const bool once = (lib.impl("mha_shared_decode", &mha_shared_decode), lib.impl("beam_select", &beam_select),
                              lib.impl("paged_fork", &paged_fork), lib.impl("paged_compact", &paged_compact), lib.impl("paged_copy", &paged_copy), true);
    static torch::Library autograd(torch::Library::IMPL, "recsys_ops", c10::DispatchKey::Autograd, __FILE__, __LINE__);
    static const bool once_more = (autograd.impl("mha_shared_decode", &Gate<kSharedName, decltype(mha_shared_decode)>::autograd),
                                   autograd.impl("beam_select", &Gate<kSelectName, decltype(beam_select)>::autograd),
                                   autograd.impl("paged_copy", &Gate<kCopyName, decltype(paged_copy)>::autograd),
                                   // whole numbers only: nothing to refuse
                                   autograd.impl("paged_fork", torch::CppFunction::makeFallthrough()),
                                   autograd.impl("paged_compact", torch::CppFunction::makeFallthrough()), true);
    static torch::Library inplace(torch::Library::IMPL, "recsys_ops", c10::DispatchKey::ADInplaceOrView, __FILE__, __LINE__);
    static const bool once_again = (inplace.impl("paged_copy", &paged_copy_inplace), true);
    (void)once;
    (void)once_more;
    (void)once_again;
  } catch (const std::exception&) {
    return 1;
  }
  return 0;
}
