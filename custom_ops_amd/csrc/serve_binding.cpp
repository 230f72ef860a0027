// The CUDA-key implementation of the serving operators over the C ABI of
// libmi355_serve.so, for PyTorch-ROCm. serve.py defines the operators (schemas,
// CPU and Meta keys); this file (libmi355_serve_ops.so) checks the arguments,
// allocates outputs and workspaces from the caching allocator and launches on the
// current stream of q's GPU. It reaches the library that the loader opened through
// mi355_serve_connect, so that opening the file changes nothing in the dispatcher,
// and it names the sources and the PyTorch it was built from (mi355_ops_stamp),
// which are read before it is opened.
//
// Every check is of shapes, types and strides, on the host; lengths, offsets, page
// and slot numbers stay on the device, where the kernels hold them to their ranges.
#include "binding.h"

#include "mi355_serve.h"

namespace {

using namespace mi355ops;

decltype(&mi355_packed_fwd) g_packed = nullptr;
decltype(&mi355_paged_decode) g_decode = nullptr;
decltype(&mi355_paged_decode_workspace_bytes) g_decode_bytes = nullptr;
decltype(&mi355_rope_paged_store) g_rope = nullptr;
decltype(&mi355_paged_layout) g_layout = nullptr;

Tensor mha_packed_fwd(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& cu_q, const Tensor& cu_k, bool causal,
                      std::optional<double> scale, double softcap, int64_t window, const Maybe& slopes, const Maybe& prefix_lens) {
  check_half(q);
  check_rows(q, q, "q", 3);
  check_rows(k, q, "k", 3);
  check_rows(v, q, "v", 3);
  const int64_t Tq = q.size(0), H = q.size(1), d = q.size(2), Tk = k.size(0), Hk = k.size(1);
  TORCH_CHECK(k.size(2) == d && v.size(2) == d, "head_dim mismatch between q/k/v");
  TORCH_CHECK(v.size(0) == Tk, "token count mismatch between k/v");
  TORCH_CHECK(v.size(1) == Hk, "n_kv_heads mismatch between k/v");
  check_groups(H, Hk);
  check_head_dim(d);
  TORCH_CHECK(Tq <= (1 << 30) && Tk <= (1 << 30), "at most 2^30 tokens");
  TORCH_CHECK(cu_q.dim() == 1 && cu_q.size(0) >= 1, "cu_q must be 1D with n_seqs + 1 elements");
  const int64_t n = cu_q.size(0) - 1;
  TORCH_CHECK(n <= (1 << 30), "at most 2^30 sequences");
  check_ints(cu_q, q, "cu_q", at::kInt, n + 1);
  check_ints(cu_k, q, "cu_k", at::kInt, n + 1);
  if (prefix_lens.has_value()) check_ints(*prefix_lens, q, "prefix_lens", at::kInt, n);
  check_scores(scale, softcap, window);
  mi355_packed_params p{};
  p.slopes = slopes_of(slopes, q, H);

  c10::hip::HIPGuardMasqueradingAsCUDA guard(q.device());
  Tensor out = fresh(q, {Tq, H, d}, q.scalar_type());
  if (out.numel() == 0) return out;
  // rows of v that overlap in memory, as of one row expanded over the tokens, get their own
  const Tensor vr = Tk > 1 && v.stride(0) < d ? v.clone(at::MemoryFormat::Contiguous) : v;
  p.q = q.data_ptr(); p.k = k.data_ptr(); p.v = vr.data_ptr(); p.o = out.data_ptr();
  p.cu_q = cu_q.data_ptr<int>(); p.cu_k = cu_k.data_ptr<int>();
  p.prefix_lens = prefix_lens.has_value() && n > 0 ? prefix_lens->data_ptr<int>() : nullptr;
  p.q_token_stride = step(q, 0); p.q_head_stride = step(q, 1);
  p.k_token_stride = step(k, 0); p.k_head_stride = step(k, 1);
  p.v_token_stride = step(vr, 0); p.v_head_stride = step(vr, 1);
  p.o_token_stride = H * d; p.o_head_stride = d;
  p.total_q = (int)Tq; p.total_k = (int)Tk; p.n_seqs = (int)n;
  p.h = (int)H; p.h_k = (int)Hk; p.d = (int)d; p.dtype = type_of(q);
  p.causal = causal; p.window = (int)window;
  p.scale = scale.has_value() ? (float)*scale : 1.0f / std::sqrt((float)d);
  p.softcap = (float)softcap;
  char err[512] = {0};
  finish(g_packed(&p, stream_of(q), err, sizeof err), err);
  return out;
}

Tensor mha_paged_decode(const Tensor& q, const Tensor& k_cache, const Tensor& v_cache, const Tensor& block_table, const Tensor& kv_lens,
                        std::optional<double> scale, double softcap, int64_t window, const Maybe& slopes) {
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
  TORCH_CHECK(P <= INT_MAX && B <= INT_MAX, "too many pages or requests");
  check_gpu(block_table, q, "block_table");
  TORCH_CHECK(block_table.scalar_type() == at::kInt && block_table.dim() == 2 && block_table.size(0) == B,
              "block_table must be int32 of shape (batch, pages)");
  TORCH_CHECK(block_table.size(1) <= 1 || block_table.stride(1) == 1, "block_table must have an innermost stride of 1");
  TORCH_CHECK(block_table.size(1) <= (1 << 30) / page, "block_table must span at most 2^30 keys");
  check_ints(kv_lens, q, "kv_lens", at::kInt, B);
  check_scores(scale, softcap, window);
  mi355_decode_params p{};
  p.slopes = slopes_of(slopes, q, H);

  c10::hip::HIPGuardMasqueradingAsCUDA guard(q.device());
  Tensor out = fresh(q, {B, H, d}, q.scalar_type());
  if (out.numel() == 0) return out;
  p.q = q.data_ptr(); p.k_cache = k_cache.data_ptr(); p.v_cache = v_cache.data_ptr(); p.o = out.data_ptr();
  p.block_table = block_table.numel() ? block_table.data_ptr<int>() : nullptr;
  p.kv_lens = kv_lens.data_ptr<int>();
  p.q_batch_stride = step(q, 0); p.q_head_stride = step(q, 1);
  p.o_batch_stride = H * d; p.o_head_stride = d;
  p.k_page_stride = step(k_cache, 0); p.k_head_stride = step(k_cache, 1); p.k_row_stride = step(k_cache, 2);
  p.v_page_stride = step(v_cache, 0); p.v_head_stride = step(v_cache, 1); p.v_row_stride = step(v_cache, 2);
  p.table_stride = block_table.size(0) <= 1 ? 0 : block_table.stride(0);
  p.b = (int)B; p.h = (int)H; p.h_k = (int)Hk; p.d = (int)d; p.dtype = type_of(q);
  p.num_pages = (int)P; p.page_size = (int)page; p.table_cols = (int)block_table.size(1);
  p.window = (int)window;
  p.scale = scale.has_value() ? (float)*scale : 1.0f / std::sqrt((float)d);
  p.softcap = (float)softcap;
  Tensor ws;
  if (const size_t n = g_decode_bytes(&p)) {
    ws = fresh(q, {(int64_t)n}, at::kByte);
    p.workspace = ws.data_ptr();
    p.workspace_bytes = n;
  }
  char err[512] = {0};
  finish(g_decode(&p, stream_of(q), err, sizeof err), err);
  return out;
}

std::tuple<Tensor, Tensor> rope_paged_store(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& positions, const Tensor& inv_freq,
                                            const Tensor& slot_map, const Tensor& k_cache, const Tensor& v_cache, bool interleaved,
                                            double amplitude) {
  check_half(q);
  check_rows(q, q, "q", 3);
  check_rows(k, q, "k", 3);
  check_rows(v, q, "v", 3);
  check_rows(k_cache, q, "k_cache", 4);
  check_rows(v_cache, q, "v_cache", 4);
  const int64_t T = q.size(0), H = q.size(1), d = q.size(2), Hk = k.size(1), P = k_cache.size(0), page = k_cache.size(2);
  TORCH_CHECK(k.size(0) == T && v.size(0) == T, "token count mismatch between q/k/v");
  TORCH_CHECK(k.size(2) == d && v.size(2) == d, "head_dim mismatch between q/k/v");
  TORCH_CHECK(v.size(1) == Hk, "n_kv_heads mismatch between k/v");
  TORCH_CHECK(k_cache.size(1) == Hk && k_cache.size(3) == d, "k_cache must be (pages, n_kv_heads, page_size, head_dim)");
  TORCH_CHECK(v_cache.sizes() == k_cache.sizes(), "k_cache and v_cache must have the same shape");
  at::assert_no_internal_overlap(k_cache);   // written in place
  at::assert_no_internal_overlap(v_cache);
  at::assert_no_overlap(k_cache, v_cache);
  TORCH_CHECK(!share(k_cache, v_cache), "k_cache and v_cache must not overlap");
  for (const Tensor* x : {&q, &k, &v}) {
    at::assert_no_overlap(k_cache, *x);
    at::assert_no_overlap(v_cache, *x);
  }
  check_groups(H, Hk);
  check_head_dim(d);
  TORCH_CHECK(T <= (1 << 30) && P <= INT_MAX && page <= INT_MAX, "too many tokens or pages");
  TORCH_CHECK(page >= 1, "page_size must be positive");
  check_ints(positions, q, "positions", at::kInt, T);
  check_ints(slot_map, q, "slot_map", at::kLong, T);
  TORCH_CHECK(inv_freq.dim() == 1 && inv_freq.size(0) % 8 == 0 && 2 * inv_freq.size(0) <= d,
              "inv_freq must be 1D, a multiple of 8 pairs and at most head_dim / 2");
  check_ints(inv_freq, q, "inv_freq", at::kDouble, inv_freq.size(0));
  TORCH_CHECK(std::isfinite(amplitude) && std::isfinite((float)amplitude), "amplitude must be finite");

  c10::hip::HIPGuardMasqueradingAsCUDA guard(q.device());
  Tensor qo = fresh(q, {T, H, d}, q.scalar_type()), ko = fresh(q, {T, Hk, d}, q.scalar_type());
  if (T == 0) return {qo, ko};
  mi355_rope_params p{};
  p.q = q.data_ptr(); p.k = k.data_ptr(); p.v = v.data_ptr(); p.q_out = qo.data_ptr(); p.k_out = ko.data_ptr();
  p.k_cache = k_cache.data_ptr(); p.v_cache = v_cache.data_ptr();
  p.positions = positions.data_ptr<int>();
  p.inv_freq = inv_freq.numel() ? inv_freq.data_ptr<double>() : nullptr;
  p.slot_map = slot_map.data_ptr<int64_t>();
  p.q_token_stride = step(q, 0); p.q_head_stride = step(q, 1);
  p.k_token_stride = step(k, 0); p.k_head_stride = step(k, 1);
  p.v_token_stride = step(v, 0); p.v_head_stride = step(v, 1);
  p.qo_token_stride = H * d; p.qo_head_stride = d;
  p.ko_token_stride = Hk * d; p.ko_head_stride = d;
  p.kc_page_stride = step(k_cache, 0); p.kc_head_stride = step(k_cache, 1); p.kc_row_stride = step(k_cache, 2);
  p.vc_page_stride = step(v_cache, 0); p.vc_head_stride = step(v_cache, 1); p.vc_row_stride = step(v_cache, 2);
  p.t = (int)T; p.h = (int)H; p.h_k = (int)Hk; p.d = (int)d; p.dtype = type_of(q);
  p.rot = (int)(2 * inv_freq.size(0)); p.interleaved = interleaved;
  p.num_pages = (int)P; p.page_size = (int)page; p.amplitude = (float)amplitude;
  char err[512] = {0};
  finish(g_rope(&p, stream_of(q), err, sizeof err), err);
  return {qo, ko};
}

std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor> paged_layout(const Tensor& seq_lens, const Tensor& new_lens, const Tensor& block_table,
                                                                        const Tensor& free_pages, int64_t page_size, int64_t max_tokens) {
  TORCH_CHECK(seq_lens.is_cuda(), "seq_lens must be a CUDA tensor");
  TORCH_CHECK(seq_lens.dim() == 1, "seq_lens must be 1D");
  const int64_t n = seq_lens.size(0);
  TORCH_CHECK(n <= MI355_SERVE_MAX_REQUESTS, "at most ", MI355_SERVE_MAX_REQUESTS, " requests");
  check_ints(seq_lens, seq_lens, "seq_lens", at::kInt, n);
  check_ints(new_lens, seq_lens, "new_lens", at::kInt, n);
  check_gpu(block_table, seq_lens, "block_table");
  TORCH_CHECK(block_table.scalar_type() == at::kInt && block_table.dim() == 2 && block_table.size(0) == n,
              "block_table must be int32 of shape (requests, pages)");
  const int64_t M = block_table.size(1);
  TORCH_CHECK(M <= 1 || block_table.stride(1) == 1, "block_table must have an innermost stride of 1");
  TORCH_CHECK(free_pages.dim() == 1, "free_pages must be 1D");
  check_ints(free_pages, seq_lens, "free_pages", at::kInt, free_pages.size(0));
  TORCH_CHECK(page_size >= 1 && page_size <= INT_MAX, "page_size must be positive");
  TORCH_CHECK(max_tokens >= 0 && max_tokens <= INT_MAX, "max_tokens must be in 0 .. 2^31 - 1");
  TORCH_CHECK(M <= INT_MAX && free_pages.size(0) <= INT_MAX, "too many pages");

  c10::hip::HIPGuardMasqueradingAsCUDA guard(seq_lens.device());
  auto make = [&](at::IntArrayRef sizes) { return fresh(seq_lens, sizes, at::kInt); };
  Tensor kv_lens = make({n}), cu = make({n + 1}), positions = make({max_tokens}), table = make({n, M}), counts = make({3});
  Tensor slots = fresh(seq_lens, {max_tokens}, at::kLong);
  mi355_layout_params p{};
  auto ints = [](const Tensor& x) { return x.numel() ? x.data_ptr<int>() : nullptr; };
  p.seq_lens = ints(seq_lens); p.new_lens = ints(new_lens); p.block_table = ints(block_table); p.free_pages = ints(free_pages);
  p.kv_lens = ints(kv_lens); p.cu_new = ints(cu); p.positions = ints(positions);
  p.slot_map = max_tokens ? slots.data_ptr<int64_t>() : nullptr;
  p.table = ints(table); p.counts = ints(counts);
  p.table_stride = n <= 1 ? 0 : block_table.stride(0);
  p.n = (int)n; p.table_cols = (int)M; p.n_free = (int)free_pages.size(0); p.page_size = (int)page_size; p.max_tokens = (int)max_tokens;
  char err[512] = {0};
  finish(g_layout(&p, stream_of(seq_lens), err, sizeof err), err);
  return {kv_lens, cu, positions, slots, table, counts};
}

// ── autograd ──────────────────────────────────────────────────────────────────
constexpr char kPackedName[] = "recsys_ops::mha_packed_fwd", kDecodeName[] = "recsys_ops::mha_paged_decode",
               kRopeName[] = "recsys_ops::rope_paged_store";

// The caches' version counters move, so that autograd notices a cache that it saved for
// another operator. (Inference tensors have none.)
std::tuple<Tensor, Tensor> rope_paged_store_inplace(c10::DispatchKeySet keys, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& positions,
                                                    const Tensor& inv_freq, const Tensor& slot_map, const Tensor& k_cache, const Tensor& v_cache,
                                                    bool interleaved, double amplitude) {
  auto out = [&] {
    at::AutoDispatchBelowADInplaceOrView below;
    return Gate<kRopeName, decltype(rope_paged_store)>::op().redispatch(keys & c10::after_ADInplaceOrView_keyset, q, k, v, positions, inv_freq, slot_map,
                                                                        k_cache, v_cache, interleaved, amplitude);
  }();
  for (const Tensor* x : {&k_cache, &v_cache})
    if (!x->is_inference()) x->unsafeGetTensorImpl()->bump_version();
  return out;
}

}  // namespace

extern "C" __attribute__((used, visibility("default"))) const char mi355_ops_stamp[] = MI355_OPS_STAMP;

// Takes the entry points of the library opened at `handle` (a dlopen handle) and
// registers the implementations, once. 1, and nothing registered, where the library
// is of another ABI than this file was compiled for.
extern "C" int mi355_serve_connect(void* handle) {
  auto version = reinterpret_cast<decltype(&mi355_serve_abi_version)>(dlsym(handle, "mi355_serve_abi_version"));
  if (!version || version() != MI355_SERVE_ABI_VERSION) return 1;
  g_packed = reinterpret_cast<decltype(g_packed)>(dlsym(handle, "mi355_packed_fwd"));
  g_decode = reinterpret_cast<decltype(g_decode)>(dlsym(handle, "mi355_paged_decode"));
  g_decode_bytes = reinterpret_cast<decltype(g_decode_bytes)>(dlsym(handle, "mi355_paged_decode_workspace_bytes"));
  g_rope = reinterpret_cast<decltype(g_rope)>(dlsym(handle, "mi355_rope_paged_store"));
  g_layout = reinterpret_cast<decltype(g_layout)>(dlsym(handle, "mi355_paged_layout"));
  if (!g_packed || !g_decode || !g_decode_bytes || !g_rope || !g_layout) return 1;
  try {
    static torch::Library lib(torch::Library::IMPL, "recsys_ops", c10::DispatchKey::CUDA, __FILE__, __LINE__);
    static const bool once = (lib.impl("mha_packed_fwd", &mha_packed_fwd), lib.impl("mha_paged_decode", &mha_paged_decode),
                              lib.impl("rope_paged_store", &rope_paged_store), lib.impl("paged_layout", &paged_layout), true);
    static torch::Library autograd(torch::Library::IMPL, "recsys_ops", c10::DispatchKey::Autograd, __FILE__, __LINE__);
    static const bool once_more = (autograd.impl("mha_packed_fwd", &Gate<kPackedName, decltype(mha_packed_fwd)>::autograd),
                                   autograd.impl("mha_paged_decode", &Gate<kDecodeName, decltype(mha_paged_decode)>::autograd),
                                   autograd.impl("rope_paged_store", &Gate<kRopeName, decltype(rope_paged_store)>::autograd),
                                   // whole numbers only: nothing to refuse
                                   autograd.impl("paged_layout", torch::CppFunction::makeFallthrough()), true);
    static torch::Library inplace(torch::Library::IMPL, "recsys_ops", c10::DispatchKey::ADInplaceOrView, __FILE__, __LINE__);
    static const bool once_again = (inplace.impl("rope_paged_store", &rope_paged_store_inplace), true);
    (void)once;
    (void)once_more;
    (void)once_again;
  } catch (const std::exception&) {
    return 1;
  }
  return 0;
}
