// The paged latent cache in cuda_extension (shapes and rules: include/cuda_agent_b200.h):
//   mla_rope_forward(x [T, H, R], positions [T], freq [R/2] fp64, interleaved=False, mscale=1, inverse=False,
//                    out=None) -> out
//   mla_rope_append_forward(q_pe [T, H, 64], c_kv [T, 512], k_pe [T, 64], cache [P, page, 576], page_table,
//                           q_start, kv_len, freq [32], q_out=None, interleaved=False, mscale=1, check=False) -> q_out
//   mla_paged_attention_forward(q [T, H, 576], cache, page_table, q_start, kv_len, softmax_scale, causal=True,
//                               window=0, out=None, lse=None, check=False) -> (out [T, H, 512], lse [T, H])
//   mla_pages_copy(pages [layers, P, page, ...], src, dst, check=False) -> pages
//   mla_pages_extend(page_table, length, refcount, seqs, new_length, page_size, check=False)
//   mla_pages_fork(pages, page_table, length, refcount, src, dst, check=False)
//   mla_pages_free(page_table, length, refcount, seqs, page_size, check=False)
//   mla_pages_compact(pages, page_table, length, refcount, check=False)
// Parts of heads, rows of a joint projection and single layers of a cache are views: x, q_pe, c_kv, k_pe, cache and
// the outputs may have any strides whose last is 1. check=True synchronises and raises on a kernel's status.
// Registered with the other mla ops, by mla_binding.cpp.
#include "binding_common.h"

#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDACachingAllocator.h>

namespace {
using cab_binding::check_cuda_contig;
using cab_binding::check_same_device;
using cab_binding::check_status;
using cab_binding::current_stream;
using cab_binding::ptr;

int dtype_code(const torch::Tensor& t, const char* name, bool allow_f32) {
  if (t.scalar_type() == torch::kBFloat16) return CAB_BF16;
  if (t.scalar_type() == torch::kHalf) return CAB_F16;
  TORCH_CHECK(allow_f32 && t.scalar_type() == torch::kFloat32, name, " must be bfloat16", allow_f32 ? ", float16 or float32" : " or float16",
              ", got ", c10::toString(t.scalar_type()));
  return CAB_F32;
}

void check_view(const torch::Tensor& t, const char* name, int64_t dims) {
  TORCH_CHECK(t.is_cuda(), name, " must be CUDA tensor");
  TORCH_CHECK(t.dim() == dims, name, " must have ", cab_binding::text(dims), " dimensions");
  TORCH_CHECK(t.size(-1) <= 1 || t.stride(-1) == 1, name, ": the last dimension must be contiguous");
}

// Outputs and scratch memory without the dispatcher: a decode step's calls are short.
torch::Tensor fresh(at::IntArrayRef sizes, const torch::Tensor& like, c10::ScalarType type) {
  return at::detail::empty_cuda(sizes, type, like.device(), c10::nullopt);
}
c10::DataPtr scratch_bytes(size_t bytes) { return c10::cuda::CUDACachingAllocator::get()->allocate(bytes); }

// A stride that is never used must not cost the wide accesses.
int64_t stride_of(const torch::Tensor& t, int64_t d) { return t.size(d) <= 1 ? 0 : t.stride(d); }

// Rows of an output [n, m, row] must not lie in one another.
void check_rows_apart(const torch::Tensor& t, const char* name) {
  const int64_t n = t.size(0), m = t.size(1), row = t.size(2), a = t.stride(0), b = t.stride(1);
  const bool outer = (m <= 1 || b >= row) && (n <= 1 || a >= (m - 1) * b + row);
  const bool inner = (n <= 1 || a >= row) && (m <= 1 || b >= (n - 1) * a + row);
  TORCH_CHECK(t.numel() == 0 || outer || inner, name, ": rows of the output overlap");
}

// The bytes of a view: base + any sum of k * stride, k < n, over its dimensions (the last one: the bytes of a row).
struct Dim { int64_t n, stride; };
using Dims = std::vector<Dim>;
int64_t extent(const Dims& dims) {
  int64_t last = 0;
  for (const Dim& d : dims) last += (d.n - 1) * d.stride;
  return last + 1;
}
// Whether two sets of bytes, b's base `shift` behind a's, may have one in common; false is certain. Beside the ranges as a whole
// it knows views that lie in one another's gaps: for a period w, strides that are multiples of w drop out.
bool may_share(const Dims& a, const Dims& b, int64_t shift) {
  if (shift >= extent(a) || -shift >= extent(b)) return false;
  for (const Dims* from : {&a, &b})
    for (const Dim& by : *from) {
      const int64_t w = by.stride;
      if (w <= 1 || by.n <= 1) continue;
      Dims x, y;
      for (const Dim& d : a) if (d.n > 1 && d.stride % w) x.push_back(d);
      for (const Dim& d : b) if (d.n > 1 && d.stride % w) y.push_back(d);
      const int64_t ex = extent(x), ey = extent(y), s = ((shift % w) + w) % w;
      if (ex > w || ey > w) continue;
      if (s >= ex && s + ey <= w) return false;                // each has its own part of the period
      // both within one period, wherever it is taken to begin: alike only where they are alike in it
      if (s + ey <= w && !may_share(x, y, s)) return false;
      if (ex <= s && !may_share(x, y, s - w)) return false;
    }
  return true;
}
Dims bytes_of(const torch::Tensor& t) {
  Dims dims;
  for (int64_t d = 0; d < t.dim(); ++d) dims.push_back({t.size(d), t.stride(d) * (int64_t)t.element_size()});
  dims.push_back({(int64_t)t.element_size(), 1});
  return dims;
}
// Two tensors may share a program's one buffer, but not its bytes. (The ends are kept: a call compares a tensor with many.)
struct Place {
  const torch::Tensor& t;
  const char *begin, *end;
  Place(const torch::Tensor& x) : t(x), begin(static_cast<const char*>(x.data_ptr())), end(begin) {
    if (!x.numel()) return;
    int64_t last = 0;
    const auto n = x.sizes(), stride = x.strides();
    for (size_t d = 0; d < n.size(); ++d) last += (n[d] - 1) * stride[d];
    end = begin + (last + 1) * (int64_t)x.element_size();
  }
};
bool overlap(const Place& a, const Place& b) {
  if (a.begin == a.end || b.begin == b.end) return false;      // no elements
  if (a.begin >= b.end || b.begin >= a.end) return false;      // the common case
  return may_share(bytes_of(a.t), bytes_of(b.t), b.begin - a.begin);
}

// An output is its input itself, or lies elsewhere.
void check_apart(const torch::Tensor& out, const torch::Tensor& in, const char* what) {
  bool same = out.data_ptr() == in.data_ptr() && out.sizes() == in.sizes();
  for (int64_t d = 0; same && d < out.dim(); ++d) same = out.size(d) <= 1 || out.stride(d) == in.stride(d);
  TORCH_CHECK(same || !overlap(out, in), what, " overlap without being the same view");
}

int to_int(int64_t v, const char* name) {
  TORCH_CHECK(v >= 0 && v <= INT32_MAX, name, " too large");
  return static_cast<int>(v);
}

void raise_status(const torch::Tensor& status, const char* op) {
  const int code = status.item<int>();
  const char* text = code == CAB_PAGED_BAD_PAGE      ? "a needed page table entry lies outside the pool, or names a page that counts as free"
                     : code == CAB_PAGED_BAD_INDEX   ? "a listed page or sequence is out of range or listed twice, or q_start descends, does not begin "
                                                       "at 0 or passes the tokens"
                     : code == CAB_PAGED_NO_ROOM     ? "not enough free pages, or a sequence longer than its table row"
                     : code == CAB_PAGED_NOT_EMPTY   ? "a fork's child is in use"
                                                     : "a bounded wait gave up";
  TORCH_CHECK(code == 0, op, ": ", text, " (code ", cab_binding::text(code), ")");
}

cab_mla_paged_batch batch_of(const torch::Tensor& cache, const torch::Tensor& page_table, const torch::Tensor& q_start,
                             const torch::Tensor& kv_len) {
  check_view(cache, "cache", 3);
  TORCH_CHECK(cache.size(2) == 576 && cache.size(0) > 0 && cache.size(1) > 0, "cache must be [pages, page_size, 576]");
  check_cuda_contig(page_table, "page_table", torch::kInt32);
  check_cuda_contig(q_start, "q_start", torch::kInt32);
  check_cuda_contig(kv_len, "kv_len", torch::kInt32);
  TORCH_CHECK(kv_len.dim() == 1, "kv_len must be [batch]");
  const int64_t B = kv_len.size(0);
  TORCH_CHECK(q_start.dim() == 1 && q_start.size(0) == B + 1, "q_start must be [batch + 1]");
  TORCH_CHECK(page_table.dim() == 2 && page_table.size(0) == B && page_table.size(1) > 0,
              "page_table must be [batch, max_pages]");
  for (const torch::Tensor* t : {&page_table, &q_start, &kv_len}) check_same_device(cache, *t, "cache", "every other argument");
  // a dimension of one row has no stride of its own: any valid one does
  const int64_t token = cache.size(1) > 1 ? cache.stride(1) : 576;
  const int64_t page = cache.size(0) > 1 ? cache.stride(0) : std::max<int64_t>(token * cache.size(1), 576);
  TORCH_CHECK(token >= 576 && page >= 576 && token % 8 == 0 && page % 8 == 0,
              "cache: rows must not overlap, and page and row strides must be multiples of 8 elements");
  cab_mla_paged_batch b;
  b.rows = cache.data_ptr();
  b.page_stride = page;
  b.token_stride = token;
  b.num_pages = to_int(cache.size(0), "pages");
  b.page_size = to_int(cache.size(1), "page_size");
  b.page_table = ptr<const int>(page_table);
  b.q_start = ptr<const int>(q_start);
  b.kv_len = ptr<const int>(kv_len);
  b.batch = to_int(B, "batch");
  b.max_pages = to_int(page_table.size(1), "max_pages");
  b.dtype = dtype_code(cache, "cache", false);
  return b;
}

torch::Tensor mla_rope_forward(torch::Tensor x, torch::Tensor positions, torch::Tensor freq, bool interleaved, double mscale,
                               bool inverse, c10::optional<torch::Tensor> out_arg, int config) {
  check_view(x, "x", 3);
  const int dtype = dtype_code(x, "x", true);
  check_cuda_contig(positions, "positions", torch::kInt32);
  check_cuda_contig(freq, "freq", torch::kFloat64);
  const int64_t T = x.size(0), H = x.size(1), R = x.size(2);
  TORCH_CHECK(R > 0 && R % 2 == 0, "x must have an even number of columns");
  TORCH_CHECK(positions.dim() == 1 && positions.size(0) == T, "positions must be [T]");
  TORCH_CHECK(freq.dim() == 1 && freq.size(0) == R / 2, "freq must be [R / 2]");
  check_same_device(x, positions, "x", "positions");
  check_same_device(x, freq, "x", "freq");
  c10::cuda::CUDAGuard guard(x.device());
  torch::Tensor out = out_arg.has_value() ? *out_arg : fresh({T, H, R}, x, x.scalar_type());
  if (out_arg.has_value()) {
    check_view(out, "out", 3);
    TORCH_CHECK(out.sizes() == x.sizes() && out.scalar_type() == x.scalar_type(), "out must have the shape and type of x");
    check_same_device(x, out, "x", "out");
    check_rows_apart(out, "out");
    check_apart(out, x, "x and out");
    for (const torch::Tensor* t : {&positions, &freq}) TORCH_CHECK(!overlap(out, *t), "out must not overlap positions or freq");
  }
  check_status(mla_rope_launcher(out.data_ptr(), x.data_ptr(), ptr<const int>(positions), ptr<const double>(freq), to_int(T, "T"),
                                 to_int(H, "H"), to_int(R, "R"), stride_of(x, 0), stride_of(x, 1), stride_of(out, 0),
                                 stride_of(out, 1), dtype, interleaved, inverse, (float)mscale, config, current_stream()),
               "mla_rope_forward");
  return out;
}

torch::Tensor mla_rope_append_forward(torch::Tensor q_pe, torch::Tensor c_kv, torch::Tensor k_pe, torch::Tensor cache,
                                      torch::Tensor page_table, torch::Tensor q_start, torch::Tensor kv_len,
                                      torch::Tensor freq, c10::optional<torch::Tensor> q_out_arg, bool interleaved,
                                      double mscale, bool check, int config) {
  const cab_mla_paged_batch batch = batch_of(cache, page_table, q_start, kv_len);
  check_view(q_pe, "q_pe", 3);
  check_view(c_kv, "c_kv", 2);
  check_view(k_pe, "k_pe", 2);
  check_cuda_contig(freq, "freq", torch::kFloat64);
  const int64_t T = q_pe.size(0), H = q_pe.size(1);
  TORCH_CHECK(q_pe.size(2) == 64, "q_pe must be [T, H, 64]");
  TORCH_CHECK(c_kv.size(0) == T && c_kv.size(1) == 512, "c_kv must be [T, 512]");
  TORCH_CHECK(k_pe.size(0) == T && k_pe.size(1) == 64, "k_pe must be [T, 64]");
  TORCH_CHECK(freq.dim() == 1 && freq.size(0) == 32, "freq must be [32]");
  for (const torch::Tensor* t : {&q_pe, &c_kv, &k_pe}) {
    TORCH_CHECK(t->scalar_type() == cache.scalar_type(), "q_pe, c_kv and k_pe must have the cache's type");
    check_same_device(cache, *t, "cache", "every other argument");
  }
  check_same_device(cache, freq, "cache", "freq");
  c10::cuda::CUDAGuard guard(cache.device());
  // a fresh output holds zeros where no sequence has a token
  torch::Tensor out = q_out_arg.has_value() ? *q_out_arg : torch::zeros({T, H, 64}, q_pe.options());
  if (q_out_arg.has_value()) {
    check_view(out, "q_out", 3);
    TORCH_CHECK(out.sizes() == q_pe.sizes() && out.scalar_type() == q_pe.scalar_type(), "q_out must have the shape and type of q_pe");
    check_same_device(cache, out, "cache", "q_out");
    check_rows_apart(out, "q_out");
    check_apart(out, q_pe, "q_pe and q_out");
  }
  const Place to(out), rows(cache);
  TORCH_CHECK(!overlap(q_pe, rows) && !overlap(to, rows), "the new rows and q_out must not overlap the cache");
  for (const torch::Tensor* t : {&c_kv, &k_pe, &freq, &page_table, &q_start, &kv_len}) {
    const Place in(*t);
    TORCH_CHECK(!overlap(in, rows), "the new rows, freq and the batch's tables must not overlap the cache");
    // a CTA may have written its rows before another one has read these
    TORCH_CHECK(!overlap(to, in), "q_out must not overlap an input but q_pe");
  }
  torch::Tensor status;
  if (check) status = torch::empty({1}, q_start.options());
  check_status(mla_rope_append_launcher(out.data_ptr(), q_pe.data_ptr(), c_kv.data_ptr(), k_pe.data_ptr(), &batch,
                                        ptr<const double>(freq), to_int(T, "T"), to_int(H, "H"), stride_of(out, 0),
                                        stride_of(out, 1), stride_of(q_pe, 0), stride_of(q_pe, 1), stride_of(c_kv, 0),
                                        stride_of(k_pe, 0), interleaved, (float)mscale, check ? ptr<int>(status) : nullptr,
                                        config, current_stream()),
               "mla_rope_append_forward");
  if (check) raise_status(status, "mla_rope_append_forward");
  return out;
}

std::tuple<torch::Tensor, torch::Tensor> mla_paged_attention_forward(
    torch::Tensor q, torch::Tensor cache, torch::Tensor page_table, torch::Tensor q_start, torch::Tensor kv_len,
    double softmax_scale, bool causal, int64_t window, c10::optional<torch::Tensor> out_arg,
    c10::optional<torch::Tensor> lse_arg, bool check, int config) {
  const cab_mla_paged_batch batch = batch_of(cache, page_table, q_start, kv_len);
  check_cuda_contig(q, "q", cache.scalar_type());
  check_same_device(cache, q, "cache", "q");
  TORCH_CHECK(q.dim() == 3 && q.size(2) == 576 && q.size(1) > 0, "q must be [T, H, 576]");
  TORCH_CHECK(window >= 0 && window <= INT32_MAX, "window must not be negative");
  TORCH_CHECK(softmax_scale > 0, "softmax_scale must be positive");
  const int64_t T = q.size(0), H = q.size(1);
  c10::cuda::CUDAGuard guard(cache.device());
  torch::Tensor out, lse;
  if (out_arg.has_value()) {
    out = *out_arg;
    check_cuda_contig(out, "out", q.scalar_type());
    TORCH_CHECK(out.dim() == 3 && out.size(0) == T && out.size(1) == H && out.size(2) == 512, "out must be [T, H, 512]");
    check_same_device(cache, out, "cache", "out");
    for (const torch::Tensor* t : {&q, &cache, &page_table, &q_start, &kv_len})
      TORCH_CHECK(!overlap(out, *t), "out must not overlap an input");
  } else {
    out = fresh({T, H, 512}, q, q.scalar_type());
    config |= 256;                             // tokens behind the last sequence: zeros in a fresh output
  }
  if (lse_arg.has_value()) {
    lse = *lse_arg;
    check_cuda_contig(lse, "lse", torch::kFloat32);
    TORCH_CHECK(lse.dim() == 2 && lse.size(0) == T && lse.size(1) == H, "lse must be [T, H]");
    check_same_device(cache, lse, "cache", "lse");
    TORCH_CHECK(out_arg.has_value(), "lse is given together with out");
    for (const torch::Tensor* t : {&q, &cache, &page_table, &q_start, &kv_len, &out})
      TORCH_CHECK(!overlap(lse, *t), "lse must not overlap out or an input");
  } else {
    lse = out_arg.has_value() ? torch::full({T, H}, -INFINITY, q.options().dtype(torch::kFloat32))
                              : fresh({T, H}, q, torch::kFloat32);
  }
  const size_t bytes = mla_paged_attention_workspace_bytes(to_int(T, "T"), to_int(H, "H"));
  const c10::DataPtr workspace = scratch_bytes(bytes);
  torch::Tensor status;
  if (check) status = torch::empty({1}, q_start.options());
  check_status(mla_paged_attention_launcher(out.data_ptr(), ptr<float>(lse), q.data_ptr(), &batch, (int)T, (int)H,
                                            (float)softmax_scale, causal, (int)window, workspace.get(),
                                            bytes, check ? ptr<int>(status) : nullptr, config, current_stream()),
               "mla_paged_attention_forward");
  if (check) raise_status(status, "mla_paged_attention_forward");
  return {out, lse};
}

// ------------------------------------------------------------------------------------------------ pages
struct Pages {
  void* data;
  long long layer_stride, page_bytes;
  int layers, num_pages, page_size;
};
Pages pages_of(const torch::Tensor& t) {
  TORCH_CHECK(t.is_cuda(), "pages must be CUDA tensor");
  TORCH_CHECK(t.dim() >= 3 && t.size(1) > 0 && t.size(2) > 0, "pages must be [layers, pages, page_size, ...]");
  int64_t inner = 1;
  for (int64_t d = t.dim() - 1; d >= 1; --d) {
    TORCH_CHECK(t.size(d) <= 1 || t.stride(d) == inner, "pages: the pages of a layer must be contiguous");
    inner *= t.size(d);
  }
  TORCH_CHECK(inner > 0, "pages must not be empty");
  TORCH_CHECK(t.size(0) <= 1 || t.stride(0) >= inner, "pages: layers must not overlap");
  Pages p;
  p.data = t.data_ptr();
  p.layers = to_int(t.size(0), "layers");
  p.num_pages = to_int(t.size(1), "pages");
  p.page_size = to_int(t.size(2), "page_size");
  p.page_bytes = inner / t.size(1) * t.element_size();
  p.layer_stride = (t.size(0) <= 1 ? inner : t.stride(0)) * t.element_size();
  return p;
}

struct PoolArgs { int slots, max_pages, num_pages; };
PoolArgs pool_of(const torch::Tensor& page_table, const torch::Tensor& length, const torch::Tensor& refcount) {
  check_cuda_contig(page_table, "page_table", torch::kInt32);
  check_cuda_contig(length, "length", torch::kInt32);
  check_cuda_contig(refcount, "refcount", torch::kInt32);
  TORCH_CHECK(page_table.dim() == 2 && page_table.numel() > 0, "page_table must be [slots, max_pages]");
  TORCH_CHECK(length.dim() == 1 && length.size(0) == page_table.size(0), "length must be [slots]");
  TORCH_CHECK(refcount.dim() == 1 && refcount.numel() > 0, "refcount must be [pages]");
  check_same_device(page_table, length, "page_table", "length");
  check_same_device(page_table, refcount, "page_table", "refcount");
  TORCH_CHECK(!overlap(page_table, length) && !overlap(page_table, refcount) && !overlap(length, refcount),
              "page_table, length and refcount must not overlap");
  return {to_int(page_table.size(0), "slots"), to_int(page_table.size(1), "max_pages"), to_int(refcount.size(0), "pages")};
}
// A list is read again after the pool changed, so it must lie outside it.
int list_of(const torch::Tensor& t, const char* name, std::initializer_list<const torch::Tensor*> pool) {
  check_cuda_contig(t, name, torch::kInt32);
  TORCH_CHECK(t.dim() == 1, name, " must be a list");
  for (const torch::Tensor* part : pool) {
    check_same_device(t, *part, name, "the pool");
    TORCH_CHECK(!overlap(t, *part), name, " must not overlap the pool");
  }
  return to_int(t.size(0), name);
}
// On the current device and stream.
c10::DataPtr scratch_for(int num_pages, int n) { return scratch_bytes(mla_pages_scratch_bytes(num_pages, n)); }
torch::Tensor status_if(bool check, const torch::Tensor& like) {
  return check ? torch::empty({1}, like.options().dtype(torch::kInt32)) : torch::Tensor();
}
int* status_ptr(const torch::Tensor& t) { return t.defined() ? ptr<int>(t) : nullptr; }

torch::Tensor mla_pages_copy(torch::Tensor pages, torch::Tensor src, torch::Tensor dst, bool check) {
  const Pages p = pages_of(pages);
  const int n = list_of(src, "src", {&pages});
  TORCH_CHECK(list_of(dst, "dst", {&pages}) == n, "src and dst must be equally long");
  c10::cuda::CUDAGuard guard(pages.device());
  const auto scratch = scratch_for(p.num_pages, n);
  const auto status = status_if(check, pages);
  check_status(mla_pages_copy_launcher(p.data, p.layer_stride, p.layers, p.num_pages, p.page_bytes, ptr<const int>(src),
                                       ptr<const int>(dst), n, scratch.get(), status_ptr(status), 0, current_stream()),
               "mla_pages_copy");
  if (check) raise_status(status, "mla_pages_copy");
  return pages;
}

void mla_pages_extend(torch::Tensor page_table, torch::Tensor length, torch::Tensor refcount, torch::Tensor seqs,
                      torch::Tensor new_length, int64_t page_size, bool check) {
  const PoolArgs q = pool_of(page_table, length, refcount);
  const int n = list_of(seqs, "seqs", {&page_table, &length, &refcount});
  TORCH_CHECK(list_of(new_length, "new_length", {&page_table, &length, &refcount}) == n, "seqs and new_length must be equally long");
  c10::cuda::CUDAGuard guard(length.device());
  const auto scratch = scratch_for(q.num_pages, n);
  const auto status = status_if(check, length);
  check_status(mla_pages_extend_launcher(ptr<int>(page_table), ptr<int>(length), ptr<int>(refcount), q.slots, q.max_pages,
                                         q.num_pages, to_int(page_size, "page_size"), ptr<const int>(seqs),
                                         ptr<const int>(new_length), n, scratch.get(), status_ptr(status), 0,
                                         current_stream()),
               "mla_pages_extend");
  if (check) raise_status(status, "mla_pages_extend");
}

void mla_pages_fork(torch::Tensor pages, torch::Tensor page_table, torch::Tensor length, torch::Tensor refcount,
                    torch::Tensor src, torch::Tensor dst, bool check) {
  const Pages p = pages_of(pages);
  const PoolArgs q = pool_of(page_table, length, refcount);
  TORCH_CHECK(q.num_pages == p.num_pages, "refcount must have an entry for each page");
  check_same_device(pages, length, "pages", "length");
  for (const torch::Tensor* t : {&page_table, &length, &refcount})
    TORCH_CHECK(!overlap(*t, pages), "pages must not overlap page_table, length or refcount");
  const int n = list_of(src, "src", {&page_table, &length, &refcount, &pages});
  TORCH_CHECK(list_of(dst, "dst", {&page_table, &length, &refcount, &pages}) == n, "src and dst must be equally long");
  c10::cuda::CUDAGuard guard(length.device());
  const auto scratch = scratch_for(q.num_pages, n);
  const auto status = status_if(check, length);
  check_status(mla_pages_fork_launcher(p.data, p.layer_stride, p.layers, p.page_bytes, ptr<int>(page_table), ptr<int>(length),
                                       ptr<int>(refcount), q.slots, q.max_pages, q.num_pages, p.page_size,
                                       ptr<const int>(src), ptr<const int>(dst), n, scratch.get(), status_ptr(status), 0,
                                       current_stream()),
               "mla_pages_fork");
  if (check) raise_status(status, "mla_pages_fork");
}

void mla_pages_free(torch::Tensor page_table, torch::Tensor length, torch::Tensor refcount, torch::Tensor seqs,
                    int64_t page_size, bool check) {
  const PoolArgs q = pool_of(page_table, length, refcount);
  const int n = list_of(seqs, "seqs", {&page_table, &length, &refcount});
  c10::cuda::CUDAGuard guard(length.device());
  auto status = status_if(check, length);
  check_status(mla_pages_free_launcher(ptr<int>(page_table), ptr<int>(length), ptr<int>(refcount), q.slots, q.max_pages,
                                       q.num_pages, to_int(page_size, "page_size"), ptr<const int>(seqs), n,
                                       status_ptr(status), 0, current_stream()),
               "mla_pages_free");
  if (check) raise_status(status, "mla_pages_free");
}

void mla_pages_compact(torch::Tensor pages, torch::Tensor page_table, torch::Tensor length, torch::Tensor refcount,
                       bool check) {
  const Pages p = pages_of(pages);
  const PoolArgs q = pool_of(page_table, length, refcount);
  TORCH_CHECK(q.num_pages == p.num_pages, "refcount must have an entry for each page");
  check_same_device(pages, length, "pages", "length");
  for (const torch::Tensor* t : {&page_table, &length, &refcount})
    TORCH_CHECK(!overlap(*t, pages), "pages must not overlap page_table, length or refcount");
  c10::cuda::CUDAGuard guard(length.device());
  const auto scratch = scratch_for(q.num_pages, 0);
  const auto status = status_if(check, length);
  check_status(mla_pages_compact_launcher(p.data, p.layer_stride, p.layers, p.page_bytes, ptr<int>(page_table),
                                          ptr<const int>(length), ptr<int>(refcount), q.slots, q.max_pages, q.num_pages,
                                          p.page_size, scratch.get(), status_ptr(status), 0, current_stream()),
               "mla_pages_compact");
  if (check) raise_status(status, "mla_pages_compact");
}
}  // namespace

void register_mla_paged(pybind11::module& m) {
  m.def("mla_rope_forward", &mla_rope_forward, py::arg("x"), py::arg("positions"), py::arg("freq"),
        py::arg("interleaved") = false, py::arg("mscale") = 1.0, py::arg("inverse") = false, py::arg("out") = py::none(),
        py::arg("config") = 0);
  m.def("mla_rope_append_forward", &mla_rope_append_forward, py::arg("q_pe"), py::arg("c_kv"), py::arg("k_pe"),
        py::arg("cache"), py::arg("page_table"), py::arg("q_start"), py::arg("kv_len"), py::arg("freq"),
        py::arg("q_out") = py::none(), py::arg("interleaved") = false, py::arg("mscale") = 1.0, py::arg("check") = false,
        py::arg("config") = 0);
  m.def("mla_paged_attention_forward", &mla_paged_attention_forward, py::arg("q"), py::arg("cache"), py::arg("page_table"),
        py::arg("q_start"), py::arg("kv_len"), py::arg("softmax_scale"), py::arg("causal") = true, py::arg("window") = 0,
        py::arg("out") = py::none(), py::arg("lse") = py::none(), py::arg("check") = false, py::arg("config") = 0);
  m.def("mla_pages_copy", &mla_pages_copy, py::arg("pages"), py::arg("src"), py::arg("dst"), py::arg("check") = false);
  m.def("mla_pages_extend", &mla_pages_extend, py::arg("page_table"), py::arg("length"), py::arg("refcount"),
        py::arg("seqs"), py::arg("new_length"), py::arg("page_size"), py::arg("check") = false);
  m.def("mla_pages_fork", &mla_pages_fork, py::arg("pages"), py::arg("page_table"), py::arg("length"), py::arg("refcount"),
        py::arg("src"), py::arg("dst"), py::arg("check") = false);
  m.def("mla_pages_free", &mla_pages_free, py::arg("page_table"), py::arg("length"), py::arg("refcount"), py::arg("seqs"),
        py::arg("page_size"), py::arg("check") = false);
  m.def("mla_pages_compact", &mla_pages_compact, py::arg("pages"), py::arg("page_table"), py::arg("length"),
        py::arg("refcount"), py::arg("check") = false);
}
