// torch.ops.flashoverlap_op.{prompt_attention, paged_attention, cache_append, copy_pages}: checks of the arguments, and the
// launches.  What a tensor on the GPU holds (lengths, page numbers) is not read here: the kernels check it themselves.
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/library.h>

#include <atomic>
#include <cmath>
#include <cstring>
#include <limits>
#include <mutex>
#include <unordered_set>

#include "../kernels/attention.h"
#include "checks.h"

namespace fo {

namespace {

void check_launch(cudaError_t e, const char* op) {
  TORCH_CHECK(e == cudaSuccess, op, " launch failed: ", cudaGetErrorString(e));
}

// There are no derivatives: neither a gradient nor a forward-mode tangent is dropped without a word.
void check_no_derivative(const at::Tensor& t, const char* name) {
  TORCH_CHECK(!(at::GradMode::is_enabled() && t.requires_grad()), name,
              " requires a gradient: these operators have no backward pass, call them under torch.no_grad()");
  TORCH_CHECK(!t._fw_grad(0).defined(), name, " carries a forward-mode tangent: these operators have no derivative");
}
// A change that autograd is to know of.
void count_change(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// [.., head_dim] rows on 16-byte boundaries.  A dimension of one entry may have any stride.
void check_rows(const at::Tensor& t, const char* name, int64_t dims) {
  TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
  TORCH_CHECK(t.dim() == dims, name, " must be ", dims, "-D, got ", t.dim(), "-D");
  dtype_of(t);
  check_no_derivative(t, name);
  TORCH_CHECK(t.size(-1) <= 1 || t.stride(-1) == 1, name, ": the last dimension must be contiguous");
  for (int64_t d = 0; d + 1 < dims; ++d) {
    TORCH_CHECK(t.size(d) <= 1 || t.stride(d) % 8 == 0, name, ": strides must be multiples of 16 bytes");
  }
  TORCH_CHECK(t.numel() == 0 || reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0, name,
              " must start on a 16-byte boundary");
}
void check_same(const at::Tensor& t, const at::Tensor& like, const char* name) {
  TORCH_CHECK(t.scalar_type() == like.scalar_type(), name, " must have the dtype of the other tensors");
  TORCH_CHECK(t.device() == like.device(), name, " must be on the device of the other tensors");
}
void check_ints(const at::Tensor& t, const char* name, int64_t n, const at::Tensor& like) {
  TORCH_CHECK(t.scalar_type() == at::kInt, name, " must be int32");
  TORCH_CHECK(t.is_cuda() && t.device() == like.device(), name, " must be on the device of the other tensors");
  TORCH_CHECK(t.dim() == 1 && t.size(0) == n, name, " must hold ", n, " entries");
  TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
}
// Bytes from the first to the last value of a tensor.
std::pair<const char*, const char*> extent(const at::Tensor& t) {
  const char* lo = static_cast<const char*>(t.data_ptr());
  if (t.numel() == 0) return {lo, lo};
  int64_t last = 0;
  for (int64_t d = 0; d < t.dim(); ++d) last += (t.size(d) - 1) * t.stride(d);
  return {lo, lo + (last + 1) * static_cast<int64_t>(t.element_size())};
}
void check_apart(const at::Tensor& out, const at::Tensor& in, const char* out_name, const char* in_name) {
  const auto a = extent(out), b = extent(in);
  TORCH_CHECK(a.second <= b.first || b.second <= a.first, out_name, " must not share memory with ", in_name);
}
int64_t stride_of(const at::Tensor& t, int64_t d) { return t.size(d) <= 1 ? 0 : t.stride(d); }

void check_head_dim(int64_t dim) {
  TORCH_CHECK(dim == 64 || dim == 128, "head_dim must be 64 or 128, got ", dim);
}
void check_heads(int64_t heads, int64_t kv_heads) {
  TORCH_CHECK(kv_heads > 0 && heads > 0 && heads % kv_heads == 0, "query heads (", heads,
              ") must be a multiple of key and value heads (", kv_heads, ")");
  TORCH_CHECK(heads / kv_heads <= 128, "at most 128 query heads may share a key and value head");
}
void check_window(int64_t window, int64_t sinks) {
  TORCH_CHECK(window >= 0 && window <= std::numeric_limits<int>::max(), "window must be zero (none) or positive");
  TORCH_CHECK(sinks >= 0 && sinks <= std::numeric_limits<int>::max(), "sinks must not be negative");
}
float scale_or(c10::optional<double> scale, int64_t dim) {
  const float s = static_cast<float>(scale.has_value() ? *scale : 1.0 / std::sqrt(static_cast<double>(dim)));
  TORCH_CHECK(std::isfinite(s), "scale must be a finite number");
  return s;
}

// [pages, 2, kv_heads, page_size, head_dim]; a page is contiguous, pages may lie apart (one layer of a cache of several).
PageLayout check_cache(const at::Tensor& cache) {
  check_rows(cache, "cache", 5);
  TORCH_CHECK(cache.size(1) == 2, "cache must be [pages, 2, kv_heads, page_size, head_dim]");
  const int64_t kv = cache.size(2), page = cache.size(3), dim = cache.size(4);
  TORCH_CHECK(kv > 0 && page > 0 && dim > 0 && dim % 8 == 0, "cache: empty pages, or head_dim no multiple of 8");
  TORCH_CHECK(cache.size(0) <= std::numeric_limits<int>::max(), "cache has too many pages");
  TORCH_CHECK(kv * page * dim < (1ll << 30), "cache: a page holds too much");
  const int64_t inner[4] = {kv * page * dim, page * dim, dim, 1};
  for (int64_t d = 1; d < 5; ++d) {
    TORCH_CHECK(cache.size(d) <= 1 || cache.stride(d) == inner[d - 1], "cache: a page must be contiguous");
  }
  TORCH_CHECK(cache.size(0) <= 1 || cache.stride(0) >= 2 * inner[0], "cache: pages must not overlap");
  PageLayout l;
  l.page_stride = stride_of(cache, 0);
  l.page_size = static_cast<int>(page);
  l.head_dim = static_cast<int>(dim);
  l.kv_heads = static_cast<int>(kv);
  l.pages = static_cast<int>(cache.size(0));
  l.by_page = FastDiv(static_cast<uint32_t>(page));
  return l;
}
void check_table(const at::Tensor& table, int64_t seqs, const PageLayout& l, const at::Tensor& like) {
  TORCH_CHECK(table.scalar_type() == at::kInt, "page_table must be int32");
  TORCH_CHECK(table.is_cuda() && table.device() == like.device(), "page_table must be on the device of the other tensors");
  TORCH_CHECK(table.dim() == 2 && table.size(0) == seqs, "page_table must be [", seqs, ", pages of a sequence]");
  TORCH_CHECK(table.size(1) <= 1 || table.stride(1) == 1, "page_table: a row must be contiguous");
  TORCH_CHECK(table.size(1) * static_cast<int64_t>(l.page_size) <= std::numeric_limits<int>::max() - 1024,
              "page_table covers more than 2^31 - 1024 tokens");
}

// What the prompt kernel reports of waits that ran out: a word for each device, in host memory that all devices see under
// its own address, read before each call without waiting for anything.  Allocated at the first call, also where that is
// being captured, and kept.
constexpr int kStatusDevices = 64;
std::atomic<StatusWord*> status_words{nullptr};
std::atomic<int64_t> prompt_wait_ns{10000000000};

StatusWord* status_of(int device) {
  TORCH_CHECK(device >= 0 && device < kStatusDevices, "attention: device number out of range");
  static std::mutex mu;
  if (status_words.load(std::memory_order_acquire) == nullptr) {
    std::lock_guard<std::mutex> lock(mu);
    if (status_words.load() == nullptr) {
      cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;  // the allocation is no part of a graph
      check_launch(cudaThreadExchangeStreamCaptureMode(&mode), "attention: status");
      void* words = nullptr;
      const size_t bytes = kStatusDevices * sizeof(StatusWord);
      const cudaError_t e = cudaHostAlloc(&words, bytes, cudaHostAllocMapped | cudaHostAllocPortable);
      cudaThreadExchangeStreamCaptureMode(&mode);
      check_launch(e, "attention: status");
      std::memset(words, 0, bytes);
      status_words.store(static_cast<StatusWord*>(words), std::memory_order_release);
    }
  }
  return status_words.load() + device;
}
void check_previous(StatusWord* word, const char* op) {
  const volatile StatusWord* s = word;
  TORCH_CHECK(s->code == ST_OK, op, ": a wait of an earlier call of prompt_attention on this device ran out (warp ", s->where,
              " of CTA ", s->seen, "); rows that it had not finished are NaN (attention_reset() clears the state)");
}

}  // namespace

// {code, warp, CTA} of what has been reported for a device since the last reset; code 0: nothing.  Does not wait.
static std::vector<int64_t> attention_status_op(int64_t device) {
  if (status_words.load() == nullptr) return {ST_OK, 0, 0};
  const volatile StatusWord* s = status_of(static_cast<int>(device));
  return {s->code, s->where, s->seen};
}
static void attention_reset_op(int64_t device) {
  if (status_words.load() == nullptr) return;
  std::memset(status_of(static_cast<int>(device)), 0, sizeof(StatusWord));
}
// Limit of the waits in kernels launched from now on; returns the one before.
static int64_t attention_set_timeout_ns_op(int64_t ns) {
  TORCH_CHECK(ns >= 0 && ns <= 3600000000000, "timeout must be at most an hour");
  return prompt_wait_ns.exchange(ns);
}

// out[b, t, h] of q [batch, sq, heads, head_dim], k and v [batch, sk, kv_heads, head_dim]; see attention.h.
static void prompt_attention_op(at::Tensor q, at::Tensor k, at::Tensor v, at::Tensor out, int64_t window, int64_t sinks,
                                c10::optional<at::Tensor> lengths, c10::optional<double> scale) {
  check_rows(q, "q", 4);
  check_rows(k, "k", 4);
  check_rows(v, "v", 4);
  check_rows(out, "out", 4);
  check_same(k, q, "k");
  check_same(v, q, "v");
  check_same(out, q, "out");
  const int64_t batch = q.size(0), sq = q.size(1), heads = q.size(2), dim = q.size(3), sk = k.size(1), kv = k.size(2);
  check_head_dim(dim);
  check_heads(heads, kv);
  check_window(window, sinks);
  TORCH_CHECK(k.sizes() == v.sizes(), "k and v must have one shape");
  TORCH_CHECK(k.size(0) == batch && k.size(3) == dim, "k and v must have q's batch and head_dim");
  TORCH_CHECK(sq <= sk, "the queries are the last tokens of the sequence: ", sq, " queries, ", sk, " keys");
  TORCH_CHECK(sk <= (1ll << 30), "at most 2^30 tokens");
  TORCH_CHECK(batch * heads <= std::numeric_limits<int>::max(), "batch too large");
  TORCH_CHECK(out.sizes() == q.sizes() && out.is_contiguous(), "out must be contiguous and have the shape of q");
  check_apart(out, q, "out", "q");
  check_apart(out, k, "out", "k");
  check_apart(out, v, "out", "v");
  PromptParams p{};
  if (lengths.has_value()) {
    check_ints(*lengths, "lengths", batch, q);
    check_apart(out, *lengths, "out", "lengths");
    p.lengths = lengths->data_ptr<int>();
  }
  p.q = q.data_ptr();
  p.k = k.data_ptr();
  p.v = v.data_ptr();
  p.out = out.data_ptr();
  for (int d = 0; d < 3; ++d) {
    p.q_stride[d] = stride_of(q, d);
    p.k_stride[d] = stride_of(k, d);
    p.v_stride[d] = stride_of(v, d);
  }
  p.batch = static_cast<int>(batch);
  p.sq = static_cast<int>(sq);
  p.sk = static_cast<int>(sk);
  p.heads = static_cast<int>(heads);
  p.kv_heads = static_cast<int>(kv);
  p.head_dim = static_cast<int>(dim);
  p.window = static_cast<int>(window);
  p.sinks = static_cast<int>(sinks);
  p.scale = scale_or(scale, dim);
  c10::cuda::CUDAGuard guard(q.device());
  p.status = status_of(q.get_device());
  check_previous(p.status, "prompt_attention");
  p.wait_ns = static_cast<unsigned long long>(prompt_wait_ns.load());
  // from the caching allocator, for this call alone: calls on other streams and captured graphs have their own
  at::Tensor workspace;
  if (const size_t bytes = prompt_workspace_bytes(p)) {
    workspace = at::empty({static_cast<int64_t>(bytes)}, q.options().dtype(at::kByte));
    p.workspace = workspace.data_ptr();
  }
  count_change(out);
  check_launch(launch_prompt_attention(p, dtype_of(q), at::cuda::getCurrentCUDAStream().stream()), "prompt_attention");
}

static at::Tensor prompt_attention_new_op(at::Tensor q, at::Tensor k, at::Tensor v, int64_t window, int64_t sinks,
                                          c10::optional<at::Tensor> lengths, c10::optional<double> scale) {
  TORCH_CHECK(q.is_cuda(), "q must be a CUDA tensor");
  at::Tensor out = at::empty(q.sizes(), q.options());
  prompt_attention_op(q, k, v, out, window, sinks, lengths, scale);
  return out;
}

// out[s, h] of q [seqs, heads, head_dim]: the last token of every sequence, which has lengths[s] tokens in the cache.
static void paged_attention_op(at::Tensor q, at::Tensor cache, at::Tensor page_table, at::Tensor lengths, at::Tensor out,
                               int64_t window, int64_t sinks, c10::optional<double> scale) {
  check_rows(q, "q", 3);
  check_rows(out, "out", 3);
  PagedParams p{};
  p.pages = check_cache(cache);
  check_same(cache, q, "cache");
  check_same(out, q, "out");
  const int64_t seqs = q.size(0), heads = q.size(1), dim = q.size(2), kv = p.pages.kv_heads;
  check_head_dim(dim);
  TORCH_CHECK(p.pages.head_dim == dim, "cache and q have different head_dim");
  check_heads(heads, kv);
  check_window(window, sinks);
  check_table(page_table, seqs, p.pages, q);
  check_ints(lengths, "lengths", seqs, q);
  TORCH_CHECK(out.sizes() == q.sizes() && out.is_contiguous(), "out must be contiguous and have the shape of q");
  check_apart(out, q, "out", "q");
  check_apart(out, cache, "out", "cache");
  check_apart(out, page_table, "out", "page_table");
  check_apart(out, lengths, "out", "lengths");
  const int64_t width = page_table.size(1);
  TORCH_CHECK(seqs * heads * (width * p.pages.page_size / 64 + 3) <= std::numeric_limits<int>::max(),
              "too many tokens in one call");
  p.q = q.data_ptr();
  p.cache = cache.data_ptr();
  p.out = out.data_ptr();
  p.table = page_table.data_ptr<int>();
  p.lengths = lengths.data_ptr<int>();
  p.q_stride[0] = stride_of(q, 0);
  p.q_stride[1] = stride_of(q, 1);
  p.table_stride = stride_of(page_table, 0);
  p.seqs = static_cast<int>(seqs);
  p.heads = static_cast<int>(heads);
  p.width = static_cast<int>(width);
  p.window = static_cast<int>(window);
  p.sinks = static_cast<int>(sinks);
  p.scale = scale_or(scale, dim);
  if (seqs == 0) return;
  c10::cuda::CUDAGuard guard(q.device());
  at::Tensor workspace;  // as above
  if (const size_t bytes = paged_workspace_bytes(p)) {
    workspace = at::empty({static_cast<int64_t>(bytes)}, q.options().dtype(at::kByte));
    p.workspace = workspace.data_ptr();
  }
  count_change(out);
  check_launch(launch_paged_attention(p, dtype_of(q), at::cuda::getCurrentCUDAStream().stream()), "paged_attention");
}

static at::Tensor paged_attention_new_op(at::Tensor q, at::Tensor cache, at::Tensor page_table, at::Tensor lengths,
                                         int64_t window, int64_t sinks, c10::optional<double> scale) {
  TORCH_CHECK(q.is_cuda(), "q must be a CUDA tensor");
  at::Tensor out = at::empty(q.sizes(), q.options());
  paged_attention_op(q, cache, page_table, lengths, out, window, sinks, scale);
  return out;
}

// Stores token i of sequence s (k and v [seqs, tokens, kv_heads, head_dim]) at position starts[s] + i, for i < counts[s].
static void cache_append_op(at::Tensor k, at::Tensor v, at::Tensor cache, at::Tensor page_table, at::Tensor starts,
                            c10::optional<at::Tensor> counts) {
  check_rows(k, "k", 4);
  check_rows(v, "v", 4);
  AppendParams p{};
  p.pages = check_cache(cache);
  check_same(v, k, "v");
  check_same(cache, k, "cache");
  TORCH_CHECK(k.sizes() == v.sizes(), "k and v must have one shape");
  const int64_t seqs = k.size(0), tokens = k.size(1);
  TORCH_CHECK(k.size(2) == p.pages.kv_heads && k.size(3) == p.pages.head_dim, "k and v must have the cache's heads");
  TORCH_CHECK(seqs * tokens < (1ll << 31), "too many tokens in one call");
  check_table(page_table, seqs, p.pages, k);
  check_ints(starts, "starts", seqs, k);
  check_apart(cache, k, "cache", "k");
  check_apart(cache, v, "cache", "v");
  check_apart(cache, page_table, "cache", "page_table");
  check_apart(cache, starts, "cache", "starts");
  if (counts.has_value()) {
    check_ints(*counts, "counts", seqs, k);
    check_apart(cache, *counts, "cache", "counts");
    p.counts = counts->data_ptr<int>();
  }
  p.k = k.data_ptr();
  p.v = v.data_ptr();
  p.cache = cache.data_ptr();
  p.table = page_table.data_ptr<int>();
  p.starts = starts.data_ptr<int>();
  for (int d = 0; d < 3; ++d) {
    p.k_stride[d] = stride_of(k, d);
    p.v_stride[d] = stride_of(v, d);
  }
  p.table_stride = stride_of(page_table, 0);
  p.seqs = static_cast<int>(seqs);
  p.tokens = static_cast<int>(tokens);
  p.width = static_cast<int>(page_table.size(1));
  c10::cuda::CUDAGuard guard(k.device());
  count_change(cache);
  check_launch(launch_cache_append(p, at::cuda::getCurrentCUDAStream().stream()), "cache_append");
}

// moves [n, 2] on the CPU: page moves[i][0] of `cache` is copied to page moves[i][1].  Any tensor whose entries along the
// first dimension are contiguous is a cache here.
template <typename Int>
static void read_moves(const at::Tensor& moves, int64_t pages, std::vector<int>& list) {
  const Int* at = moves.const_data_ptr<Int>();
  const int64_t n = moves.size(0), row = moves.stride(0), col = moves.stride(1);
  list.resize(static_cast<size_t>(2 * n));
  std::vector<bool> target(static_cast<size_t>(pages), false);
  for (int64_t i = 0; i < n; ++i) {
    for (int64_t e = 0; e < 2; ++e) {
      const int64_t page = at[i * row + e * col];
      TORCH_CHECK(page >= 0 && page < pages, "moves names page ", page, ", outside [0, ", pages, ")");
      list[static_cast<size_t>(2 * i + e)] = static_cast<int>(page);
    }
    const size_t to = static_cast<size_t>(list[static_cast<size_t>(2 * i + 1)]);
    TORCH_CHECK(!target[to], "moves writes page ", to, " twice");
    target[to] = true;
  }
  for (int64_t i = 0; i < n; ++i) {
    const size_t from = static_cast<size_t>(list[static_cast<size_t>(2 * i)]);
    TORCH_CHECK(!target[from], "moves reads page ", from, " and writes it");
  }
}
static void copy_pages_op(at::Tensor cache, at::Tensor moves) {
  TORCH_CHECK(cache.dim() >= 1 && cache.size(0) <= std::numeric_limits<int>::max(), "cache must have pages");
  TORCH_CHECK(moves.device().is_cpu(), "moves must be a CPU tensor");
  TORCH_CHECK(moves.scalar_type() == at::kInt || moves.scalar_type() == at::kLong, "moves must be int32 or int64");
  TORCH_CHECK(moves.dim() == 2 && moves.size(1) == 2, "moves must be [n, 2]: from page, to page");
  std::vector<int> list;
  if (moves.scalar_type() == at::kInt) read_moves<int>(moves, cache.size(0), list);
  else read_moves<int64_t>(moves, cache.size(0), list);
  check_no_derivative(cache, "cache");
  TORCH_CHECK(cache.is_cuda(), "cache must be a CUDA tensor");
  if (list.empty()) return;
  int64_t values = 1;
  for (int64_t d = cache.dim() - 1; d >= 1; --d) {
    TORCH_CHECK(cache.size(d) == 1 || cache.stride(d) == values, "cache: a page must be contiguous");
    values *= cache.size(d);
  }
  const int64_t size = static_cast<int64_t>(cache.element_size());
  const int64_t bytes = values * size, stride = cache.size(0) > 1 ? cache.stride(0) * size : bytes;
  if (bytes == 0) return;
  TORCH_CHECK(stride >= bytes, "cache: pages must not overlap");
  TORCH_CHECK(bytes % 16 == 0 && stride % 16 == 0 && reinterpret_cast<uintptr_t>(cache.data_ptr()) % 16 == 0,
              "cache: pages must begin and end on 16-byte boundaries");
  TORCH_CHECK(bytes < (1ll << 33), "cache: a page holds too much");
  c10::cuda::CUDAGuard guard(cache.device());
  count_change(cache);
  check_launch(launch_copy_pages(cache.data_ptr(), bytes, stride, list.data(), static_cast<int>(list.size() / 2),
                                 at::cuda::getCurrentCUDAStream().stream()),
               "copy_pages");
}

// Where a paged token lies, by the functions the kernels use: {page, place in the page, offset of its key in values} for
// position `pos` of a sequence with the given table row (page -1: nowhere).  For tests and tools, without a GPU.
static std::vector<int64_t> page_place_op(std::vector<int64_t> row, int64_t pos, int64_t pages, int64_t kv_heads,
                                          int64_t page_size, int64_t head_dim, int64_t head) {
  TORCH_CHECK(pos >= 0 && pos <= std::numeric_limits<int>::max() && pages >= 0 && kv_heads > 0 && page_size > 0 &&
                  head_dim > 0 && head >= 0 && head < kv_heads, "page_place: bad arguments");
  PageLayout l;
  l.page_stride = 2 * kv_heads * page_size * head_dim;
  l.page_size = static_cast<int>(page_size);
  l.head_dim = static_cast<int>(head_dim);
  l.kv_heads = static_cast<int>(kv_heads);
  l.pages = static_cast<int>(pages);
  l.by_page = FastDiv(static_cast<uint32_t>(page_size));
  std::vector<int> r;
  for (int64_t x : row) {
    r.push_back(static_cast<int>(std::max<int64_t>(std::min<int64_t>(x, std::numeric_limits<int>::max()), -1)));
  }
  int place = 0;
  const int page = l.find(r.data(), static_cast<int>(r.size()), static_cast<int>(pos), place);
  return {page, place, page < 0 ? -1 : l.key_offset(page, static_cast<int>(head), place)};
}
// The tokens that position i sees in a sequence of `length` tokens, by the function the kernels use.
static std::vector<int64_t> seen_tokens_op(int64_t i, int64_t length, int64_t window, int64_t sinks) {
  TORCH_CHECK(i >= 0 && i < (1 << 20) && length >= 0 && length <= std::numeric_limits<int>::max(), "seen_tokens: bad arguments");
  check_window(window, sinks);
  std::vector<int64_t> out;
  for (int64_t j = 0; j <= i + 1; ++j) {
    if (is_visible(static_cast<int>(i), static_cast<int>(j), static_cast<int>(length), static_cast<int>(window),
                   static_cast<int>(sinks))) out.push_back(j);
  }
  return out;
}
// First tokens of the tiles of `tile` tokens that the positions [p0, p1] of a sequence look at, by the function the kernels use.
static std::vector<int64_t> seen_tiles_op(int64_t p0, int64_t p1, int64_t length, int64_t window, int64_t sinks, int64_t tile,
                                          int64_t align) {
  TORCH_CHECK(p0 >= -1 && p0 <= p1 && p1 < std::numeric_limits<int>::max() && length >= 0 &&
                  length <= std::numeric_limits<int>::max() - 1024 && tile > 0 && tile <= 1024 && align > 0 && tile % align == 0, "seen_tiles: bad arguments");
  check_window(window, sinks);
  const SeenTiles t = seen_tiles(static_cast<int>(p0), static_cast<int>(p1), static_cast<int>(length),
                                 static_cast<int>(window), static_cast<int>(sinks), static_cast<int>(tile),
                                 static_cast<int>(align));
  std::vector<int64_t> out;
  for (int i = 0; i < t.count(); ++i) out.push_back(t.start(i));
  return out;
}

}  // namespace fo

TORCH_LIBRARY_FRAGMENT(flashoverlap_op, m) {
  // (a!): what a call changes
  m.def("prompt_attention(Tensor q, Tensor k, Tensor v, Tensor(a!) out, int window, int sinks, Tensor? lengths, float? scale)"
        " -> ()", &fo::prompt_attention_op);
  m.def("prompt_attention_new(Tensor q, Tensor k, Tensor v, int window, int sinks, Tensor? lengths, float? scale) -> Tensor",
        &fo::prompt_attention_new_op);
  m.def("paged_attention(Tensor q, Tensor cache, Tensor page_table, Tensor lengths, Tensor(a!) out, int window, int sinks,"
        " float? scale) -> ()", &fo::paged_attention_op);
  m.def("paged_attention_new(Tensor q, Tensor cache, Tensor page_table, Tensor lengths, int window, int sinks, float? scale)"
        " -> Tensor", &fo::paged_attention_new_op);
  m.def("cache_append(Tensor k, Tensor v, Tensor(a!) cache, Tensor page_table, Tensor starts, Tensor? counts) -> ()",
        &fo::cache_append_op);
  m.def("copy_pages(Tensor(a!) cache, Tensor moves) -> ()", &fo::copy_pages_op);
  m.def("attention_status", &fo::attention_status_op);
  m.def("attention_reset", &fo::attention_reset_op);
  m.def("attention_set_timeout_ns", &fo::attention_set_timeout_ns_op);
  m.def("page_place", &fo::page_place_op);
  m.def("seen_tokens", &fo::seen_tokens_op);
  m.def("seen_tiles", &fo::seen_tiles_op);
}
