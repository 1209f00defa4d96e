// Attention over keys and values of a decoder: launch interface of the kernels (no PyTorch types), and the rules that the
// kernels and the host share.
//
//   visible(i, j) = j <= i < length and (window == 0 or j > i - window or j < sinks)
//   out_i = sum_j exp(scale q_i k_j) v_j / sum_j exp(scale q_i k_j) over the visible j, zero where there is none.
//
// A cache is [pages, 2, kv_heads, page_size, head_dim], keys at 0 and values at 1: what a page holds for one head is one
// contiguous block, and a page is one contiguous block of its own.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "gemm_launch.h"

namespace fo {

// n / d for 0 <= n < 2^31 and a divisor that is known before the launch: a multiplication by ceil(2^(31 + l) / d), l =
// ceil(log2 d), and a shift (Granlund and Montgomery, Division by invariant integers using multiplication, 1994).
struct FastDiv {
  uint32_t d = 1, mul = 0, shift = 0;
  FastDiv() = default;
  explicit FastDiv(uint32_t divisor) : d(divisor) {
    if (d <= 1) return;
    uint32_t l = 0;
    while ((1ull << l) < d) ++l;
    mul = static_cast<uint32_t>(((1ull << (31 + l)) + d - 1) / d);
    shift = l - 1;
  }
  __host__ __device__ uint32_t div(uint32_t n) const {
    if (d <= 1) return n;
#ifdef __CUDA_ARCH__
    return __umulhi(n, mul) >> shift;
#else
    return static_cast<uint32_t>((static_cast<uint64_t>(n) * mul) >> 32) >> shift;
#endif
  }
};

// Where the tokens of a paged sequence lie.
struct PageLayout {
  long long page_stride;  // values from one page to the next (a page of several layers holds more than this cache's part)
  int page_size, head_dim, kv_heads, pages;
  FastDiv by_page;
  // Value offset of the first key of (page, head, place in the page); its value stands value_offset() behind it.
  __host__ __device__ long long key_offset(int page, int head, int place) const {
    return static_cast<long long>(page) * page_stride +
           (static_cast<long long>(head) * page_size + place) * head_dim;
  }
  __host__ __device__ long long value_offset() const { return static_cast<long long>(kv_heads) * page_size * head_dim; }
  // Page and place of position `pos` (>= 0) of a sequence whose table row is `row`; -1 if the row ends before it or names a
  // page that the cache does not have.
  __host__ __device__ int find(const int* row, int width, int pos, int& place) const {
    const int slot = static_cast<int>(by_page.div(static_cast<uint32_t>(pos)));
    place = pos - slot * page_size;
    if (slot >= width) return -1;
    return has(row[slot]) ? row[slot] : -1;
  }
  __host__ __device__ bool has(int page) const { return page >= 0 && page < pages; }
};

// Tiles of `tile` tokens: the first n_sink of the sequence, then n from token `first` on.
struct SeenTiles {
  int n_sink, first, n, tile;
  __host__ __device__ int count() const { return n_sink + n; }
  __host__ __device__ int start(int i) const { return i < n_sink ? i * tile : first + (i - n_sink) * tile; }
};
// The tiles that hold the tokens which some position of [p0, p1] sees in a sequence of `length` tokens, p0 <= p1.  A window's
// tiles begin with the first token it shows, rounded down to a multiple of `align` (which divides `tile`), and not at a
// multiple of the tile.
__host__ __device__ inline SeenTiles seen_tiles(int p0, int p1, int length, int window, int sinks, int tile, int align) {
  SeenTiles t;
  const int end = p1 < length ? p1 + 1 : length;  // behind the last visible token
  // (p0 - window may be far below zero, never below the smallest int)
  const int lo = window > 0 && p0 >= window ? p0 - window + 1 : 0;
  int sink = sinks < lo ? sinks : lo;  // visible tokens in front of the window
  if (sink > end) sink = end;
  t.tile = tile;
  t.n_sink = sink > 0 ? (sink - 1) / tile + 1 : 0;
  const int behind = t.n_sink * tile;  // (below the largest int: a tile more than a length of at most 2^31 - 1024)
  t.first = lo > behind ? lo - lo % align : behind;
  if (t.first < behind) t.first = behind;
  t.n = end > t.first ? (end - t.first - 1) / tile + 1 : 0;
  return t;
}
__host__ __device__ inline bool is_visible(int i, int j, int length, int window, int sinks) {
  return j <= i && i < length && (window == 0 || i - j < window || j < sinks);
}

struct PromptParams {
  const void *q, *k, *v;
  void* out;           // [batch, sq, heads, head_dim], contiguous
  const int* lengths;  // [batch] or null: every sequence has sk tokens
  long long q_stride[3], k_stride[3], v_stride[3];  // values: batch, token, head
  int batch, sq, sk, heads, kv_heads, head_dim;
  int window, sinks;
  float scale;
  void* workspace;  // prompt_workspace_bytes(), 16-byte aligned, contents arbitrary
  // Limit of each wait inside the kernel.  A CTA whose wait runs out writes `status` (mapped host memory, ST_TIMEOUT_PIPE, the
  // warp that gave up and the CTA) and makes the rows that it has taken and not finished NaN.
  unsigned long long wait_ns;
  StatusWord* status;
};
size_t prompt_workspace_bytes(const PromptParams& p);
// head_dim 64 or 128, heads a multiple of kv_heads (at most 128 times), sq <= sk; addresses and strides in whole 16 bytes.
cudaError_t launch_prompt_attention(const PromptParams& p, DType dt, cudaStream_t stream);

struct PagedParams {
  const void *q, *cache;
  void* out;  // [seqs, heads, head_dim], contiguous
  const int *table, *lengths;
  long long q_stride[2];  // values: sequence, head
  long long table_stride;
  PageLayout pages;
  int seqs, heads, width;
  int window, sinks;
  float scale;
  void* workspace;  // paged_workspace_bytes(), 16-byte aligned, contents arbitrary
};
size_t paged_workspace_bytes(const PagedParams& p);
cudaError_t launch_paged_attention(const PagedParams& p, DType dt, cudaStream_t stream);

struct AppendParams {
  const void *k, *v;
  void* cache;
  const int *table, *starts, *counts;  // counts may be null
  long long k_stride[3], v_stride[3];  // values: sequence, token, head
  long long table_stride;
  PageLayout pages;
  int seqs, tokens, width;
};
cudaError_t launch_cache_append(const AppendParams& p, cudaStream_t stream);

// Copies page moves[2 i] to page moves[2 i + 1] for every i < n; `moves` is read before the call returns.  No page may be a
// destination twice, or a source and a destination (the caller has checked it).
cudaError_t launch_copy_pages(void* cache, long long page_bytes, long long page_stride_bytes, const int* moves, int n,
                              cudaStream_t stream);

}  // namespace fo
