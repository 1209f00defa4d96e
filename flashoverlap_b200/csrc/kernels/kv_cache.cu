// Storing new keys and values in a paged cache, and copying its pages.  Both only move bytes and are bound by HBM (or, at
// the sizes of a decode step, by the launch).  4000 pages of 64 KB: 88 us (6.0 TB/s); eight of 256 KB: 2.1 us on the device, 4.7
// a call.  64 tokens of 8 heads of 128: 2.1 us on the device, 5.6 a call; a padded batch of 2 x 4096 (6144 in all, 50 MB): 13 us
// (3.8 TB/s: two rounds of four tokens a thread, each as long as a trip to memory; two or eight tokens, more or fewer
// CTAs took 12.5 to 17).
#include <algorithm>

#include "attention.h"
#include "sm100_ptx.cuh"

namespace fo {

namespace {

constexpr int kThreads = 256;

template <typename... Params, typename... Args>
cudaError_t launch_after(void (*kernel)(Params...), long long grid, cudaStream_t stream, const Args&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(grid), 1, 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// A token is `items` chunks of 16 bytes: its keys head by head, then its values.  A thread keeps its chunk and walks tokens
// (`rows` of them per CTA at a time), several in flight.
constexpr int kTokensInFlight = 4;
__global__ void __launch_bounds__(kThreads) cache_append_kernel(const __grid_constant__ AppendParams p, int items, int rows,
                                                                FastDiv by_tokens) {
  ptx::wait_for_previous_kernel();
  ptx::allow_next_kernel();
  const int chunks = p.pages.head_dim >> 3;
  const long long total = static_cast<long long>(p.seqs) * p.tokens;
  const int row = rows > 1 ? threadIdx.x / items : 0;
  if (row >= rows) return;
  for (int item = threadIdx.x - row * items; item < items; item += kThreads) {
    const int of_keys = items >> 1;
    const bool is_value = item >= of_keys;
    const int within = item - (is_value ? of_keys : 0);
    const int head = within / chunks, col = (within - head * chunks) * 8;
    const uint16_t* src = static_cast<const uint16_t*>(is_value ? p.v : p.k) +
                          head * (is_value ? p.v_stride[2] : p.k_stride[2]) + col;
    const long long seq_stride = is_value ? p.v_stride[0] : p.k_stride[0];
    const long long tok_stride = is_value ? p.v_stride[1] : p.k_stride[1];
    uint16_t* dst = static_cast<uint16_t*>(p.cache) + (is_value ? p.pages.value_offset() : 0) + col;
    const long long step = static_cast<long long>(gridDim.x) * rows;
    for (long long t0 = static_cast<long long>(blockIdx.x) * rows + row; t0 < total; t0 += step * kTokensInFlight) {
      uint4 v[kTokensInFlight];
      long long to[kTokensInFlight];
      // (the page is looked up while the token is on its way)
#pragma unroll
      for (int u = 0; u < kTokensInFlight; ++u) {
        const long long t = t0 + u * step;
        to[u] = -1;
        if (t < total) {
          const int s = static_cast<int>(by_tokens.div(static_cast<uint32_t>(t)));
          const int i = static_cast<int>(t - static_cast<long long>(s) * p.tokens);
          if (p.counts == nullptr || i < __ldg(p.counts + s)) {
            v[u] = __ldg(reinterpret_cast<const uint4*>(src + s * seq_stride + i * tok_stride));
            const int start = __ldg(p.starts + s);
            int place;
            const int page = start >= 0 && start <= INT32_MAX - i ? p.pages.find(p.table + s * p.table_stride, p.width, start + i, place) : -1;
            if (page >= 0) to[u] = p.pages.key_offset(page, head, place);
          }
        }
      }
#pragma unroll
      for (int u = 0; u < kTokensInFlight; ++u) {
        if (to[u] >= 0) *reinterpret_cast<uint4*>(dst + to[u]) = v[u];
      }
    }
  }
}

// The list of moves travels with the launch: nothing to upload, nothing to keep alive, and a captured launch holds its own.
template <int CAP>
struct Moves {
  int2 at[CAP];  // from, to
};
constexpr int kChunksPerThread = 4;
template <int CAP>
__global__ void __launch_bounds__(kThreads) copy_pages_kernel(char* cache, long long stride, FastDiv by_chunks, unsigned total,
                                                              const __grid_constant__ Moves<CAP> moves) {
  ptx::wait_for_previous_kernel();
  ptx::allow_next_kernel();
  for (unsigned base = blockIdx.x * (kThreads * kChunksPerThread) + threadIdx.x; base < total;
       base += gridDim.x * (kThreads * kChunksPerThread)) {
    uint4 v[kChunksPerThread];
    char* to[kChunksPerThread];
#pragma unroll
    for (int u = 0; u < kChunksPerThread; ++u) {
      const unsigned c = min(base + u * kThreads, total - 1);  // past the end: the last chunk again, with the same value
      const unsigned m = by_chunks.div(c);
      const long long within = static_cast<long long>(c - m * by_chunks.d) << 4;
      const int2 mv = moves.at[m];
      to[u] = cache + mv.y * stride + within;
      v[u] = *reinterpret_cast<const uint4*>(cache + mv.x * stride + within);
    }
#pragma unroll
    for (int u = 0; u < kChunksPerThread; ++u) *reinterpret_cast<uint4*>(to[u]) = v[u];
  }
}

template <int CAP>
cudaError_t copy_some(char* cache, long long chunks, long long stride, const int* moves, int n, cudaStream_t stream) {
  Moves<CAP> list;
  for (int i = 0; i < n; ++i) list.at[i] = make_int2(moves[2 * i], moves[2 * i + 1]);
  for (int i = n; i < CAP; ++i) list.at[i] = make_int2(0, 0);
  const long long total = chunks * n;
  const long long per_cta = kThreads * kChunksPerThread;
  const long long grid = std::min<long long>((total + per_cta - 1) / per_cta, 8ll * device_sm_count());
  return launch_after(copy_pages_kernel<CAP>, grid, stream, cache, stride, FastDiv(static_cast<uint32_t>(chunks)),
                      static_cast<unsigned>(total), list);
}

}  // namespace

cudaError_t launch_cache_append(const AppendParams& p, cudaStream_t stream) {
  const long long total = static_cast<long long>(p.seqs) * p.tokens;
  if (total == 0) return cudaSuccess;
  if (total >= (1ll << 31) || p.pages.head_dim % 8 != 0) return cudaErrorInvalidValue;
  const int items = 2 * p.pages.kv_heads * (p.pages.head_dim / 8);
  const int rows = std::max(1, kThreads / items);
  const long long per_cta = static_cast<long long>(rows) * kTokensInFlight;
  // few tokens: one per thread, so that all SMs take part
  const long long want = std::max((total + per_cta - 1) / per_cta,
                                  std::min<long long>((total + rows - 1) / rows, device_sm_count()));
  const long long grid = std::min<long long>(want, 8ll * device_sm_count());
  return launch_after(cache_append_kernel, grid, stream, p, items, rows, FastDiv(static_cast<uint32_t>(p.tokens)));
}

cudaError_t launch_copy_pages(void* cache, long long page_bytes, long long page_stride_bytes, const int* moves, int n,
                              cudaStream_t stream) {
  constexpr int kFew = 60, kSome = 480, kMany = 4000;  // launch parameters of 512 bytes, 4 KB and 32 KB (the most there can be)
  if (page_bytes <= 0 || page_bytes % 16 != 0 || page_stride_bytes % 16 != 0) return cudaErrorInvalidValue;
  const long long chunks = page_bytes / 16;
  if (chunks >= (1ll << 30)) return cudaErrorInvalidValue;
  // (chunk numbers of one launch stay below 2^30)
  const int most = static_cast<int>(std::min<long long>(kMany, std::max<long long>(1, (1ll << 30) / chunks)));
  for (int at = 0; at < n;) {
    const int some = std::min(n - at, most);
    const auto copy = some <= kFew ? copy_some<kFew> : some <= kSome ? copy_some<kSome> : copy_some<kMany>;
    const cudaError_t e = copy(static_cast<char*>(cache), chunks, page_stride_bytes, moves + 2 * at, some, stream);
    if (e != cudaSuccess) return e;
    at += some;
  }
  return cudaSuccess;
}

}  // namespace fo
