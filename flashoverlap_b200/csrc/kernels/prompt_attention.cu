// Attention of a prompt: causal, with an optional window of recent tokens and first tokens that stay visible.
#include <algorithm>
#include <cmath>

#include "attention_common.cuh"

namespace fo {

using namespace attn;

namespace {

// One row (a token and a query head) by one warp, token by token: the definition, with a running largest score.
template <int D, bool BF16>
__device__ void exact_row(const PromptParams& p, int b, int t, int head, int length, float scale_log2) {
  constexpr int V = D / 32;
  const int lane = threadIdx.x & 31;
  const int kv_head = head / (p.heads / p.kv_heads);
  const int i = p.sk - p.sq + t;
  auto load = [&](const void* base, const long long (&stride)[3], int tok, int h, float (&x)[V]) {
    const uint16_t* src = static_cast<const uint16_t*>(base) + b * stride[0] + tok * stride[1] + h * stride[2] + lane * V;
#pragma unroll
    for (int v = 0; v < V; ++v) x[v] = widen<BF16>(src[v]);
  };
  float q[V], o[V] = {}, m = -INFINITY, l = 0.f;
  load(p.q, p.q_stride, t, head, q);
  if (i < length) {
    const int lo = p.window > 0 && i >= p.window ? i - p.window + 1 : 0;
    for (int j = 0; j <= i; ++j) {
      if (j < lo && j >= p.sinks) j = lo;
      float x[V], s = 0.f;
      load(p.k, p.k_stride, j, kv_head, x);
#pragma unroll
      for (int v = 0; v < V; ++v) s += q[v] * x[v];
#pragma unroll
      for (int w = 16; w > 0; w >>= 1) s += __shfl_xor_sync(0xffffffffu, s, w);
      s *= scale_log2;
      const float top = fmaxf(m, s);
      const float base = top == -INFINITY ? 0.f : top;
      const float alpha = exp2_fast(m - base), w = exp2_fast(s - base);
      m = top;
      l = l * alpha + w;
      load(p.v, p.v_stride, j, kv_head, x);
#pragma unroll
      for (int v = 0; v < V; ++v) o[v] = o[v] * alpha + w * x[v];
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  uint16_t* dst = static_cast<uint16_t*>(p.out) + ((static_cast<long long>(b) * p.sq + t) * p.heads + head) * D + lane * V;
#pragma unroll
  for (int v = 0; v < V; v += 2) *reinterpret_cast<uint32_t*>(dst + v) = pack<BF16>(o[v] * inv, o[v + 1] * inv);
}

template <int D, bool BF16>
__global__ void __launch_bounds__(256) prompt_rows_kernel(const __grid_constant__ PromptParams p) {
  ptx::wait_for_previous_kernel();
  ptx::allow_next_kernel();
  const long long rows = static_cast<long long>(p.batch) * p.sq * p.heads;
  for (long long row = static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5); row < rows; row += gridDim.x * 8ll) {
    const long long token = row / p.heads;
    const int head = static_cast<int>(row - token * p.heads);
    const int b = static_cast<int>(token / p.sq), t = static_cast<int>(token - static_cast<long long>(b) * p.sq);
    const int length = p.lengths == nullptr ? p.sk : min(__ldg(p.lengths + b), p.sk);
    exact_row<D, BF16>(p, b, t, head, length, p.scale * kLog2e);
  }
}

template <int D, bool BF16>
cudaError_t launch_typed(const PromptParams& p, cudaStream_t stream) {
  const long long rows = static_cast<long long>(p.batch) * p.sq * p.heads;
  const long long grid = std::min<long long>((rows + 7) / 8, 8ll * device_sm_count());
  return launch_after(prompt_rows_kernel<D, BF16>, dim3(static_cast<unsigned>(grid)), 256, 0, stream, p);
}

}  // namespace

cudaError_t launch_prompt_attention(const PromptParams& p, DType dt, cudaStream_t stream) {
  if (p.batch == 0 || p.sq == 0) return cudaSuccess;
  if (p.head_dim == 128) return dt == DT_BF16 ? launch_typed<128, true>(p, stream) : launch_typed<128, false>(p, stream);
  if (p.head_dim == 64) return dt == DT_BF16 ? launch_typed<64, true>(p, stream) : launch_typed<64, false>(p, stream);
  return cudaErrorInvalidValue;
}

}  // namespace fo
