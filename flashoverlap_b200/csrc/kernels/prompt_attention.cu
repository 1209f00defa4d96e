// Attention of a prompt: causal, with an optional window of recent tokens and first tokens that stay visible.
//
// A CTA takes two tiles of 128 rows of one key and value head; a row is a token and one of the query heads that share the
// head, so that a tile of grouped heads spans few tokens and little of it is hidden by the diagonal.  For every tile of 128
// visible tokens, scores S = Q K^T go from the tensor cores into TMEM, a thread per row turns its 128 scores into weights,
// P goes back into TMEM over S, and O += P V accumulates there.  While the tensor cores work for one tile of rows, 128 threads
// compute the weights of the other.
//
//   warps 0-3, 4-7   softmax of the two tiles: warp w reads the TMEM lanes 32 (w % 4) .. + 31, a thread is a row
//   warp 8           TMA: Q, then K and V tile by tile into a ring of buffers
//   warp 9           tcgen05.mma: S_i = Q_i K_j^T from shared memory, O_i += P_i V_j with P_i in TMEM
//   warps 10, 11     look at the values of tiles that are not seen whole (below)
//
// A CTA that has six tiles of keys of its pair left asks the hardware for a CTA that has not been launched yet and takes its
// place (clusterlaunchcontrol): its loads and first scores run under the last weights and the stores of the pair before.
// Pairs with the most keys are launched first.  Where there are fewer pairs than half of the SMs, the keys of a pair are
// divided over several CTAs, and a second kernel joins the parts in their order.
//
// A hidden token's weight is zero, and zero times infinity is not: in tiles that some row does not see whole, values behind
// the length become zero, and should any other not be finite, the rows of the pair are computed one by one at the end: 32 rows
// a warp, 0.5 to 1 us for each token that a row sees (16384 tokens: 0.44 s), during which no wait of the CTA runs out.
//
// TMEM (512 columns of 32 bits): S_0, S_1 (128 each; P_i, 16-bit pairs, over the first 64 of S_i), O_0, O_1 (head_dim each).
// Heads of 64 leave room for weights of their own, so that the next scores need not wait for the products; then both groups
// of softmax warps ask for their powers at the same time and leave the unit idle at the same time (16384 tokens 377 us as it
// is, 408 so).
//
// The running largest score of a row only moves when it grows by more than 8 (in powers of two): until then weights are up
// to 2^8 instead of 1, which costs no accuracy (P is a floating-point type, sums are fp32), and O is not rescaled.  In fp16,
// which has numbers from 2^-24 to 2^16, weights and their sum carry a factor of 2^7 besides: a weight of 2^-25 of the largest
// would vanish from P and not from the sum, and 10^5 of them are more than a step of the result.
//
// What bounds it: a tile of keys takes a pair 2950 clocks (head_dim 128), 2048 of them tensor work.  The 128 weights of a
// thread take some 1700 (200 until the scores are in registers, 300 for the largest, 1250 for powers, sums and their way to
// TMEM; 16 powers a clock and SM would be 1024), the products and the next scores 1000; the two groups of warps run half a
// turn apart.  Long calls run at the power cap: 16384 tokens, 8 heads on 1, fp16, 494 to 506 us call after call (1.1 PFLOP/s,
// 0.8 of cuBLAS's sustained bf16 rate), 445 in a short burst.  2 x 4096 tokens, 32 heads on 8, window 1024, bf16: 160 to 164 us
// (the cap again; 145 in a short burst), ten tiles of keys for 8.3 that are seen, and 7000 clocks a pair for its first scores
// and its results.  3 x 500 tokens behind 4503, 12 heads of 64 on 4, window 2048: 32 us; 77 tokens: 7.7 a call.
//
// Tried and slower: two threads a row (16 warps of softmax; 16384 tokens 588 us), results stored by TMA or row by row, the
// second half of the scores read again after the first weights have left, tiles multiplied and weighed by quarters.  A lane
// that walks the tiles alone, and not its whole warp, takes 80 clocks to issue an instruction.
#include <algorithm>
#include <cmath>

#include <cuda.h>
#include <cudaTypedefs.h>

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

// ---------------------------------------------------------------------------------------------------------------------
constexpr int kTileRows = 128, kTileKeys = 128;
constexpr int kSoftmaxThreads = 256, kPromptThreads = 384;
constexpr int kPolyEvery = 8;                    // every eighth pair of weights comes from the polynomial (16384 tokens, heads of
                                                 // 64: 359 us; the others before the last step: 370, 396 with none, 387 with every fourth)
constexpr float kRaise = 8.f;                    // powers of two that a row's largest score may grow before O is rescaled
template <bool BF16>
constexpr float kFactor = BF16 ? 0.f : 7.f;      // powers of two in the weights: at most 2^(8 + 7) of fp16's 2^16

template <int D>
constexpr int ring_buffers() {
  return D == 128 ? 4 : 8;
}
template <int D>
constexpr int key_tile_bytes() {
  return kTileKeys * D * 2;
}
template <int D>
constexpr int out_column(int tile) {
  return 2 * kTileKeys + tile * D;
}
constexpr int kStageBytes = 32 * 128;  // 64 columns of a warp's results, on their way out
// shared memory behind the first 1024-byte boundary: two Q tiles, the ring, a stage for each softmax warp
template <int D>
constexpr int prompt_smem_bytes() {
  return 2 * kTileRows * D * 2 + ring_buffers<D>() * key_tile_bytes<D>() + 8 * kStageBytes + 1024;
}

struct PromptArgs {
  PromptParams p;
  CUtensorMap q, k, v;
  int group, tokens;         // query heads of a head, tokens of a tile
  FastDiv by_parts, by_row, by_kv, by_group;  // parts; batch * kv_heads; kv_heads; group
  int single;                // all CTAs fit the chip: there is nothing to take over
  // Few pairs of tiles: the keys of a pair are divided over `parts` CTAs, which leave unscaled results in fp32, for each row
  // the largest score (times log2 e) and the sum of weights, and for each tile whether a value was not finite.
  int parts;
  float* part_out;
  float2* part_ml;
  int* part_odd;
  int blocks, q_batch, k_batch, v_batch, k_head, v_head, q_head;  // pairs of tiles; 0 where a dimension is broadcast, else 1
  float scale_log2;
};

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int x, int y, int z, int w) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(ptx::smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w)
      : "memory");
}
// B as stored by a TMA load of [tokens][64 values] boxes, 128-byte swizzle, read along the tokens (MN-major): groups of 8
// tokens are 1024 bytes apart, the next 64 columns `block_bytes`.
__device__ __forceinline__ uint64_t make_smem_desc_mn_sw128(uint32_t smem_addr, uint32_t block_bytes) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((smem_addr & 0x3ffffu) >> 4);
  d |= static_cast<uint64_t>(block_bytes >> 4) << 16;
  d |= static_cast<uint64_t>(1024 >> 4) << 32;
  d |= static_cast<uint64_t>(1) << 46;
  d |= static_cast<uint64_t>(2) << 61;
  return d;
}
// D[TMEM] (+)= A[TMEM] B[shared memory]
__device__ __forceinline__ void umma_f16_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t desc_b, uint32_t idesc,
                                            uint32_t accumulate) {
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t"
      "}"
      ::"r"(tmem_d), "r"(tmem_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void tmem_st_32x32b_x32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};"
      ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
        "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
        "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]), "r"(taddr)
      : "memory");
}
// One lane of a converged warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t e;
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t"
      "}"
      : "=r"(e));
  return e != 0;
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Bits lo .. hi (inclusive) of a 32-bit word; none if hi < lo.
__device__ __forceinline__ uint32_t bit_range(int lo, int hi) {
  lo = max(lo, 0);
  hi = min(hi, 31);
  return hi < lo ? 0u : (0xffffffffu >> (31 - hi)) & (0xffffffffu << lo);
}
// Largest magnitude of two 16-bit values, as integers: infinities and NaN are the largest of all.
__device__ __forceinline__ uint32_t magnitudes(uint32_t m, const uint4& v) {
  m = __vmaxu2(m, v.x & 0x7fff7fffu);
  m = __vmaxu2(m, v.y & 0x7fff7fffu);
  m = __vmaxu2(m, v.z & 0x7fff7fffu);
  return __vmaxu2(m, v.w & 0x7fff7fffu);
}
template <bool BF16>
__device__ __forceinline__ bool all_finite(uint32_t m) {
  constexpr uint32_t inf = BF16 ? 0x7f80u : 0x7c00u;
  return (m & 0xffffu) < inf && (m >> 16) < inf;
}

// Scores whose bit is not set become -inf.
__device__ __forceinline__ void hide(uint32_t (&s)[32], uint32_t see) {
#pragma unroll
  for (int e = 0; e < 32; ++e) {
    if (!(see & (1u << e))) s[e] = 0xff800000u;
  }
}

// What a CTA works on: a pair of tiles.
struct PromptPair {
  int b, kv_head, t0, length;  // t0: first token of the first tile
  SeenTiles tiles;
  int n;      // tiles of keys that this CTA takes; 0: none
  int first;  // the first of them
  __device__ __forceinline__ int key(int j) const { return tiles.start(first + j); }
};
__device__ __forceinline__ PromptPair prompt_pair(const PromptArgs& a, int index) {
  const PromptParams& p = a.p;
  PromptPair r;
  int part = 0;
  if (a.parts > 1) {
    const int pair = static_cast<int>(a.by_parts.div(index));
    part = index - pair * a.parts;
    index = pair;
  }
  // late tokens first: they see the most keys
  const int per = p.batch * p.kv_heads;
  const int qb = static_cast<int>(a.by_row.div(index)), rest = index - qb * per;
  r.b = static_cast<int>(a.by_kv.div(rest));
  r.kv_head = rest - r.b * p.kv_heads;
  r.t0 = (a.blocks - 1 - qb) * 2 * a.tokens;
  r.length = p.lengths == nullptr ? p.sk : min(max(__ldg(p.lengths + r.b), 0), p.sk);
  const int p0 = p.sk - p.sq + r.t0, p1 = p.sk - p.sq + min(r.t0 + 2 * a.tokens, p.sq) - 1;
  r.tiles = seen_tiles(p0, p1, r.length, p.window, p.sinks, kTileKeys, 1);
  r.n = p0 < r.length ? r.tiles.count() : 0;  // 0: no row sees anything
  r.first = 0;
  if (a.parts > 1) {
    const int per = static_cast<int>(a.by_parts.div(r.n + a.parts - 1));
    r.first = min(part * per, r.n);
    r.n = min(per, r.n - r.first);
  }
  return r;
}
// Whether every row of tile i (0, 1) sees all of a tile of keys.
__device__ __forceinline__ bool sees_whole(const PromptArgs& a, const PromptPair& r, int i, int first_key) {
  const PromptParams& p = a.p;
  const int lo = p.sk - p.sq + r.t0 + i * a.tokens, hi = min(lo + a.tokens, p.sk) - 1, last_key = first_key + kTileKeys - 1;
  return last_key <= lo && last_key < r.length && hi < r.length &&
         (p.window == 0 || hi - first_key < p.window || last_key < p.sinks);
}
__device__ __forceinline__ bool seen_by_all(const PromptArgs& a, const PromptPair& r, int first_key) {
  return sees_whole(a, r, 0, first_key) && sees_whole(a, r, 1, first_key);
}

// A place in a ring of N buffers, and how often the ring has been gone round.
template <int N>
struct Ring {
  int at = 0;
  uint32_t round = 0;
  __device__ __forceinline__ void next(int n = 1) {
    at += n;
    if (at >= N) {
      at -= N;
      ++round;
    }
  }
};

// Asks for a CTA that has not been launched; the answer (16 bytes) arrives on `bar`.
__device__ __forceinline__ void claim_cta(void* answer, uint64_t* bar) {
  asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];"
               ::"r"(ptx::smem_u32(answer)), "r"(ptx::smem_u32(bar))
               : "memory");
}
// Index of the claimed CTA, -1 if there was none left.
__device__ __forceinline__ int claimed_cta(const void* answer) {
  uint32_t ok, x;
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      ".reg .b128 r;\n\t"
      "ld.shared.b128 r, [%2];\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, r;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t"
      "mov.u32 %1, 0;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, r;\n\t"
      "}"
      : "=r"(ok), "=r"(x)
      : "r"(ptx::smem_u32(answer))
      : "memory");
  return ok ? static_cast<int>(x) : -1;
}

// A part's results of one row: 32 columns at a time through the warp's stage, so that whole lines are stored.
template <int D>
__device__ __forceinline__ void store_part(const PromptArgs& a, int index, int tile, int row, uint32_t stage, uint32_t t_o,
                                           bool any, bool odd, float m, float l) {
  const int lane = row & 31;
  const long long first = (static_cast<long long>(index) * 2 + tile) * kTileRows;
  a.part_ml[first + row] = any && m != -INFINITY ? make_float2(m * a.scale_log2, l) : make_float2(-INFINITY, 0.f);
  if (row == 0) a.part_odd[index * 2 + tile] = odd;
  if (!any) return;
#pragma unroll
  for (int q = 0; q < D / 32; ++q) {
    uint32_t o[32];
    ptx::tmem_ld_32x32b_x32(t_o + q * 32, o);
    ptx::tmem_ld_wait_for(o);
    __syncwarp();
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      ptx::st_shared_v4(stage + lane * 128 + ((e ^ (lane & 7)) << 4), make_uint4(o[e * 4], o[e * 4 + 1], o[e * 4 + 2], o[e * 4 + 3]));
    }
    __syncwarp();
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int from = e * 4 + (lane >> 3), chunk = lane & 7;
      const uint4 v = ptx::ld_shared_v4(stage + from * 128 + ((chunk ^ (from & 7)) << 4));
      ptx::st_v4(a.part_out + (first + (row & ~31) + from) * D + q * 32 + chunk * 4, v);
    }
  }
}

// Joins the parts of a pair's rows, a warp for each row; lanes take columns.
template <int D, bool BF16>
__global__ void __launch_bounds__(256) prompt_join_kernel(const __grid_constant__ PromptArgs a) {
  constexpr int V = D / 32, kBatch = 6;
  ptx::wait_for_previous_kernel();
  ptx::allow_next_kernel();
  const PromptParams& p = a.p;
  const int lane = threadIdx.x & 31, pair = blockIdx.x;
  const int rows = a.group * a.tokens;
  const int x = blockIdx.y * 8 + (threadIdx.x >> 5);  // rows of both tiles
  if (x >= 2 * rows) return;
  const int tile = x >= rows ? 1 : 0, row = x - tile * rows;
  const int token = static_cast<int>(a.by_group.div(row));
  const PromptPair r = prompt_pair(a, pair * a.parts);
  const int t = r.t0 + tile * a.tokens + token, head = r.kv_head * a.group + row - token * a.group;
  if (t >= p.sq) return;
  bool odd = false;
  float acc[V] = {}, sum = 0.f, most = -INFINITY;
  for (int i0 = 0; i0 < a.parts; i0 += kBatch) {
    float2 ml[kBatch];
    float y[kBatch][V];
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      ml[k] = make_float2(-INFINITY, 0.f);
      if (i0 + k >= a.parts) continue;
      const int part = pair * a.parts + i0 + k;
      const long long at = (static_cast<long long>(part) * 2 + tile) * kTileRows + row;
      ml[k] = a.part_ml[at];
      odd |= a.part_odd[part * 2 + tile] != 0;
      const float* src = a.part_out + at * D + lane * V;
      if constexpr (V == 4) {
        const float4 z = *reinterpret_cast<const float4*>(src);
        y[k][0] = z.x;
        y[k][1] = z.y;
        y[k][2] = z.z;
        y[k][3] = z.w;
      } else {
        const float2 z = *reinterpret_cast<const float2*>(src);
        y[k][0] = z.x;
        y[k][1] = z.y;
      }
    }
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      // (a part that saw nothing has written no results)
      if (ml[k].x == -INFINITY && ml[k].y == 0.f) {
#pragma unroll
        for (int v = 0; v < V; ++v) y[k][v] = 0.f;
      }
    }
    float top = most;
#pragma unroll
    for (int k = 0; k < kBatch; ++k) top = fmaxf(top, ml[k].x);
    const float base = top == -INFINITY ? 0.f : top;
    const float old = exp2_fast(most - base);
    most = top;
    sum *= old;
#pragma unroll
    for (int v = 0; v < V; ++v) acc[v] *= old;
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const float w = exp2_fast(ml[k].x - base);
      sum += ml[k].y * w;
#pragma unroll
      for (int v = 0; v < V; ++v) acc[v] += y[k][v] * w;
    }
  }
  if (odd) {
    exact_row<D, BF16>(p, r.b, t, head, r.length, a.scale_log2);
    return;
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  uint16_t* dst = static_cast<uint16_t*>(p.out) + ((static_cast<long long>(r.b) * p.sq + t) * p.heads + head) * D + lane * V;
#pragma unroll
  for (int v = 0; v < V; v += 2) *reinterpret_cast<uint32_t*>(dst + v) = inv == 0.f ? 0u : pack<BF16>(acc[v] * inv, acc[v + 1] * inv);
}

constexpr int kClaimTiles = 6;  // of keys that are left when a CTA claims its next pair
constexpr int kPairsAhead = 4;  // Values are looked at up to two pairs ahead of the softmax: a pair's are loaded after its Q, Q after
                                // the scores of the pair before, those after the weights of the one before that.
constexpr int kChecks = 8;    // tiles of values that may have been looked at and not used: more than the ring holds
constexpr int kReaders = 12;  // of an answer: TMA, MMA, the two warps that look at values, eight softmax warps

template <int D, bool BF16>
__global__ void __launch_bounds__(kPromptThreads, 1) prompt_attention_kernel(const __grid_constant__ PromptArgs a) {
  constexpr int NB = ring_buffers<D>(), TILE = key_tile_bytes<D>(), BLOCK = kTileKeys * 128;
  const PromptParams& p = a.p;
  extern __shared__ __align__(128) uint8_t raw[];
  __shared__ __align__(16) uint4 answers[2];
  __shared__ __align__(8) uint64_t q_full[2], q_empty, kv_full[NB], kv_empty[NB], s_full[2], p_full[2][2], o_done[2], v_ok[kChecks],
      checked[kPairsAhead], next_full[2], next_empty[2];
  __shared__ uint32_t tmem_slot;
  __shared__ int odd_pair[kPairsAhead];                           // the last pair (counted from 1) whose values are not all finite
  __shared__ int one_by_one;  // warps that compute rows one by one
  __shared__ int failed, unfinished, taken, pending, pairs[4];  // after a wait that ran out (by warp `failed` - 1), see the end
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t smem = (ptx::smem_u32(raw) + 1023u) & ~1023u;
  const uint32_t ring = smem + 2 * kTileRows * D * 2, stage = ring + NB * TILE;

  if (lane == 0 && warp < 4) {  // (a barrier at a time by one thread takes 600 clocks)
    if (warp == 0) {
      for (int i = 0; i < 2; ++i) {
        ptx::mbar_init(&q_full[i], 1);
        ptx::mbar_init(&s_full[i], 1);
        ptx::mbar_init(&p_full[i][0], kTileRows);
        ptx::mbar_init(&p_full[i][1], kTileRows);
        ptx::mbar_init(&o_done[i], 1);
      }
    } else if (warp == 1) {
      for (int i = 0; i < NB; ++i) {
        ptx::mbar_init(&kv_full[i], 1);
        ptx::mbar_init(&kv_empty[i], 1);
      }
      ptx::mbar_init(&q_empty, 1);
    } else if (warp == 2) {
      for (int i = 0; i < kChecks; ++i) ptx::mbar_init(&v_ok[i], 2);
      one_by_one = 0;
      failed = 0;
      unfinished = INT32_MAX;
      taken = 0;
      pending = -1;
    } else {
      for (int i = 0; i < kPairsAhead; ++i) {
        ptx::mbar_init(&checked[i], 2);
        odd_pair[i] = 0;
      }
      for (int i = 0; i < 2; ++i) {
        ptx::mbar_init(&next_full[i], 1);
        ptx::mbar_init(&next_empty[i], kReaders);
      }
    }
    ptx::mbar_fence_init();
    ptx::fence_proxy_async_smem();
  }
  if (warp == 8) {
    if (lane == 0) {
      ptx::prefetch_tensormap(&a.q);
      ptx::prefetch_tensormap(&a.k);
      ptx::prefetch_tensormap(&a.v);
    }
    __syncwarp();
    ptx::tmem_alloc(&tmem_slot, 512);
    ptx::tmem_relinquish();
    ptx::tc_fence_before_sync();
  }
  __syncthreads();
  ptx::tc_fence_after_sync();
  const uint32_t tmem = tmem_slot;
  ptx::wait_for_previous_kernel();

  // Each wait has a limit of its own: a CTA may work for long.  Once one has run out, all give up.  (The clock is looked at
  // every 1024th time; where the limit is short, which it is in tests, each time, and the thread is not suspended, for a
  // microsecond or more, between looks.)
  const bool brief = p.wait_ns < 1000000ull;
  auto wait = [&](uint64_t* bar, uint32_t parity) {
    if (!brief && ptx::mbar_try_wait(bar, parity)) return true;
    uint64_t deadline = 0;
    for (uint32_t tries = 1;; ++tries) {
      if (brief ? ptx::mbar_test_wait(bar, parity) : ptx::mbar_try_wait(bar, parity)) return true;
      if (brief || (tries & 0x3ffu) == 0u) {
        const uint64_t now = ptx::globaltimer_ns();
        // (the time that rows one by one take is nobody's fault, and grows with the tokens)
        if (deadline == 0 || *const_cast<volatile int*>(&one_by_one) != 0) deadline = now + p.wait_ns;
        if (*const_cast<volatile int*>(&failed) != 0) return false;
        if (now > deadline) {
          *const_cast<volatile int*>(&failed) = warp + 1;
          return false;
        }
      }
    }
  };
  // the lanes of a warp go on, or give up, together
  auto wait_warp = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, wait(bar, parity)) != 0; };
  // The pair after the it-th; -1: none, or given up.
  auto next_pair = [&](int it) {
    if (a.single) return -1;
    if (!wait_warp(&next_full[it & 1], (it >> 1) & 1u)) return -1;
    const int index = claimed_cta(&answers[it & 1]);
    __syncwarp();
    if (lane == 0) {
      ptx::fence_proxy_async_smem();
      ptx::mbar_arrive(&next_empty[it & 1]);
    }
    return index;
  };

  // 384 threads x 168 registers at launch = 128 x 56 + 256 x 224
  auto hand_over = [] { asm volatile("setmaxnreg.dec.sync.aligned.u32 56;"); };
  if (warp == 8) {
    hand_over();
    if (lane == 0) {
      const int rows = a.group * a.tokens;
      Ring<NB> buf;
      bool ok = true;
      uint32_t loaded = 0;  // pairs with keys
      int index = blockIdx.x;
      auto claim = [&](int it) {
        if (a.single) return;
        if (it >= 2) ok = wait(&next_empty[it & 1], ((it >> 1) - 1) & 1u);
        if (!ok) return;
        *const_cast<volatile int*>(&pending) = it;
        ptx::mbar_arrive_expect_tx(&next_full[it & 1], 16);
        claim_cta(&answers[it & 1], &next_full[it & 1]);
      };
      for (int it = 0;; ++it) {
        const int slot = it & 1;
        pairs[it & 3] = index;
        *const_cast<volatile int*>(&taken) = it + 1;
        const PromptPair r = prompt_pair(a, index);
        if (r.n <= kClaimTiles) claim(it);
        if (!ok) break;
        if (r.n > 0) {
          if (loaded > 0) ok = wait(&q_empty, (loaded - 1) & 1u);
          if (!ok) break;
          ++loaded;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            ptx::mbar_arrive_expect_tx(&q_full[i], rows * D * 2);
#pragma unroll
            for (int c = 0; c < D / 64; ++c) {
              tma_load_4d(smem + (i * (D / 64) + c) * (kTileRows * 128), &a.q, &q_full[i], c * 64,
                          r.kv_head * a.group * a.q_head, r.t0 + i * a.tokens, r.b * a.q_batch);
            }
          }
        }
        for (int j = 0; ok && j < r.n; ++j) {
          // Not earlier: CTAs that claim at the start of long pairs would take work from those that are done first (8192
          // tokens, 8 heads: 155 us, 120 claimed here).
          if (j > 0 && j == r.n - kClaimTiles) claim(it);
          if (!ok) break;
          const int key = r.key(j);
#pragma unroll
          for (int kv = 0; kv < 2; ++kv) {
            if (buf.round > 0) ok = ok && wait(&kv_empty[buf.at], (buf.round - 1) & 1u);
            if (!ok) break;
            ptx::mbar_arrive_expect_tx(&kv_full[buf.at], TILE);
#pragma unroll
            for (int c = 0; c < D / 64; ++c) {
              tma_load_4d(ring + buf.at * TILE + c * BLOCK, kv == 0 ? &a.k : &a.v, &kv_full[buf.at], c * 64, key,
                          r.kv_head * (kv == 0 ? a.k_head : a.v_head), r.b * (kv == 0 ? a.k_batch : a.v_batch));
            }
            buf.next();
          }
        }
        if (a.single) break;
        ok = ok && wait(&next_full[slot], (it >> 1) & 1u);
        if (!ok) break;
        index = claimed_cta(&answers[slot]);
        *const_cast<volatile int*>(&pending) = -1;
        ptx::fence_proxy_async_smem();
        ptx::mbar_arrive(&next_empty[slot]);
        if (index < 0) break;
      }
      // (a join that waits on the SMs takes longer than one that comes when they are free)
      if (a.parts == 1) ptx::allow_next_kernel();
    }
    __syncwarp();
  } else if (warp == 9) {
    hand_over();
    // The whole warp walks the tiles; one lane issues.
    constexpr int FMT = BF16 ? 1 : 0;
    constexpr uint32_t idesc_s = ptx::make_idesc_f16(FMT, kTileRows, kTileKeys);
    constexpr uint32_t idesc_o = ptx::make_idesc_f16(FMT, kTileRows, D) | (1u << 16);  // B along its rows
    const uint64_t desc_q = ptx::make_smem_desc_k_sw128(smem), desc_k = ptx::make_smem_desc_k_sw128(ring);
    const uint64_t desc_v = make_smem_desc_mn_sw128(ring, BLOCK);
    auto scores = [&](int i, int buffer) {
      const uint64_t q = desc_q + i * ((D / 64) * (kTileRows * 128) / 16), k = desc_k + buffer * (TILE / 16);
#pragma unroll
      for (int x = 0; x < D / 16; ++x) {
        const int off = (x >> 2) * (BLOCK / 16) + (x & 3) * (32 / 16);
        ptx::umma_f16_ss(tmem + i * kTileKeys, q + off, k + off, idesc_s, x > 0);
      }
      ptx::umma_commit(&s_full[i]);
    };
    auto outputs = [&](int i, int half, int buffer, bool first) {
      const uint64_t v = desc_v + buffer * (TILE / 16);
#pragma unroll
      for (int y = 0; y < kTileKeys / 32; ++y) {
        const int x = half * (kTileKeys / 32) + y;
        umma_f16_ts(tmem + out_column<D>(i), tmem + i * kTileKeys + x * 8, v + x * (16 * 128 / 16), idesc_o,
                    !first || x > 0);
      }
    };
    Ring<NB> buf;
    uint32_t loaded = 0, tiles = 0;
    bool ok = true;
    int index = blockIdx.x;
    for (int it = 0; ok && index >= 0; ++it) {
      const PromptPair r = prompt_pair(a, index);
      if (r.n > 0) {
        // the buffer of scores is free: the products before, which read the weights in it, have been issued before
        ok = wait_warp(&kv_full[buf.at], buf.round & 1u);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          ok = ok && wait_warp(&q_full[i], loaded & 1u);
          if (ok && elect_one()) {
            scores(i, buf.at);
            if (i == 1) {
              ptx::umma_commit(&kv_empty[buf.at]);
              if (r.n == 1) ptx::umma_commit(&q_empty);
            }
          }
          __syncwarp();
        }
        ++loaded;
        buf.next();
      }
      for (int j = 0; ok && j < r.n; ++j, ++tiles) {
        const int vbuf = buf.at;
        ok = wait_warp(&kv_full[vbuf], buf.round & 1u) && wait_warp(&v_ok[tiles % kChecks], (tiles / kChecks) & 1u);
        buf.next();
        const int kbuf = buf.at;
        const bool more = j + 1 < r.n;
        if (ok && more) {
          ok = wait_warp(&kv_full[kbuf], buf.round & 1u);
          buf.next();
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          // the first half of the products starts while the second half of the weights is computed
          ok = ok && wait_warp(&p_full[i][0], tiles & 1u);
          if (!ok) break;
          ptx::tc_fence_after_sync();
          if (elect_one()) outputs(i, 0, vbuf, j == 0);
          __syncwarp();
          ok = wait_warp(&p_full[i][1], tiles & 1u);
          if (!ok) break;
          ptx::tc_fence_after_sync();
          if (elect_one()) {
            outputs(i, 1, vbuf, j == 0);
            ptx::umma_commit(&o_done[i]);
            if (i == 1) ptx::umma_commit(&kv_empty[vbuf]);
            if (more) {
              scores(i, kbuf);
              if (i == 1) {
                ptx::umma_commit(&kv_empty[kbuf]);
                if (j + 2 == r.n) ptx::umma_commit(&q_empty);
              }
            }
          }
          __syncwarp();
        }
      }
      if (ok) index = next_pair(it);
    }
  } else if (warp >= 10) {
    hand_over();
    Ring<NB> buf;  // keys, values, keys, ...
    uint32_t loaded = 0, tiles = 0;
    bool ok = true;
    int index = blockIdx.x;
    for (int it = 0; ok && index >= 0; ++it) {
      const PromptPair r = prompt_pair(a, index);
      for (int j = 0; ok && j < r.n; ++j, ++tiles) {
        const int first_key = r.key(j);
        buf.next();
        ok = wait_warp(&kv_full[buf.at], buf.round & 1u);
        if (!ok) break;
        if (!seen_by_all(a, r, first_key)) {
          const uint32_t at = ring + buf.at * TILE + (threadIdx.x - 320) * 16;
          const int here = r.length - first_key;  // tokens of the tile that the sequence has
          uint32_t m = 0;
          if (here < kTileKeys) {
#pragma unroll 4
            for (int x = 0; x < TILE; x += 64 * 16) {
              if (((x + (threadIdx.x - 320) * 16) & (BLOCK - 1)) / 128 >= here) ptx::st_shared_v4(at + x, make_uint4(0, 0, 0, 0));
            }
          }
#pragma unroll 8
          for (int x = 0; x < TILE; x += 64 * 16) m = magnitudes(m, ptx::ld_shared_v4(at + x));
          if (!all_finite<BF16>(m)) *const_cast<volatile int*>(&odd_pair[loaded % kPairsAhead]) = static_cast<int>(loaded) + 1;
          ptx::fence_proxy_async_smem();
          __syncwarp();
        }
        // (for every tile: the products do not start without it, so that this warp cannot fall behind the ring)
        if (lane == 0) ptx::mbar_arrive(&v_ok[tiles % kChecks]);
        buf.next();
      }
      if (ok && r.n > 0) {
        if (lane == 0) ptx::mbar_arrive(&checked[loaded % kPairsAhead]);
        ++loaded;
      }
      if (ok) index = next_pair(it);
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
    const int tile = warp >> 2;
    const int row = threadIdx.x & 127;
    const uint32_t lanes = static_cast<uint32_t>(warp & 3) << 21;  // 32 lanes each, in the upper half of an address
    const uint32_t t_s = tmem + lanes + tile * kTileKeys, t_o = tmem + lanes + out_column<D>(tile);
    const int token = static_cast<int>(a.by_group.div(row)), head = row - token * a.group;
    const float c = a.scale_log2;
    uint32_t loaded = 0, tiles = 0;
    bool ok = true;
    int index = blockIdx.x;
    for (int it = 0; index >= 0; ++it) {
      const PromptPair r = prompt_pair(a, index);
      const int t = r.t0 + tile * a.tokens + token;
      const int pos = p.sk - p.sq + t;
      const bool real = token < a.tokens && t < p.sq;
      const int last = real && pos < r.length ? pos : -1;  // the last visible token
      const int lo = p.window > 0 && pos >= p.window ? pos - p.window + 1 : 0;
      float m = -INFINITY, l = 0.f;  // the first score that is seen raises m, however small the scale is
      for (int j = 0; j < r.n; ++j, ++tiles) {
        const int first_key = r.key(j);
        const bool masked = !sees_whole(a, r, tile, first_key);
        ok = wait_warp(&s_full[tile], tiles & 1u);
        if (!ok) break;
        ptx::tc_fence_after_sync();
        uint32_t s[4][32];
#pragma unroll
        for (int q = 0; q < 4; ++q) ptx::tmem_ld_32x32b_x32(t_s + q * 32, s[q]);
#pragma unroll
        for (int q = 0; q < 4; ++q) ptx::tmem_ld_wait_for(s[q]);
        if (masked) {
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int k0 = first_key + q * 32;
            const uint32_t see = bit_range(lo - k0, last - k0) | bit_range(0, min(p.sinks - 1, last) - k0);
            // rows of a tile are a few tokens apart: many words are full in all lanes
            if (!__all_sync(0xffffffffu, see == 0xffffffffu)) hide(s[q], see);
          }
        }
        // (NaN counts as the largest: it makes all of its row NaN)
        float top[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) top[q] = __uint_as_float(s[q][0]);
#pragma unroll
        for (int e = 1; e < 31; e += 2) {
#pragma unroll
          for (int q = 0; q < 4; ++q) top[q] = max3_nan(top[q], __uint_as_float(s[q][e]), __uint_as_float(s[q][e + 1]));
        }
        top[0] = max3_nan(top[0], __uint_as_float(s[0][31]), __uint_as_float(s[1][31]));
        top[1] = max3_nan(top[1], __uint_as_float(s[2][31]), __uint_as_float(s[3][31]));
        const float most = max3_nan(max3_nan(top[0], top[1], m), top[2], top[3]);
        // also for NaN; a row that has seen nothing stays as it is; rows that no token fills hold anything
        const bool raise = real && most != m && !((most - m) * c <= kRaise);
        if (__any_sync(0xffffffffu, raise)) {
          const float factor = raise ? exp2_fast((m - most) * c) : 1.f;
          if (raise) m = most;
          l *= factor;
          if (j > 0) {
            // the products of the tile before must have arrived; the next ones wait for this tile's weights
            ok = wait_warp(&o_done[tile], (tiles - 1) & 1u);
            if (!ok) break;
            ptx::tc_fence_after_sync();
#pragma unroll
            for (int q = 0; q < D / 32; ++q) {
              uint32_t o[32];
              ptx::tmem_ld_32x32b_x32(t_o + q * 32, o);
              ptx::tmem_ld_wait_for(o);
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * factor);
              tmem_st_32x32b_x32(t_o + q * 32, o);
            }
            tmem_st_wait();
          }
        }
        float base = m == -INFINITY ? 0.f : m * c;
        base += base - base;  // NaN if the largest score is infinite: the polynomial would hide it
        const float shift = kFactor<BF16> - base;
        const Pair c2 = make_pair(c, c), base2 = make_pair(shift, shift);
        Pair sum[2] = {make_pair(0.f, 0.f), make_pair(0.f, 0.f)};
        // Eight pairs at a time: their arguments, their powers, then what is done with them, so that nothing waits for the
        // power just asked for.
        uint32_t w[2][32];
#pragma unroll
        for (int g = 0; g < 8; ++g) {
          Pair x[8];
          float2 y[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const uint32_t* src = s[g >> 1] + (g & 1) * 16 + e * 2;
            x[e] = fma2(make_pair(__uint_as_float(src[0]), __uint_as_float(src[1])), c2, base2);
          }
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            if (e % kPolyEvery == kPolyEvery - 1) {
              y[e] = exp2_poly(x[e]);
            } else {
              y[e] = split(x[e]);
              y[e] = make_float2(exp2_fast(y[e].x), exp2_fast(y[e].y));
            }
          }
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            sum[e & 1] = add2(sum[e & 1], make_pair(y[e].x, y[e].y));
            w[g >> 2][(g & 3) * 8 + e] = pack<BF16>(y[e].x, y[e].y);
          }
          if (g == 3 || g == 7) tmem_st_32x32b_x32(t_s + (g >> 2) * 32, w[g >> 2]);
          if (g == 3 || g == 7) {  // (the first half's way to TMEM is under the next weights)
            tmem_st_wait();
            ptx::tc_fence_before_sync();
            ptx::mbar_arrive(&p_full[tile][g == 7]);
          }
        }
        const float2 total = split(add2(sum[0], sum[1]));
        l += total.x + total.y;
      }
      bool by_rows = false;
      if (ok && r.n > 0) {
        ok = wait_warp(&checked[loaded % kPairsAhead], (loaded / kPairsAhead) & 1u) && wait_warp(&o_done[tile], (tiles - 1) & 1u);
        ptx::tc_fence_after_sync();
        ++loaded;
        by_rows = *const_cast<volatile int*>(&odd_pair[(loaded - 1) % kPairsAhead]) == static_cast<int>(loaded);
      }
      if (!ok) {
        if (lane == 0) atomicMin(&unfinished, it);
        break;
      }
      if (a.parts > 1) {
        store_part<D>(a, index, tile, row, stage + warp * kStageBytes, t_o, r.n > 0, by_rows, m, l);
        ptx::tc_fence_before_sync();
      } else if (!by_rows) {
        // Through shared memory, so that a store instruction writes four whole lines and not parts of 32: a row's chunks of 16
        // bytes go in where the row's number puts them, eight lanes read a row.
        const float inv = l == 0.f ? 0.f : 1.f / l;
        const uint32_t out = stage + warp * kStageBytes;
        const int chunk = lane & 7;
        const long long mine =
            real ? ((static_cast<long long>(r.b) * p.sq + t) * p.heads + r.kv_head * a.group + head) * D : -1;
        long long to[8];  // the rows whose chunks this lane stores
#pragma unroll
        for (int e = 0; e < 8; ++e) to[e] = __shfl_sync(0xffffffffu, mine, e * 4 + (lane >> 3));
#pragma unroll
        for (int x = 0; x < D / 64; ++x) {
          uint32_t o[2][32] = {};
          if (r.n > 0) {
            ptx::tmem_ld_32x32b_x32(t_o + x * 64, o[0]);
            ptx::tmem_ld_32x32b_x32(t_o + x * 64 + 32, o[1]);
            ptx::tmem_ld_wait_for(o[0]);
            ptx::tmem_ld_wait_for(o[1]);
          }
          __syncwarp();
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            uint32_t w[4];
#pragma unroll
            for (int y = 0; y < 4; ++y) {
              const uint32_t* src = o[e >> 2] + (e & 3) * 8 + y * 2;
              // a row that sees nothing is zero, whatever its accumulator holds
              w[y] = inv == 0.f ? 0u : pack<BF16>(__uint_as_float(src[0]) * inv, __uint_as_float(src[1]) * inv);
            }
            ptx::st_shared_v4(out + lane * 128 + ((e ^ (lane & 7)) << 4), make_uint4(w[0], w[1], w[2], w[3]));
          }
          __syncwarp();
          uint4 v[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int from = e * 4 + (lane >> 3);
            v[e] = ptx::ld_shared_v4(out + from * 128 + ((chunk ^ (from & 7)) << 4));
          }
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            if (to[e] >= 0) ptx::st_v4(static_cast<uint16_t*>(p.out) + to[e] + x * 64 + chunk * 8, v[e]);
          }
        }
        ptx::tc_fence_before_sync();
      } else {
        if (lane == 0) atomicAdd(&one_by_one, 1);
        for (int x = warp & 3; x < a.group * a.tokens; x += 4) {
          const int tok = r.t0 + tile * a.tokens + x / a.group;
          if (tok < p.sq) exact_row<D, BF16>(p, r.b, tok, r.kv_head * a.group + x % a.group, r.length, c);
        }
        if (lane == 0) atomicSub(&one_by_one, 1);
      }
      index = next_pair(it);
      if (index < 0 && *const_cast<volatile int*>(&failed) != 0) {
        if (lane == 0) atomicMin(&unfinished, it + 1);
      }
    }
  }
  __syncthreads();
  if (*const_cast<volatile int*>(&failed) != 0) {
    // A wait ran out: the host is told, copies, answers and products that are still under way get time to end before their
    // memory is given back, and the rows of all pairs that this CTA has taken and not finished become NaN.
    if (threadIdx.x == 0) {  // details first, the code last; of several CTAs any may be the one that is read
      volatile StatusWord* status = p.status;
      status->where = static_cast<uint32_t>(failed - 1);
      status->seen = blockIdx.x;
      __threadfence_system();
      status->code = ST_TIMEOUT_PIPE;
      __threadfence_system();
    }
    const uint64_t until = ptx::globaltimer_ns() + 2000000ull;
    while (ptx::globaltimer_ns() < until) __nanosleep(1000);
    __syncthreads();
    const int rows = 2 * a.tokens * a.group;
    for (int it = unfinished; it <= taken; ++it) {
      int index = -1;
      if (it < taken) index = pairs[it & 3];
      else if (pending >= 0 && ptx::mbar_try_wait(&next_full[pending & 1], (pending >> 1) & 1u)) index = claimed_cta(&answers[pending & 1]);
      if (index < 0) continue;
      const PromptPair r = prompt_pair(a, index);
      if (a.parts > 1) {
        for (int x = threadIdx.x; x < 2 * kTileRows; x += kPromptThreads) {
          a.part_ml[static_cast<long long>(index) * 2 * kTileRows + x] = make_float2(0.f, NAN);
          if (x < 2) a.part_odd[index * 2 + x] = 0;
        }
        continue;
      }
      for (int x = threadIdx.x; x < rows * (D / 8); x += kPromptThreads) {
        const int y = x / (D / 8), t = r.t0 + y / a.group;
        if (t < p.sq) {
          ptx::st_v4(static_cast<uint16_t*>(p.out) +
                         ((static_cast<long long>(r.b) * p.sq + t) * p.heads + r.kv_head * a.group + y % a.group) * D +
                         (x % (D / 8)) * 8,
                     make_uint4(0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu));
        }
      }
    }
  }
  if (warp == 8) {
    ptx::tc_fence_after_sync();
    ptx::tmem_dealloc(tmem, 512);
  }
}

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static const PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult found;
    const bool ok = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &found) == cudaSuccess &&
                    found == cudaDriverEntryPointSuccess;
    return ok ? reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr) : nullptr;
  }();
  return fn;
}
// [d3, d2, d1, head_dim] of 16-bit values; strides in values.  A dimension that is broadcast (stride 0) becomes one entry.
bool make_map(CUtensorMap* map, const void* base, DType dt, int head_dim, const int (&dims)[3], const long long (&strides)[3],
              const int (&box)[2]) {
  if (encode_fn() == nullptr) return false;
  cuuint64_t size[4] = {static_cast<cuuint64_t>(head_dim), 1, 1, 1};
  cuuint64_t bytes[3];
  for (int d = 0; d < 3; ++d) {
    size[d + 1] = strides[d] == 0 ? 1 : static_cast<cuuint64_t>(dims[d]);
    bytes[d] = strides[d] == 0 ? 16 : static_cast<cuuint64_t>(strides[d]) * 2;
  }
  const cuuint32_t boxes[4] = {64, static_cast<cuuint32_t>(box[0]), static_cast<cuuint32_t>(box[1]), 1};
  const cuuint32_t step[4] = {1, 1, 1, 1};
  return encode_fn()(map, dt == DT_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
                     const_cast<void*>(base), size, bytes, boxes, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                     CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                     CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Tensors that the copy engine cannot walk (tokens or query heads that are broadcast) and scales that are not positive (the
// largest score is looked for before scaling) go row by row.
bool fits_tiles(const PromptParams& p) {
  const int group = p.heads / p.kv_heads;
  return p.scale > 0 && (p.sk == 1 || (p.k_stride[1] != 0 && p.v_stride[1] != 0)) && (p.sq == 1 || p.q_stride[1] != 0) &&
         (group == 1 || p.q_stride[2] != 0);
}

// How a call is divided: pairs of tiles, and over how many CTAs the keys of a pair.  Up to half of the SMs' number of pairs
// leave SMs without work; each part has at least kPartTiles tiles, since what a CTA costs however little it does, and
// the second kernel, take as long as some of them.
constexpr int kPartTiles = 3;
struct PromptGrid {
  int tokens, blocks, parts;
  long long pairs;
};
PromptGrid prompt_grid(const PromptParams& p) {
  PromptGrid g;
  g.tokens = kTileRows / (p.heads / p.kv_heads);
  g.blocks = (p.sq + 2 * g.tokens - 1) / (2 * g.tokens);
  g.pairs = static_cast<long long>(g.blocks) * p.batch * p.kv_heads;
  g.parts = 1;
  const int sms = device_sm_count();
  if (g.pairs * 2 <= sms) {
    const int t0 = (g.blocks - 1) * 2 * g.tokens;
    const int tiles = seen_tiles(p.sk - p.sq + t0, p.sk - 1, p.sk, p.window, p.sinks, kTileKeys, 1).count();
    const int parts = std::min(sms / static_cast<int>(g.pairs), tiles / kPartTiles);
    if (parts > 1) g.parts = parts;
  }
  return g;
}

template <int D, bool BF16>
cudaError_t launch_typed(const PromptParams& p, DType dt, cudaStream_t stream) {
  if (!fits_tiles(p)) {
    const long long rows = static_cast<long long>(p.batch) * p.sq * p.heads;
    const long long grid = std::min<long long>((rows + 7) / 8, 8ll * device_sm_count());
    return launch_after(prompt_rows_kernel<D, BF16>, dim3(static_cast<unsigned>(grid)), 256, 0, stream, 1, p);
  }
  PromptArgs a{};
  a.p = p;
  a.group = p.heads / p.kv_heads;
  const PromptGrid g = prompt_grid(p);
  a.tokens = g.tokens;
  a.blocks = g.blocks;
  a.parts = g.parts;
  a.scale_log2 = p.scale * kLog2e;
  a.q_batch = p.q_stride[0] != 0;
  a.q_head = p.q_stride[2] != 0;
  a.k_batch = p.k_stride[0] != 0;
  a.k_head = p.k_stride[2] != 0;
  a.v_batch = p.v_stride[0] != 0;
  a.v_head = p.v_stride[2] != 0;
  if (!make_map(&a.q, p.q, dt, D, {p.heads, p.sq, p.batch}, {p.q_stride[2], p.q_stride[1], p.q_stride[0]},
                {a.group, a.tokens}) ||
      !make_map(&a.k, p.k, dt, D, {p.sk, p.kv_heads, p.batch}, {p.k_stride[1], p.k_stride[2], p.k_stride[0]}, {kTileKeys, 1}) ||
      !make_map(&a.v, p.v, dt, D, {p.sk, p.kv_heads, p.batch}, {p.v_stride[1], p.v_stride[2], p.v_stride[0]}, {kTileKeys, 1})) {
    return cudaErrorInvalidValue;
  }
  const long long grid = g.pairs * g.parts;
  a.single = grid <= device_sm_count();
  a.by_parts = FastDiv(static_cast<uint32_t>(a.parts));
  a.by_row = FastDiv(static_cast<uint32_t>(p.batch * p.kv_heads));
  a.by_kv = FastDiv(static_cast<uint32_t>(p.kv_heads));
  a.by_group = FastDiv(static_cast<uint32_t>(a.group));
  if (grid > INT32_MAX) return cudaErrorInvalidValue;
  if (a.parts > 1) {
    char* ws = static_cast<char*>(p.workspace);
    a.part_out = reinterpret_cast<float*>(ws);
    ws += sizeof(float) * 2 * kTileRows * D * grid;
    a.part_ml = reinterpret_cast<float2*>(ws);
    ws += sizeof(float2) * 2 * kTileRows * grid;
    a.part_odd = reinterpret_cast<int*>(ws);
  }
  cudaError_t e = allow_smem(prompt_attention_kernel<D, BF16>, prompt_smem_bytes<D>());
  if (e != cudaSuccess) return e;
  e = launch_after(prompt_attention_kernel<D, BF16>, dim3(static_cast<unsigned>(grid)), kPromptThreads, prompt_smem_bytes<D>(),
                   stream, 1, a);
  if (e != cudaSuccess || a.parts == 1) return e;
  const int rows = 2 * a.tokens * a.group;
  return launch_after(prompt_join_kernel<D, BF16>, dim3(static_cast<unsigned>(g.pairs), (rows + 7) / 8), 256, 0, stream, 1, a);
}

}  // namespace

size_t prompt_workspace_bytes(const PromptParams& p) {
  if (p.batch == 0 || p.sq == 0 || !fits_tiles(p)) return 0;
  const PromptGrid g = prompt_grid(p);
  if (g.parts == 1) return 0;
  const size_t tiles = static_cast<size_t>(g.pairs) * g.parts * 2;
  return tiles * kTileRows * (p.head_dim * sizeof(float) + sizeof(float2)) + tiles * sizeof(int);
}

cudaError_t launch_prompt_attention(const PromptParams& p, DType dt, cudaStream_t stream) {
  if (p.batch == 0 || p.sq == 0) return cudaSuccess;
  if (p.head_dim == 128) return dt == DT_BF16 ? launch_typed<128, true>(p, dt, stream) : launch_typed<128, false>(p, dt, stream);
  if (p.head_dim == 64) return dt == DT_BF16 ? launch_typed<64, true>(p, dt, stream) : launch_typed<64, false>(p, dt, stream);
  return cudaErrorInvalidValue;
}

}  // namespace fo
