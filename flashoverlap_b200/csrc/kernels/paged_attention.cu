// Attention of one new token per sequence over a paged cache.
//
// With one query row per head the work is reading keys and values once: bound by HBM.  The query heads that share a key and
// value head are the rows of a 16-row warp matrix product, so every byte read serves all of them; the tensor pipe is far
// from its limit (two products of 16 x 16 x head_dim per 16 tokens), and rows that no head fills cost nothing that counts.
//
// The work is one line of tiles of 64 tokens: sequence by sequence, head by head, along the visible part of the length.  It
// is cut into equal stretches, one per CTA, whatever the lengths are: one long sequence and a batch of ragged ones fill the
// chip alike, in one wave, and the host needs no lengths.  Sequences that a cut goes through leave partial sums (output in
// fp32, largest score, sum of weights), which a second kernel joins in the order of the stretches: no atomics, the same
// bits every time.
//
// A warp takes 16 tokens of each tile.  They travel with cp.async into its own ring of shared memory, across the borders of
// heads and sequences, so that loads are always under way and warps meet only at the end of a sequence's stretch.
#include <algorithm>
#include <cmath>

#include "attention_common.cuh"

namespace fo {

using namespace attn;

namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kStrip = 16;               // tokens of a warp
constexpr int kTile = kWarps * kStrip;   // tokens of a CTA
constexpr int kRows = 16;                // query heads that one pass serves
constexpr int kCtasPerSm = 2;

template <int D>
constexpr int stages() {
  return D == 128 ? 3 : 4;
}
template <int D>
constexpr int strip_bytes() {
  return kStrip * D * 2;
}

// Query heads of a key and value head are served `rows` at a time, in `subs` passes of their own.
struct HeadSplit {
  int group, subs, rows;
};
HeadSplit head_split(const PagedParams& p) {
  HeadSplit h;
  h.group = p.heads / p.pages.kv_heads;
  h.subs = (h.group + kRows - 1) / kRows;
  h.rows = (h.group + h.subs - 1) / h.subs;
  return h;
}

// What the launch leaves for the joining kernel: {sequence, virtual head, slot of the first part, parts} for the CTA that
// holds the second part of a stretch, {-1, ...} for all others.
struct Partials {
  float* out;   // [2 * ctas][rows][D]: the first sequence of a CTA in slot 2 c, its last one in 2 c + 1
  float2* ml;   // [2 * ctas][rows]: largest score (times log2 e), sum of weights
  int4* joins;  // [ctas]
};

struct PagedArgs {
  PagedParams p;
  HeadSplit h;
  Partials part;
  float scale_log2;
};

// The tiles of one sequence.
struct Sequence {
  SeenTiles t;
  int length, count;
  bool bad;  // longer than its table
};
__device__ __forceinline__ Sequence sequence(const PagedParams& p, int s) {
  Sequence q;
  const long long room = static_cast<long long>(p.width) * p.pages.page_size;
  const int n = max(__ldg(p.lengths + s), 0);
  q.bad = n > room;
  q.length = q.bad ? static_cast<int>(room) : n;
  q.t = seen_tiles(q.length - 1, q.length - 1, q.length, p.window, p.sinks, kTile);
  q.count = max(q.t.count(), 1);  // an empty sequence has a tile as well, of which nothing is visible: its rows become zero
  return q;
}

// A place on the line of tiles.
struct Cursor {
  int s, head, i, left;  // sequence, virtual head, tile of the sequence, tiles to go in this CTA
  Sequence q;
  __device__ __forceinline__ int first_token() const { return q.t.start(i); }
  __device__ __forceinline__ void advance(const PagedParams& p, int heads) {
    --left;
    if (++i < q.count) return;
    i = 0;
    if (++head < heads) return;
    head = 0;
    ++s;
    if (left > 0) q = sequence(p, s);
  }
};

template <int D, bool BF16>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) paged_attention_kernel(const __grid_constant__ PagedArgs a) {
  constexpr int ST = stages<D>(), BYTES = strip_bytes<D>(), CH = D / 8;
  const PagedParams& p = a.p;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int scan[kWarps];
  __shared__ int start[3];                       // sequence, tiles in front of it, all tiles
  __shared__ float2 ml[kWarps][kRows];
  __shared__ unsigned bad_pages[kWarps][ST];
  ptx::wait_for_previous_kernel();
  ptx::allow_next_kernel();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int heads = p.pages.kv_heads * a.h.subs;

  // Where this CTA's stretch begins: a thread adds up the tiles of its share of the sequences.
  int per;
  Cursor ic;
  {
    const int share = (p.seqs + kThreads - 1) / kThreads;
    const int s0 = min(static_cast<int>(threadIdx.x) * share, p.seqs), s1 = min(s0 + share, p.seqs);
    int mine = 0;
    for (int s = s0; s < s1; ++s) mine += sequence(p, s).count;
    int sum = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += x;
    }
    if (lane == 31) scan[warp] = sum;
    __syncthreads();
    int before = sum - mine, total = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) before += scan[w];
      total += scan[w];
    }
    total *= heads;
    per = (total + static_cast<int>(gridDim.x) - 1) / static_cast<int>(gridDim.x);
    const long long first = static_cast<long long>(blockIdx.x) * per;
    if (threadIdx.x == 0) start[2] = total;
    if (first >= static_cast<long long>(before) * heads && first < static_cast<long long>(before + mine) * heads) {
      int s = s0, at = before;
      for (int n; first >= static_cast<long long>(at + (n = sequence(p, s).count)) * heads; ++s) at += n;
      start[0] = s;
      start[1] = at;
    }
    __syncthreads();
    if (first >= total) {
      if (threadIdx.x == 0) a.part.joins[blockIdx.x] = make_int4(-1, 0, 0, 0);
      return;
    }
    ic.s = start[0];
    ic.q = sequence(p, ic.s);
    const int within = static_cast<int>(first) - start[1] * heads;
    ic.head = within / ic.q.count;
    ic.i = within - ic.head * ic.q.count;
    ic.left = min(per, total - static_cast<int>(first));
    if (threadIdx.x == 0) {
      // the stretch that this CTA continues, if the CTA before it holds its beginning
      int4 join = make_int4(-1, 0, 0, 0);
      if (ic.i > 0) {
        const int begin = static_cast<int>(first) - ic.i;
        if (begin / per + 1 == static_cast<int>(blockIdx.x)) {
          join = make_int4(ic.s, ic.head, 2 * (begin / per) + (begin % per != 0), (begin + ic.q.count - 1) / per - begin / per + 1);
        }
      }
      a.part.joins[blockIdx.x] = join;
    }
  }
  Cursor cc = ic;

  const uint32_t ring = ptx::smem_u32(smem) + warp * (ST * 2 * BYTES);
  float* join_buf = reinterpret_cast<float*>(smem + kWarps * ST * 2 * BYTES);  // [2][rows][D]
  const uint16_t* cache = static_cast<const uint16_t*>(p.cache);
  const long long value_off = p.pages.value_offset();

  // Loads run ahead; the page of a token is looked up one tile before its load.
  int page = -1, place = 0;
  bool bad = false;
  auto look_up = [&] {
    page = -1;
    bad = false;
    if (ic.left > 0) {
      const int pos = ic.first_token() + warp * kStrip + (lane & (kStrip - 1));
      if (is_visible(ic.q.length - 1, pos, ic.q.length, p.window, p.sinks)) {
        page = p.pages.find(p.table + ic.s * p.table_stride, p.width, pos, place);
        bad = page < 0;
      }
    }
  };
  auto issue = [&](int slot) {
    if (ic.left > 0) {
      const int kv_head = ic.head / a.h.subs;
      const uint32_t dst = ring + slot * (2 * BYTES);
      const unsigned any_bad = __ballot_sync(0xffffffffu, bad);
      if (lane == 0) bad_pages[warp][slot] = any_bad | (ic.q.bad ? 1u : 0u);
#pragma unroll
      for (int i = 0; i < kStrip * CH / 32; ++i) {
        const int row = (i * 32 + lane) / CH, ch = lane % CH;
        const int pg = __shfl_sync(0xffffffffu, page, row), pl = __shfl_sync(0xffffffffu, place, row);
        const bool take = pg >= 0;
        const uint16_t* src = cache + (take ? p.pages.key_offset(pg, kv_head, pl) + ch * 8 : 0);
        const uint32_t to = dst + row * (D * 2) + ((ch ^ (row & 7)) << 4);
        copy16(to, src, take);
        copy16(to + BYTES, src + (take ? value_off : 0), take);
      }
      ic.advance(p, heads);
      look_up();
    }
    copy_commit();
  };
  look_up();
#pragma unroll
  for (int i = 0; i < ST - 1; ++i) issue(i);

  const int gr = lane >> 2, gc = lane & 3;  // row and column pair of a fragment
  uint32_t qf[D / 16][4];
  float o[D / 8][4], m[2], l[2];
  bool fresh = true, spoiled = false, whole_start = cc.i == 0, first_segment = true;
  int slot = 0, next_slot = ST - 1;
  while (cc.left > 0) {
    const int kv_head = cc.head / a.h.subs, sub = cc.head - kv_head * a.h.subs;
    const int head0 = kv_head * a.h.group + sub * a.h.rows;
    const int rows = min(a.h.rows, a.h.group - sub * a.h.rows);
    if (fresh) {
      const uint16_t* q = static_cast<const uint16_t*>(p.q) + cc.s * p.q_stride[0];
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = gr + (e & 1) * 8, c = ks * 16 + (e >> 1) * 8 + gc * 2;
          qf[ks][e] = r < rows ? __ldg(reinterpret_cast<const uint32_t*>(q + (head0 + r) * p.q_stride[1] + c)) : 0u;
        }
      }
#pragma unroll
      for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
      m[0] = m[1] = -INFINITY;
      l[0] = l[1] = 0.f;
      spoiled = false;
      fresh = false;
    }
    copy_wait<ST - 2>();
    __syncwarp();
    issue(next_slot);
    const uint32_t keys = ring + slot * (2 * BYTES), values = keys + BYTES;
    spoiled |= bad_pages[warp][slot] != 0;

    // scores of 16 rows and 16 tokens
    float c[2][4] = {};
    {
      const int row = (lane & 7) + ((lane >> 4) << 3), half = (lane >> 3) & 1;
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        uint32_t b[4];
        ldmatrix_x4(b, keys + row * (D * 2) + (((ks * 2 + half) ^ (row & 7)) << 4));
        mma_16x8x16<BF16>(c[0], qf[ks], b[0], b[1]);
        mma_16x8x16<BF16>(c[1], qf[ks], b[2], b[3]);
      }
    }
    const int pos0 = cc.first_token() + warp * kStrip;
    float top[2] = {m[0], m[1]};
#pragma unroll
    for (int nt = 0; nt < 2; ++nt) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int pos = pos0 + nt * 8 + gc * 2 + (e & 1);
        const bool see = is_visible(cc.q.length - 1, pos, cc.q.length, p.window, p.sinks);
        c[nt][e] = see ? c[nt][e] * a.scale_log2 : -INFINITY;
        top[e >> 1] = fmaxf(top[e >> 1], c[nt][e]);
      }
    }
    bool raised = false;
    float alpha[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
      top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
      const float base = top[r] == -INFINITY ? 0.f : top[r];
      alpha[r] = exp2_fast(m[r] - base);
      raised |= top[r] != m[r];
      m[r] = top[r];
      l[r] *= alpha[r];
      top[r] = base;
    }
    uint32_t pf[4];
#pragma unroll
    for (int nt = 0; nt < 2; ++nt) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        c[nt][e] = exp2_fast(c[nt][e] - top[e >> 1]);
        l[e >> 1] += c[nt][e];
      }
      // weights are rounded to the type of the values, as the tensor cores take them; their sum is not
      pf[nt * 2] = pack<BF16>(c[nt][0], c[nt][1]);
      pf[nt * 2 + 1] = pack<BF16>(c[nt][2], c[nt][3]);
    }
    if (__any_sync(0xffffffffu, raised)) {
#pragma unroll
      for (int i = 0; i < D / 8; ++i) {
        o[i][0] *= alpha[0];
        o[i][1] *= alpha[0];
        o[i][2] *= alpha[1];
        o[i][3] *= alpha[1];
      }
    }
    {
      const int row = (lane & 7) + (((lane >> 3) & 1) << 3), half = lane >> 4;
#pragma unroll
      for (int j = 0; j < D / 16; ++j) {
        uint32_t b[4];
        ldmatrix_x4_trans(b, values + row * (D * 2) + (((j * 2 + half) ^ (row & 7)) << 4));
        mma_16x8x16<BF16>(o[2 * j], pf, b[0], b[1]);
        mma_16x8x16<BF16>(o[2 * j + 1], pf, b[2], b[3]);
      }
    }
    slot = slot + 1 == ST ? 0 : slot + 1;
    next_slot = next_slot + 1 == ST ? 0 : next_slot + 1;

    // The end of a sequence and head, or of the CTA's stretch: the warps join.
    const bool whole_end = cc.i == cc.q.count - 1;
    if (whole_end || cc.left == 1) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
        if (spoiled) l[r] = NAN;
        if (gc == 0) ml[warp][gr + r * 8] = make_float2(m[r], l[r]);
      }
      __syncthreads();
      float scale[2], most[2], sum[2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        most[r] = -INFINITY;
        sum[r] = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) most[r] = fmaxf(most[r], ml[w][gr + r * 8].x);
        const float base = most[r] == -INFINITY ? 0.f : most[r];
#pragma unroll
        for (int w = 0; w < kWarps; ++w) sum[r] += ml[w][gr + r * 8].y * exp2_fast(ml[w][gr + r * 8].x - base);
        scale[r] = exp2_fast(m[r] - base);
      }
#pragma unroll
      for (int i = 0; i < D / 8; ++i) {
        o[i][0] *= scale[0];
        o[i][1] *= scale[0];
        o[i][2] *= scale[1];
        o[i][3] *= scale[1];
      }
      auto at = [&](int which, int r, int i) {
        return reinterpret_cast<float2*>(join_buf + (which * a.h.rows + gr + r * 8) * D + i * 8 + gc * 2);
      };
      auto put = [&](int which) {
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
          if (gr < rows) *at(which, 0, i) = make_float2(o[i][0], o[i][1]);
          if (gr + 8 < rows) *at(which, 1, i) = make_float2(o[i][2], o[i][3]);
        }
      };
      auto add = [&](int which) {
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
          if (gr < rows) {
            const float2 x = *at(which, 0, i);
            o[i][0] += x.x;
            o[i][1] += x.y;
          }
          if (gr + 8 < rows) {
            const float2 x = *at(which, 1, i);
            o[i][2] += x.x;
            o[i][3] += x.y;
          }
        }
      };
      if (warp >= 2) put(warp - 2);
      __syncthreads();
      if (warp < 2) add(warp);
      if (warp == 1) put(1);
      __syncthreads();
      if (warp == 0) {
        add(1);
        if (whole_start && whole_end) {
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            if (gr + r * 8 < rows) {
              // nothing visible: zero.  (A sum that is not a number stays one.)
              const float inv = sum[r] == 0.f ? 0.f : 1.f / sum[r];
              uint32_t* dst = reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(p.out) +
                                                          (static_cast<long long>(cc.s) * p.heads + head0 + gr + r * 8) * D) + gc;
#pragma unroll
              for (int i = 0; i < D / 8; ++i) dst[i * 4] = pack<BF16>(o[i][r * 2] * inv, o[i][r * 2 + 1] * inv);
            }
          }
        } else {
          const long long part = 2ll * blockIdx.x + (first_segment ? 0 : 1);
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            if (gr + r * 8 < rows) {
              const long long row = part * a.h.rows + gr + r * 8;
              if (gc == 0) a.part.ml[row] = make_float2(most[r], sum[r]);
              float2* dst = reinterpret_cast<float2*>(a.part.out + row * D) + gc;
#pragma unroll
              for (int i = 0; i < D / 8; ++i) dst[i * 4] = make_float2(o[i][r * 2], o[i][r * 2 + 1]);
            }
          }
        }
      }
      fresh = true;
      whole_start = true;
      first_segment = false;
    }
    cc.advance(p, heads);
  }
}

// Joins the parts of one stretch and one query head (blockIdx.y): warps take parts in turn, lanes take columns.
template <int D, bool BF16>
__global__ void __launch_bounds__(kThreads) join_kernel(const __grid_constant__ PagedArgs a) {
  constexpr int V = D / 32;
  __shared__ float red[kWarps][D];
  __shared__ float2 sums[kWarps];
  ptx::wait_for_previous_kernel();
  ptx::allow_next_kernel();
  const int4 join = a.part.joins[blockIdx.x];
  if (join.x < 0) return;
  const int kv_head = join.y / a.h.subs, sub = join.y - kv_head * a.h.subs;
  const int r = blockIdx.y;
  if (r >= min(a.h.rows, a.h.group - sub * a.h.rows)) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  auto row_of = [&](int i) {
    const long long slot = i == 0 ? join.z : 2ll * (static_cast<int>(blockIdx.x) + i - 1);
    return slot * a.h.rows + r;
  };
  float most = -INFINITY;
  for (int i = lane; i < join.w; i += 32) most = fmaxf(most, a.part.ml[row_of(i)].x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
  const float base = most == -INFINITY ? 0.f : most;
  float acc[V] = {}, sum = 0.f;
#pragma unroll 4
  for (int i = warp; i < join.w; i += kWarps) {
    const long long row = row_of(i);
    const float2 ml = a.part.ml[row];
    const float w = exp2_fast(ml.x - base);
    sum += ml.y * w;
    const float* src = a.part.out + row * D + lane * V;
    if constexpr (V == 4) {
      const float4 x = *reinterpret_cast<const float4*>(src);
      acc[0] += x.x * w;
      acc[1] += x.y * w;
      acc[2] += x.z * w;
      acc[3] += x.w * w;
    } else {
      const float2 x = *reinterpret_cast<const float2*>(src);
      acc[0] += x.x * w;
      acc[1] += x.y * w;
    }
  }
#pragma unroll
  for (int v = 0; v < V; ++v) red[warp][lane * V + v] = acc[v];
  if (lane == 0) sums[warp].x = sum;
  __syncthreads();
  if (threadIdx.x < D / 2) {
    float total = 0.f, x = 0.f, y = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      total += sums[w].x;
      x += red[w][threadIdx.x * 2];
      y += red[w][threadIdx.x * 2 + 1];
    }
    const float inv = total == 0.f ? 0.f : 1.f / total;
    const int head = kv_head * a.h.group + sub * a.h.rows + r;
    reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(a.p.out) + (static_cast<long long>(join.x) * a.p.heads + head) * D)[threadIdx.x] =
        pack<BF16>(x * inv, y * inv);
  }
}

// CTAs of a launch: all that fit the chip together, but no more than there can be tiles.
int grid_size(const PagedParams& p) {
  const long long tiles = static_cast<long long>(p.seqs) * p.pages.kv_heads * head_split(p).subs *
                          std::max<long long>(1, (static_cast<long long>(p.width) * p.pages.page_size + kTile - 1) / kTile);
  return static_cast<int>(std::min<long long>(tiles, static_cast<long long>(kCtasPerSm) * device_sm_count()));
}

template <int D, bool BF16>
cudaError_t launch_typed(const PagedParams& p, cudaStream_t stream) {
  PagedArgs a;
  a.p = p;
  a.h = head_split(p);
  a.scale_log2 = p.scale * kLog2e;
  const int grid = grid_size(p);
  char* ws = static_cast<char*>(p.workspace);
  a.part.out = reinterpret_cast<float*>(ws);
  ws += sizeof(float) * 2 * grid * a.h.rows * D;
  a.part.ml = reinterpret_cast<float2*>(ws);
  ws += (sizeof(float2) * 2 * grid * a.h.rows + 15) / 16 * 16;
  a.part.joins = reinterpret_cast<int4*>(ws);
  constexpr int ring = kWarps * stages<D>() * 2 * strip_bytes<D>();
  const size_t smem = ring + sizeof(float) * 2 * a.h.rows * D;
  // (set for every launch: it belongs to the device that is current)
  cudaError_t e = cudaFuncSetAttribute(paged_attention_kernel<D, BF16>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       ring + static_cast<int>(sizeof(float)) * 2 * kRows * D);
  if (e != cudaSuccess) return e;
  e = launch_after(paged_attention_kernel<D, BF16>, dim3(grid), kThreads, smem, stream, a);
  if (e != cudaSuccess || grid == 1) return e;
  return launch_after(join_kernel<D, BF16>, dim3(grid, a.h.rows), kThreads, 0, stream, a);
}

}  // namespace

size_t paged_workspace_bytes(const PagedParams& p) {
  const size_t rows = static_cast<size_t>(2) * grid_size(p) * head_split(p).rows;
  return rows * p.pages.head_dim * sizeof(float) + (rows * sizeof(float2) + 15) / 16 * 16 + sizeof(int4) * grid_size(p);
}

cudaError_t launch_paged_attention(const PagedParams& p, DType dt, cudaStream_t stream) {
  if (p.seqs == 0) return cudaSuccess;
  if (p.pages.head_dim == 128) {
    return dt == DT_BF16 ? launch_typed<128, true>(p, stream) : launch_typed<128, false>(p, stream);
  }
  if (p.pages.head_dim == 64) {
    return dt == DT_BF16 ? launch_typed<64, true>(p, stream) : launch_typed<64, false>(p, stream);
  }
  return cudaErrorInvalidValue;
}

}  // namespace fo
