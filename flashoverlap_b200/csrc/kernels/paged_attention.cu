// Attention of one new token per sequence over a paged cache.
//
// With one query row per head the work is reading keys and values once: bound by HBM.  The query heads that share a key and
// value head are the columns of warp matrix products whose rows are tokens, so every byte read serves all of them.
//
// The work is one line of tiles of 64 tokens: sequence by sequence, head by head, along the visible part of the length.  It
// is cut into equal stretches, one per CTA, whatever the lengths are: one long sequence and a batch of ragged ones fill the
// chip alike, in one wave, and the host needs no lengths.  Sequences that a cut goes through leave partial sums (output in
// fp32, largest score, sum of weights), which a second kernel joins in the order of the stretches: no atomics, the same
// bits every time.
//
// A warp takes 8 KB of keys and values of each tile.  They travel with cp.async into its own ring of shared memory, across
// the borders of heads and sequences, so that loads are always under way and warps meet only at the end of a sequence's
// stretch.
//
// Measured, call after call over three sets of inputs, caches larger than L2: 64 sequences of 1 to 4999 tokens, 32 heads on 8
// of 128, pages of 64: 109 us (6.0 TB/s); two of 100003 and 131072 tokens, 8 heads on 1: 27 us (4.4 TB/s; 1.4 us until a CTA
// knows its stretch, 19 at 6.2 TB/s, then the join: 1 us until its kernel runs, 3 for 150 parts of a head); 48 of up to 30000
// tokens seen through a window of 4096, heads of 64, pages of 24 tokens: 24.5 us (3.8 TB/s).  One sequence of 900 tokens: 6 us
// on the device, 7.4 a call.  With query heads as rows (16, of which 8 are filled) and addresses worked out for every row,
// a strip took 840 instructions of a warp and the first of these cases 129 us, also when everything came from L2.
#include <algorithm>
#include <cmath>

#include "attention_common.cuh"

namespace fo {

using namespace attn;

namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kRows = 16;      // query heads that one pass serves
constexpr int kCtasPerSm = 2;
constexpr int kMaxCluster = 8;
constexpr int kAhead = 4;      // lengths that a lane asks for at a time
// Powers of two in the weights: fp16 has numbers from 2^-24 to 2^16, and a weight of 2^-25 of the largest would vanish from the
// products and not from the sum; 10^5 of them are more than a step of the result.
template <bool BF16>
constexpr float kFactor = BF16 ? 0.f : 15.f;
constexpr int kStages = 3;     // of a warp's ring, 8 KB each (two CTAs then take all of an SM's shared memory)

// Tokens of a warp and of a CTA.  8 KB of keys and values either way: with 16 tokens of 64 values, what a warp does for every
// strip whatever its size (maxima, page numbers, the end of the loop) took longer than the data.
template <int D>
constexpr int strip_tokens() {
  return D == 128 ? 16 : 32;
}
template <int D>
constexpr int tile_tokens() {
  return kWarps * strip_tokens<D>();
}
template <int D>
constexpr int strip_bytes() {
  return strip_tokens<D>() * D * 2;
}
template <int D>
constexpr int paged_smem_bytes() {
  return kWarps * kStages * 2 * strip_bytes<D>() + kWarps * 8 * D * static_cast<int>(sizeof(float));
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

// What the launch leaves for the joining kernel.
struct Partials {
  float* out;   // [2 * ctas][rows][D]: the first sequence of a CTA in slot 2 c, its last one in 2 c + 1
  float2* ml;   // [2 * ctas][rows]: largest score (times log2 e), sum of weights
  // {sequence, virtual head, slot of the first part, parts}, -1: nothing to join.  One for each sequence and virtual head, or
  // for each CTA (the one that holds the first part) where those are fewer.
  int4* joins;
  int by_unit;
};

struct PagedArgs {
  PagedParams p;
  HeadSplit h;
  Partials part;
  int cluster;
  // The scale is positive; the scores are multiplied by 1, by -1 where it was negative, or by 0.
  float scale_log2, sign;
};

__device__ __forceinline__ float2 ld_cluster_f2(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ float4 ld_cluster_f4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}

// The tiles of one sequence.
struct Sequence {
  SeenTiles t;
  int length, count;
  bool bad;  // longer than its table
};
__device__ __forceinline__ Sequence sequence(const PagedParams& p, int length, int tile) {
  Sequence q;
  const long long room = static_cast<long long>(p.width) * p.pages.page_size;
  const int n = max(length, 0);
  q.bad = n > room;
  q.length = q.bad ? static_cast<int>(room) : n;
  q.t = seen_tiles(q.length - 1, q.length - 1, q.length, p.window, p.sinks, tile, tile / kWarps);
  q.count = max(q.t.count(), 1);  // an empty sequence has a tile as well, of which nothing is visible: its rows become zero
  return q;
}

// A place on the line of tiles.
template <int TILE>
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
    if (left > 0) q = sequence(p, __ldg(p.lengths + s), TILE);
  }
};

// NT: query heads of a pass, in eights.  SHORT: see launch_typed.
template <int D, int NT, bool SHORT, bool BF16>
__global__ void __launch_bounds__(kThreads, kCtasPerSm) paged_attention_kernel(const __grid_constant__ PagedArgs a) {
  constexpr int ST = kStages, BYTES = strip_bytes<D>(), CH = D / 8, TOK = strip_tokens<D>(), TILE = tile_tokens<D>();
  const PagedParams& p = a.p;
  extern __shared__ __align__(256) uint8_t smem[];  // (rows of up to 256 bytes are addressed with exclusive ors)
  __shared__ float2 ml[kWarps][kRows];
  __shared__ unsigned bad_pages[kWarps][ST];
  ptx::wait_for_previous_kernel();
  ptx::allow_next_kernel();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int heads = p.pages.kv_heads * a.h.subs;

  // SHORT: the cluster has one sequence and head, and each of its CTAs an equal part of the tiles, perhaps none.
  // Else: where this CTA's stretch begins.  Every warp finds it by itself, 32 sequences at a time: no barrier, one trip to memory
  // for up to 32 sequences.
  int per, at_tile;  // tiles of a CTA; place on the line of the tile at the cursor
  Cursor<TILE> ic;
  if constexpr (SHORT) {
    const int unit = blockIdx.x / a.cluster, rank = blockIdx.x - unit * a.cluster;
    ic.s = unit / heads;
    ic.head = unit - ic.s * heads;
    ic.q = sequence(p, __ldg(p.lengths + ic.s), TILE);
    per = (ic.q.count + a.cluster - 1) / a.cluster;
    at_tile = 0;
    ic.i = rank * per;
    ic.left = max(min(per, ic.q.count - ic.i), 0);
  } else {
    int total = 0, mine = 0, n[kAhead];
#pragma unroll 1
    for (int s0 = 0; s0 < p.seqs; s0 += 32 * kAhead) {  // (kAhead lengths of a lane are asked for together)
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const int s = s0 + k * 32 + lane;
        n[k] = s < p.seqs ? __ldg(p.lengths + s) : 0;
      }
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        if (k > 0 && s0 + k * 32 >= p.seqs) break;
        mine = s0 + k * 32 + lane < p.seqs ? sequence(p, n[k], TILE).count : 0;
        total += mine;
      }
    }
    total = __reduce_add_sync(0xffffffffu, total) * heads;
    per = (total + static_cast<int>(gridDim.x) - 1) / static_cast<int>(gridDim.x);
    const long long first = static_cast<long long>(blockIdx.x) * per;
    if (first >= total) {
      if (threadIdx.x == 0 && !a.part.by_unit) a.part.joins[blockIdx.x] = make_int4(-1, 0, 0, 0);
      return;
    }
    at_tile = static_cast<int>(first);
    int before = 0;
#pragma unroll 1
    for (int s0 = 0;; s0 += 32) {
      if (p.seqs > 32) {
        n[0] = s0 + lane < p.seqs ? __ldg(p.lengths + s0 + lane) : 0;
        mine = s0 + lane < p.seqs ? sequence(p, n[0], TILE).count : 0;
      }
      // most chunks end before the stretch begins
      const int all = __reduce_add_sync(0xffffffffu, mine);
      if ((before + all) * heads <= at_tile) {
        before += all;
        continue;
      }
      int sum = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += x;
      }
      // the first sequence that ends behind the stretch's beginning
      const int which = __ffs(__ballot_sync(0xffffffffu, (before + sum) * heads > at_tile)) - 1;
      ic.s = s0 + which;
      ic.q = sequence(p, __shfl_sync(0xffffffffu, n[0], which), TILE);
      const int within = at_tile - (before + __shfl_sync(0xffffffffu, sum - mine, which)) * heads;
      ic.head = within / ic.q.count;
      ic.i = within - ic.head * ic.q.count;
      break;
    }
    ic.left = min(per, total - at_tile);
  }
  Cursor<TILE> cc = ic;
  const int cc_s = ic.s, cc_head = ic.head;
  const bool idle = ic.left == 0;

  const uint32_t ring = ptx::smem_u32(smem) + warp * (ST * 2 * BYTES);
  float* join_buf = reinterpret_cast<float*>(smem + kWarps * ST * 2 * BYTES);  // [warps][8][D]
  // SHORT: what this CTA has to join, over the ring
  float* result = reinterpret_cast<float*>(smem);
  float2* result_ml = reinterpret_cast<float2*>(smem + kRows * D * sizeof(float));
  const uint16_t* cache = static_cast<const uint16_t*>(p.cache);
  const long long value_off = p.pages.value_offset();

  // Loads run ahead, and the page of a lane's token is asked for one strip before its load: nothing here waits for it.
  int page = 0, place = 0;
  bool seen = false, listed = false;
  auto look_up = [&] {
    seen = false;
    if (ic.left > 0) {
      const int pos = ic.first_token() + warp * TOK + (lane & (TOK - 1));
      seen = is_visible(ic.q.length - 1, pos, ic.q.length, p.window, p.sinks);
      const int slot = static_cast<int>(p.pages.by_page.div(static_cast<uint32_t>(pos)));
      place = pos - slot * p.pages.page_size;
      listed = seen && slot < p.width;
      if (listed) page = __ldg(p.table + ic.s * p.table_stride + slot);
    }
  };
  auto issue = [&](int slot) {
    if (ic.left > 0) {
      const int kv_head = ic.head / a.h.subs;
      const uint32_t dst = ring + slot * (2 * BYTES);
      const bool found = listed && p.pages.has(page);
      const long long mine = found ? p.pages.key_offset(page, kv_head, place) : -1;
      const unsigned any_bad = __ballot_sync(0xffffffffu, seen && !found);
      if (lane == 0) bad_pages[warp][slot] = any_bad | (ic.q.bad ? 1u : 0u);
      // A strip that is seen whole and lies in one stretch of memory (pages of whole strips) needs one address; else each row's
      // comes from the lane that looked its token up.
      constexpr int ROWS = 32 / CH;  // of an instruction
      const int row0 = lane / CH, ch = lane % CH;
      const uint32_t to = dst + row0 * (D * 2) + ((ch ^ row0) << 4);
      const long long begin = __shfl_sync(0xffffffffu, mine, 0);
      if (__all_sync(0xffffffffu, found && mine == begin + (lane & (TOK - 1)) * D)) {
        const uint16_t* src = cache + begin + row0 * D + ch * 8;
        const uint16_t* src_v = src + value_off;
#pragma unroll
        for (int i = 0; i < TOK / ROWS; ++i) {
          const uint32_t at = (to ^ (((i * ROWS) & 7) << 4)) + i * ROWS * (D * 2);
          copy16(at, src + i * ROWS * D);
          copy16(at + BYTES, src_v + i * ROWS * D);
        }
      } else {
#pragma unroll
        for (int i = 0; i < TOK / ROWS; ++i) {
          const long long off = __shfl_sync(0xffffffffu, mine, i * ROWS + row0);
          const bool take = off >= 0;
          const uint16_t* src = cache + (take ? off + ch * 8 : 0);
          const uint32_t at = (to ^ (((i * ROWS) & 7) << 4)) + i * ROWS * (D * 2);
          copy16(at, src, take);
          copy16(at + BYTES, src + (take ? value_off : 0), take);
        }
      }
      ic.advance(p, heads);
      look_up();
    }
    copy_commit();
  };
  look_up();
#pragma unroll
  for (int i = 0; i < ST - 1; ++i) issue(i);

  // Tokens are the rows of the products and query heads their columns, eight at a time: S^T = K q^T, O^T += V^T P^T.  (The
  // other way round up to eight heads would fill half of 16 rows.)
  const int gr = lane >> 2, gc = lane & 3;  // row and column pair of a fragment
  uint32_t qf[D / 16][NT][2];
  float o[D / 16][NT][4], m[NT][2], l[NT][2];
  bool fresh = true, spoiled = false, whole_start = cc.i == 0, first_segment = true;
  int4 join = make_int4(-1, 0, 0, 0);
  int slot = 0, next_slot = ST - 1;
  auto load_queries = [&](int s, int head) {
    const int kv_head = head / a.h.subs, sub = head - kv_head * a.h.subs;
    const int rows = min(a.h.rows, a.h.group - sub * a.h.rows);
    const uint16_t* q = static_cast<const uint16_t*>(p.q) + s * p.q_stride[0] +
                        (kv_head * a.h.group + sub * a.h.rows) * p.q_stride[1] + gc * 2;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int r = nt * 8 + gr;
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          qf[ks][nt][e] = r < rows ? __ldg(reinterpret_cast<const uint32_t*>(q + r * p.q_stride[1] + ks * 16 + e * 8)) : 0u;
        }
      }
    }
  };
  if (cc.left > 0) load_queries(cc.s, cc.head);
  while (cc.left > 0) {
    const int kv_head = cc.head / a.h.subs, sub = cc.head - kv_head * a.h.subs;
    const int head0 = kv_head * a.h.group + sub * a.h.rows;
    const int rows = min(a.h.rows, a.h.group - sub * a.h.rows);
    if (fresh) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int i = 0; i < D / 16; ++i) o[i][nt][0] = o[i][nt][1] = o[i][nt][2] = o[i][nt][3] = 0.f;
        m[nt][0] = m[nt][1] = -INFINITY;
        l[nt][0] = l[nt][1] = 0.f;
      }
      spoiled = false;
      fresh = false;
    }
    copy_wait<ST - 2>();
    __syncwarp();
    issue(next_slot);
    const uint32_t keys = ring + slot * (2 * BYTES), values = keys + BYTES;
    spoiled |= bad_pages[warp][slot] != 0;

    float c[TOK / 16][NT][4];
#pragma unroll
    for (int t = 0; t < TOK / 16; ++t) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) c[t][nt][0] = c[t][nt][1] = c[t][nt][2] = c[t][nt][3] = 0.f;
    }
    {
      const int row = lane & 15;
      const uint32_t at = keys + row * (D * 2) + (((lane >> 4) ^ (row & 7)) << 4);
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
#pragma unroll
        for (int t = 0; t < TOK / 16; ++t) {
          uint32_t k[4];
          ldmatrix_x4(k, (at ^ (ks << 5)) + t * 16 * (D * 2));
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma_16x8x16<BF16>(c[t][nt], k, qf[ks][nt][0], qf[ks][nt][1]);
        }
      }
    }
    if (a.sign != 1.f) {  // (the largest score is looked for before scaling)
#pragma unroll
      for (int t = 0; t < TOK / 16; ++t) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
          for (int e = 0; e < 4; ++e) c[t][nt][e] *= a.sign;
        }
      }
    }
    const int pos0 = cc.first_token() + warp * TOK;
    const int asks = cc.q.length - 1;  // the position that asks
    if (pos0 + TOK > cc.q.length || (p.window > 0 && asks - pos0 >= p.window && pos0 + TOK > p.sinks)) {
#pragma unroll
      for (int t = 0; t < TOK / 16; ++t) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          if (!is_visible(asks, pos0 + t * 16 + e * 8 + gr, cc.q.length, p.window, p.sinks)) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) c[t][nt][e * 2] = c[t][nt][e * 2 + 1] = -INFINITY;
          }
        }
      }
    }
    bool raised = false;
    float alpha[NT][2];
    uint32_t pf[TOK / 16][NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        float top = m[nt][x];
#pragma unroll
        for (int t = 0; t < TOK / 16; ++t) top = fmaxf(top, fmaxf(c[t][nt][x], c[t][nt][x + 2]));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
        const float base = top == -INFINITY ? 0.f : top * a.scale_log2, shift = kFactor<BF16> - base;
        alpha[nt][x] = exp2_fast(m[nt][x] * a.scale_log2 - base);
        raised |= top != m[nt][x];
        m[nt][x] = top;
        l[nt][x] *= alpha[nt][x];
#pragma unroll
        for (int t = 0; t < TOK / 16; ++t) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float& w = c[t][nt][e * 2 + x];
            w = exp2_fast(w * a.scale_log2 + shift);
            l[nt][x] += w;
          }
        }
      }
      // weights are rounded to the type of the values, as the tensor cores take them; their sum, which has the same factor, is not
#pragma unroll
      for (int t = 0; t < TOK / 16; ++t) {
        pf[t][nt][0] = transpose_8x8(pack<BF16>(c[t][nt][0], c[t][nt][1]));
        pf[t][nt][1] = transpose_8x8(pack<BF16>(c[t][nt][2], c[t][nt][3]));
      }
    }
    if (__any_sync(0xffffffffu, raised)) {
#pragma unroll
      for (int i = 0; i < D / 16; ++i) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
          for (int e = 0; e < 4; ++e) o[i][nt][e] *= alpha[nt][e & 1];
        }
      }
    }
    {
      const int row = (lane & 7) + ((lane >> 4) << 3);
      const uint32_t at = values + row * (D * 2) + ((((lane >> 3) & 1) ^ (row & 7)) << 4);
#pragma unroll
      for (int t = 0; t < TOK / 16; ++t) {
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          uint32_t v[4];
          ldmatrix_x4_trans(v, (at ^ (i << 5)) + t * 16 * (D * 2));
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma_16x8x16<BF16>(o[i][nt], v, pf[t][nt][0], pf[t][nt][1]);
        }
      }
    }
    slot = slot + 1 == ST ? 0 : slot + 1;
    next_slot = next_slot + 1 == ST ? 0 : next_slot + 1;

    // The end of a sequence and head, or of the CTA's stretch: the warps join, eight rows at a time.
    const bool whole_end = cc.i == cc.q.count - 1;
    if (whole_end || cc.left == 1) {
      // the next sequence's or head's queries are on their way meanwhile
      if (!SHORT && cc.left > 1) {
        const bool same = cc.head + 1 < heads;
        load_queries(same ? cc.s : cc.s + 1, same ? cc.head + 1 : 0);
      }
      const bool whole = SHORT ? a.cluster == 1 : whole_start && whole_end;
      const long long part = 2ll * blockIdx.x + (first_segment ? 0 : 1);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          l[nt][x] += __shfl_xor_sync(0xffffffffu, l[nt][x], 4);
          l[nt][x] += __shfl_xor_sync(0xffffffffu, l[nt][x], 8);
          l[nt][x] += __shfl_xor_sync(0xffffffffu, l[nt][x], 16);
          if (spoiled) l[nt][x] = NAN;
          if (gr == 0) ml[warp][nt * 8 + gc * 2 + x] = make_float2(m[nt][x] * a.scale_log2, l[nt][x]);
        }
      }
#pragma unroll
      for (int r = 0; r < NT; ++r) {
        const int rows_here = min(rows - r * 8, 8);
        if (rows_here > 0) {
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            const int row = gc * 2 + x;
            if (row < rows_here) {  // (columns exchanged so that rows begin in different banks)
              float* to = join_buf + (warp * 8 + row) * D;
#pragma unroll
              for (int i = 0; i < D / 16; ++i) {
                to[(i * 16 + gr) ^ (gc << 3)] = o[i][r][x];
                to[(i * 16 + 8 + gr) ^ (gc << 3)] = o[i][r][x + 2];
              }
            }
          }
          __syncthreads();
          for (int x = threadIdx.x; x < rows_here * (D / 4); x += kThreads) {
            const int row = x / (D / 4), col = (x - row * (D / 4)) * 4;
            float most = -INFINITY;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) most = fmaxf(most, ml[w][row + r * 8].x);
            const float base = most == -INFINITY ? 0.f : most;
            float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
            float sum = 0.f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
              const float2 its = ml[w][row + r * 8];
              const float scale = exp2_fast(its.x - base);
              const float4 z = *reinterpret_cast<const float4*>(join_buf + (w * 8 + row) * D + (col ^ ((row >> 1) << 3)));
              sum += its.y * scale;
              y.x += z.x * scale;
              y.y += z.y * scale;
              y.z += z.z * scale;
              y.w += z.w * scale;
            }
            if (whole) {
              // nothing visible: zero.  (A sum that is not a number stays one.)
              const float inv = sum == 0.f ? 0.f : 1.f / sum;
              *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) +
                                        (static_cast<long long>(cc.s) * p.heads + head0 + r * 8 + row) * D + col) =
                  make_uint2(pack<BF16>(y.x * inv, y.y * inv), pack<BF16>(y.z * inv, y.w * inv));
            } else if constexpr (SHORT) {
              // (nothing is on its way into the ring any more)
              *reinterpret_cast<float4*>(result + (r * 8 + row) * D + col) = y;
              if (col == 0) result_ml[r * 8 + row] = make_float2(most, sum);
            } else {
              const long long to = part * a.h.rows + r * 8 + row;
              *reinterpret_cast<float4*>(a.part.out + to * D + col) = y;
              if (col == 0) a.part.ml[to] = make_float2(most, sum);
            }
          }
          __syncthreads();
        }
      }
      if (!SHORT && whole_start) {
        const int begin = at_tile - cc.i;  // first tile of this sequence and head
        const int4 mine = whole_end ? make_int4(-1, 0, 0, 0)
                                    : make_int4(cc.s, cc.head, static_cast<int>(part),
                                                (begin + cc.q.count - 1) / per - static_cast<int>(blockIdx.x) + 1);
        if (!whole_end) join = mine;
        if (a.part.by_unit && threadIdx.x == 0) a.part.joins[cc.s * heads + cc.head] = mine;
      }
      fresh = true;
      whole_start = true;
      first_segment = false;
    }
    ++at_tile;
    cc.advance(p, heads);
  }
  if constexpr (SHORT) {
    if (a.cluster == 1) return;
    // The CTAs of the cluster join what they have: each takes an equal share of the rows' columns.
    const int kv_head = cc_head / a.h.subs, sub = cc_head - kv_head * a.h.subs;
    const int head0 = kv_head * a.h.group + sub * a.h.rows;
    const int rows = min(a.h.rows, a.h.group - sub * a.h.rows);
    const int rank = static_cast<int>(blockIdx.x) - static_cast<int>(blockIdx.x) / a.cluster * a.cluster;
    if (idle && threadIdx.x < kRows) result_ml[threadIdx.x] = make_float2(-INFINITY, 0.f);
    ptx::cluster_sync();
    const uint32_t from = ptx::smem_u32(result), from_ml = ptx::smem_u32(result_ml);
    for (int x = rank * kThreads + threadIdx.x; x < rows * (D / 4); x += a.cluster * kThreads) {
      const int row = x / (D / 4), col = (x - row * (D / 4)) * 4;
      float2 its[kMaxCluster];
      float4 z[kMaxCluster];
      float most = -INFINITY;
#pragma unroll
      for (int c = 0; c < kMaxCluster; ++c) {
        its[c] = make_float2(-INFINITY, 0.f);
        if (c < a.cluster) {
          its[c] = ld_cluster_f2(ptx::mapa_shared(from_ml + row * 8, c));
          z[c] = ld_cluster_f4(ptx::mapa_shared(from + (row * D + col) * 4, c));
        }
      }
#pragma unroll
      for (int c = 0; c < kMaxCluster; ++c) most = fmaxf(most, its[c].x);
      const float base = most == -INFINITY ? 0.f : most;
      float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
      float sum = 0.f;
#pragma unroll
      for (int c = 0; c < kMaxCluster; ++c) {
        if (its[c].x == -INFINITY && its[c].y == 0.f) continue;  // nothing visible there, perhaps nothing written
        const float scale = exp2_fast(its[c].x - base);
        sum += its[c].y * scale;
        y.x += z[c].x * scale;
        y.y += z[c].y * scale;
        y.z += z[c].z * scale;
        y.w += z[c].w * scale;
      }
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + (static_cast<long long>(cc_s) * p.heads + head0 + row) * D + col) =
          make_uint2(pack<BF16>(y.x * inv, y.y * inv), pack<BF16>(y.z * inv, y.w * inv));
    }
    ptx::cluster_sync();  // nobody leaves while its results are read
  } else {
    if (!a.part.by_unit && threadIdx.x == 0) a.part.joins[blockIdx.x] = join;
  }
}

// Joins the parts of one sequence and query head (blockIdx.y): warps take parts in turn, lanes take columns.
template <int D, int WARPS, bool BF16>
__global__ void __launch_bounds__(WARPS * 32) join_kernel(const __grid_constant__ PagedArgs a) {
  constexpr int V = D / 32;
  __shared__ __align__(16) float red[WARPS][D];
  __shared__ float2 sums[WARPS];
  ptx::wait_for_previous_kernel();
  ptx::allow_next_kernel();
  const int4 join = a.part.joins[blockIdx.x];
  if (join.x < 0) return;
  const int kv_head = join.y / a.h.subs, sub = join.y - kv_head * a.h.subs;
  const int r = blockIdx.y;
  if (r >= min(a.h.rows, a.h.group - sub * a.h.rows)) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  auto row_of = [&](int i) {
    const long long slot = i == 0 ? join.z : 2ll * ((join.z >> 1) + i);
    return slot * a.h.rows + r;
  };
  // kBatch parts of a warp in flight, with a running largest score
  constexpr int kBatch = WARPS == 4 ? 4 : 5;
  float acc[V] = {}, sum = 0.f, most = -INFINITY;
  for (int i0 = warp; i0 < join.w; i0 += WARPS * kBatch) {
    float2 ml[kBatch];
    float x[kBatch][V];
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const int i = i0 + k * WARPS;
      const long long row = row_of(min(i, join.w - 1));
      ml[k] = a.part.ml[row];
      const float* src = a.part.out + row * D + lane * V;
      if constexpr (V == 4) {
        const float4 y = *reinterpret_cast<const float4*>(src);
        x[k][0] = y.x;
        x[k][1] = y.y;
        x[k][2] = y.z;
        x[k][3] = y.w;
      } else {
        const float2 y = *reinterpret_cast<const float2*>(src);
        x[k][0] = y.x;
        x[k][1] = y.y;
      }
      if (i >= join.w) ml[k] = make_float2(-INFINITY, 0.f);
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
      // (a part of weight zero adds nothing, also where it is not a number: its sum is then not one either)
#pragma unroll
      for (int v = 0; v < V; ++v) acc[v] += x[k][v] * w;
    }
  }
#pragma unroll
  for (int v = 0; v < V; ++v) red[warp][lane * V + v] = acc[v];
  if (lane == 0) sums[warp] = make_float2(most, sum);
  __syncthreads();
  if (threadIdx.x < D / 2) {
    // a lane has a warp's largest score and sum
    const float2 its = lane < WARPS ? sums[lane] : make_float2(-INFINITY, 0.f);
    float top = its.x;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float mine = exp2_fast(its.x - (top == -INFINITY ? 0.f : top));
    float total = its.y * mine, x = 0.f, y = 0.f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
#pragma unroll 4
    for (int w = 0; w < WARPS; ++w) {
      const float scale = __shfl_sync(0xffffffffu, mine, w);
      const float2 z = *reinterpret_cast<const float2*>(&red[w][threadIdx.x * 2]);
      x += z.x * scale;
      y += z.y * scale;
    }
    const float inv = total == 0.f ? 0.f : 1.f / total;
    const int head = kv_head * a.h.group + sub * a.h.rows + r;
    reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(a.p.out) + (static_cast<long long>(join.x) * a.p.heads + head) * D)[threadIdx.x] =
        pack<BF16>(x * inv, y * inv);
  }
}

// Sequences and virtual heads.
long long unit_count(const PagedParams& p) {
  return static_cast<long long>(p.seqs) * p.pages.kv_heads * head_split(p).subs;
}

// The most tiles that a sequence can have, by what the host knows: the width of its table, and the window.
long long most_tiles(const PagedParams& p) {
  const int tile = p.pages.head_dim == 128 ? tile_tokens<128>() : tile_tokens<64>();
  long long tokens = static_cast<long long>(p.width) * p.pages.page_size;
  // (a tile more for the sinks' end, one for the window's)
  if (p.window > 0) tokens = std::min(tokens, static_cast<long long>(p.window) + p.sinks + 2 * tile);
  return std::max<long long>(1, (tokens + tile - 1) / tile);
}
// CTAs of the general form: all that fit the chip together, but no more than there can be tiles.
int grid_size(const PagedParams& p) {
  return static_cast<int>(std::min<long long>(unit_count(p) * most_tiles(p), static_cast<long long>(kCtasPerSm) * device_sm_count()));
}
// Few tiles for each sequence and head: a cluster of CTAs takes them, joins in its shared memory and needs neither
// workspace nor a second kernel.  Returns the CTAs of a cluster, 0 for the general form.  Up to eight tiles a CTA where the
// clusters fill at least half of the chip's places, else up to two: 32 sequences of 256 tokens on 8 heads of 128 take 7.2 us
// (10.3 in the general form), 8 of 2048 13.0 (15.0), one of 1024 6.2 (7.2), one of 4096 would 11.9 (9.0).  In up to two waves: 64
// sequences of up to 512 tokens 20.9 (23.4); with 128 of 256 tokens there is no difference, 256 would lose.  Longer ones go
// the general way although equal lengths would not lose: it does not depend on them.
int short_cluster(const PagedParams& p) {
  const long long units = unit_count(p), tiles = most_tiles(p), slots = static_cast<long long>(kCtasPerSm) * device_sm_count();
  int c = 1;
  while (c < kMaxCluster && c < tiles && units * c * 2 <= slots) c *= 2;
  return (units * c <= slots || units <= 2 * slots) && (tiles + c - 1) / c <= (units * c * 2 >= slots ? 8 : 2) ? c : 0;
}

template <int D, bool BF16>
cudaError_t launch_typed(const PagedParams& p, cudaStream_t stream) {
  PagedArgs a;
  a.p = p;
  a.h = head_split(p);
  a.scale_log2 = p.scale == 0.f ? 1.f : std::fabs(p.scale) * kLog2e;
  a.sign = p.scale > 0.f ? 1.f : p.scale < 0.f ? -1.f : 0.f;
  a.cluster = short_cluster(p);
  a.part = Partials{};
  const long long units = unit_count(p);
  const bool two = a.h.rows > 8;
  cudaError_t e;
  if (a.cluster > 0) {
    const auto kernel = two ? paged_attention_kernel<D, 2, true, BF16> : paged_attention_kernel<D, 1, true, BF16>;
    e = allow_smem(kernel, paged_smem_bytes<D>());
    if (e != cudaSuccess) return e;
    return launch_after(kernel, dim3(static_cast<unsigned>(units * a.cluster)), kThreads, paged_smem_bytes<D>(), stream, a.cluster, a);
  }
  const int grid = grid_size(p);
  char* ws = static_cast<char*>(p.workspace);
  a.part.out = reinterpret_cast<float*>(ws);
  ws += sizeof(float) * 2 * grid * a.h.rows * D;
  a.part.ml = reinterpret_cast<float2*>(ws);
  ws += (sizeof(float2) * 2 * grid * a.h.rows + 15) / 16 * 16;
  a.part.joins = reinterpret_cast<int4*>(ws);
  a.part.by_unit = units < grid;
  const auto kernel = two ? paged_attention_kernel<D, 2, false, BF16> : paged_attention_kernel<D, 1, false, BF16>;
  e = allow_smem(kernel, paged_smem_bytes<D>());
  if (e != cudaSuccess) return e;
  e = launch_after(kernel, dim3(grid), kThreads, paged_smem_bytes<D>(), stream, 1, a);
  if (e != cudaSuccess || grid == 1) return e;
  // Few sequences have many parts (160 in flight in 32 warps), many have few, and then most of these CTAs find nothing to do:
  // small ones come and go faster (16 warps everywhere: 64 sequences 114 us, 109 now; the window's 27.4, 24.5 now).
  const bool many_parts = units * 8 <= grid;
  const auto join = many_parts ? join_kernel<D, 32, BF16> : join_kernel<D, 4, BF16>;
  return launch_after(join, dim3(static_cast<unsigned>(std::min<long long>(units, grid)), a.h.rows), many_parts ? 1024 : 128, 0,
                      stream, 1, a);
}

}  // namespace

size_t paged_workspace_bytes(const PagedParams& p) {
  if (p.seqs == 0 || short_cluster(p) > 0) return 0;
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
