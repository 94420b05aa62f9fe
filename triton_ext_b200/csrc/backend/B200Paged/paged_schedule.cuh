// How the work of one paged-attention call is shared out, on the device and without the host knowing any length.
//
// The work is a line of tiles, in order of sequence, key head and query tile (T new tokens with the G query heads of one key
// head: T * G rows); a tile is as long as the KV blocks that its rows see, plus a constant for what a tile costs besides.
// Few long tiles (a single sequence over a long cache, a batch of single tokens): the line is cut into n equal stretches, one
// a CTA. Many tiles: the first F * n are dealt out whole, wave by wave, every second wave in reverse, so that the CTAs that
// run at the same time are at neighbouring tiles and share their keys and values through L2 (all CTAs on contiguous
// stretches took 4.74 ms for 32 heads of 16384 tokens of 128, this 3.85: every head's keys were in use at once); the
// rest of the line is cut so that all CTAs come to the same length. Either way a CTA has at most two parts of tiles:
// those leave their unnormalised output, maximum and sum in the workspace, and a second kernel joins them in order.
// Nothing waits for another CTA, nothing is counted with atomics, and the order of every sum depends on the lengths alone.
//
// Every CTA finds its borders itself, from the lengths: one pass over the batch for the total and one for the places.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "paged_host.h"
#include "sm100_ptx.cuh"

namespace txp {

using namespace txd;

constexpr uint32_t kWaitRanOut = kTimeout | kStatusIsBits;  // what the kernels' bounded waits report

struct Sched {
  const int32_t *kv_lens, *cu_q;
  int32_t batch, tokens, kv_heads, group;
  int32_t tile_tokens;         // T
  int32_t causal, window;      // window 0: none
  int32_t max_kv;              // what the page table has room for
  int32_t block_shift;         // log2 of the KV block
  int32_t tile_cost;           // of a tile besides its blocks, in blocks
  int32_t min_part;            // no part is shorter, in blocks
  int32_t min_share;           // no stretch is shorter (there are fewer then)
  int32_t waves;               // at most so many waves of whole tiles
  uint32_t *status;
};

struct SeqInfo {
  int q0, q, kv;
};

struct Cut {  // a place on the line: before block `blk` of a tile
  int b, h, i, blk;
};

struct TileInfo {
  int t0, t1;       // new tokens [t0, t1)
  int off;          // position of new token 0
  int lo, hi;       // keys that some row of the tile sees: [lo, hi)
  int blk0, n;      // first block and number of blocks
};

__device__ __forceinline__ SeqInfo seq_info(const Sched &s, int b) {
  SeqInfo r;
  if (s.cu_q) {
    r.q0 = min(max(s.cu_q[b], 0), s.tokens);
    r.q = max(min(s.cu_q[b + 1], s.tokens), r.q0) - r.q0;
  } else {
    r.q0 = b;
    r.q = b < s.tokens ? 1 : 0;
  }
  r.kv = min(max(s.kv_lens[b], 0), s.max_kv);
  return r;
}

__device__ __forceinline__ TileInfo tile_info(const Sched &s, const SeqInfo &q, int i) {
  TileInfo t;
  t.t0 = i * s.tile_tokens;
  t.t1 = min(t.t0 + s.tile_tokens, q.q);
  t.off = q.kv - q.q;
  t.hi = s.causal ? max(t.off + t.t1, 0) : q.kv;
  t.lo = s.window ? min(max(t.off + t.t0 + 1 - s.window, 0), t.hi) : 0;
  t.blk0 = t.lo >> s.block_shift;
  t.n = t.hi > t.lo ? ((t.hi + (1 << s.block_shift) - 1) >> s.block_shift) - t.blk0 : 0;
  return t;
}

__device__ __forceinline__ int tiles_of(const Sched &s, const SeqInfo &q) {
  return (q.q + s.tile_tokens - 1) / s.tile_tokens;
}

// One thread adds a sequence's tiles up, and resolve walks them again: 0.1 us a tile. Nothing next to the work of a prompt with
// keys, but all there is to a call of very many empty tiles (32768 new tokens of 64 query heads to a key head and no keys, 8192
// tiles: 904 us as one sequence, 97 as 128).
__device__ __forceinline__ long long head_cost(const Sched &s, const SeqInfo &q) {
  long long c = 0;
  for (int t = 0, i = 0; t < q.q; t += s.tile_tokens, ++i) c += tile_info(s, q, i).n + s.tile_cost;
  return c;
}

// The tile after tile (b, h, i); sequences without new tokens have none. `q` follows to the sequence.
__device__ __forceinline__ void next_tile(const Sched &s, Cut &c, SeqInfo &q) {
  c.blk = 0;
  if (++c.i * s.tile_tokens < q.q) return;
  c.i = 0;
  if (++c.h < s.kv_heads) return;
  c.h = 0;
  while (++c.b < s.batch) {
    q = seq_info(s, c.b);
    if (q.q > 0) return;
  }
}

__device__ __forceinline__ bool same_tile(const Cut &a, const Cut &b) { return a.b == b.b && a.h == b.h && a.i == b.i; }

// Quotient of non-negative numbers, by the short division where both are short.
__device__ __forceinline__ long long quotient(long long a, long long b) {
  if (((a | b) >> 32) == 0) return static_cast<uint32_t>(a) / static_cast<uint32_t>(b);
  return a / b;
}

// The place at distance r along the tiles of sequence b, moved to a tile's start where a part would be too short.
__device__ __forceinline__ Cut resolve(const Sched &s, int b, long long distance, long long per_head) {
  SeqInfo q = seq_info(s, b);
  const int h = static_cast<int>(quotient(distance, per_head));
  long long r = distance - h * per_head;
  Cut c = {b, h, 0, 0};
  TileInfo t = tile_info(s, q, 0);
  while (r >= t.n + s.tile_cost) {
    r -= t.n + s.tile_cost;
    t = tile_info(s, q, ++c.i);
  }
  c.blk = max(static_cast<int>(r) - s.tile_cost, 0);
  if (c.blk < s.min_part) c.blk = 0;
  else if (t.n - c.blk < s.min_part) next_tile(s, c, q);
  return c;
}

// Exclusive prefix sums over a block, of one or two values a thread at once; their totals for everyone.
template <int kThreads, int kValues>
__device__ __forceinline__ void block_scan(long long (&x)[kValues], long long (&total)[kValues], long long *sums) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  constexpr int kWarps = kThreads / 32;
#pragma unroll
  for (int v = 0; v < kValues; ++v) {
    long long sum = x[v];
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const long long y = __shfl_up_sync(0xffffffffu, sum, d);
      if (lane >= d) sum += y;
    }
    if (lane == 31) sums[v * 32 + warp] = sum;
    x[v] = sum - x[v];
  }
  __syncthreads();
#pragma unroll
  for (int v = 0; v < kValues; ++v) {
    long long before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const long long y = sums[v * 32 + w];
      if (w < warp) before += y;
      all += y;
    }
    x[v] += before;
    total[v] = all;
  }
  __syncthreads();
}

constexpr int kMaxWaves = 16;

struct SchedSmem {
  long long sums[64];
  long long x[2];               // this CTA's stretch
  int waves;
  Cut cut[kMaxWaves + 2];       // its whole tiles, then the ends of its stretch
};

// What the dealing-out of whole tiles needs of every sequence; one entry a thread.
struct SeqTable {
  int *tiles_before, *q, *kv;   // tiles of the sequences before; the sequence's lengths
};

__device__ __forceinline__ Cut tile_at(const Sched &s, const SeqTable &tab, int index) {
  int lo = 0, hi = s.batch - 1;  // the last sequence whose tiles start at or before the index
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (tab.tiles_before[mid] <= index) lo = mid;
    else hi = mid - 1;
  }
  const int per_head = (tab.q[lo] + s.tile_tokens - 1) / s.tile_tokens;
  const int r = index - tab.tiles_before[lo], h = r / per_head;
  return Cut{lo, h, r - h * per_head, 0};
}

__device__ __forceinline__ int tile_length(const Sched &s, const SeqTable &tab, const Cut &c) {
  return tile_info(s, SeqInfo{0, tab.q[c.b], tab.kv[c.b]}, c.i).n + s.tile_cost;
}

// For all threads of a CTA: its work goes to *sm, and the first border of its stretch also to `borders` (b = -1 where no
// tile is cut; block -1 where the stretch is empty), for the joining kernel. kWaves: whole tiles are dealt out (`scratch`:
// 3 * kThreads ints of shared memory).
template <int kThreads, bool kWaves>
__device__ __forceinline__ void find_work(const Sched &s, SchedSmem *sm, int4 *borders, int *scratch) {
  const int cta = blockIdx.x, n = gridDim.x, tid = threadIdx.x;
  const bool one_pass = s.batch <= kThreads;
  long long mine = 0, per_head = 0;
  SeqInfo q = {0, 0, 0};
  for (int b = tid; b < s.batch; b += kThreads) {
    q = seq_info(s, b);
    if (cta == 0) {
      // what seq_info has cut to size (fewer cached tokens than new ones are allowed: the first ones see nothing)
      const int len = s.kv_lens[b];
      uint32_t bad = len > s.max_kv ? kNoRoomInRow : len < 0 ? kBadLength : 0u;
      if (s.cu_q && (s.cu_q[b] < 0 || s.cu_q[b + 1] < s.cu_q[b] || s.cu_q[b + 1] > s.tokens)) bad |= kBadOffsets;
      if (bad) atomicOr(s.status, bad);
    }
    per_head = head_cost(s, q);
    mine += per_head * s.kv_heads;
  }
  if (tid < kMaxWaves + 2) sm->cut[tid] = Cut{s.batch, 0, 0, 0};
  if (tid == 0) sm->waves = kMaxWaves, sm->x[0] = sm->x[1] = -1;
  constexpr int kSums = kWaves ? 2 : 1;
  long long before[kSums], totals[kSums];
  before[0] = mine;
  if constexpr (kWaves) before[1] = tid < s.batch ? static_cast<long long>(tiles_of(s, q)) * s.kv_heads : 0;
  block_scan<kThreads, kSums>(before, totals, sm->sums);
  const long long total = totals[0];
  long long skipped = 0;  // length of what is dealt out whole
  int waves = 0;
  long long dealt[2] = {0, 0}, dealt_all[2] = {0, 1};  // thread c: CTA c's whole tiles, and what is left for its stretch
  if constexpr (kWaves) if (one_pass && n <= kThreads && totals[1] >= n && totals[1] < INT32_MAX) {
    const SeqTable tab = {scratch, scratch + kThreads, scratch + 2 * kThreads};
    tab.tiles_before[tid] = static_cast<int>(before[1]);
    tab.q[tid] = q.q;
    tab.kv[tid] = q.kv;
    __syncthreads();
    const int most = min(static_cast<int>(totals[1]) / n, s.waves);
    const long long target = quotient(total, n);
    auto tile_of = [&](int f) { return tile_at(s, tab, f * n + ((f & 1) ? n - 1 - tid : tid)); };
    // only as many waves as no CTA's whole tiles alone are more than its share of the work
    int fit = 0;
    if (tid < n) {
      for (; fit < most; ++fit) {
        const Cut c = tile_of(fit);
        const int length = tile_length(s, tab, c);
        if (dealt[0] + length > target + s.tile_cost) break;
        dealt[0] += length;
        if (tid == cta) sm->cut[fit] = c;
      }
      atomicMin(&sm->waves, fit);
    }
    __syncthreads();
    waves = sm->waves;
    for (int f = waves; f < fit; ++f) dealt[0] -= tile_length(s, tab, tile_of(f));
    if (tid < n) dealt[1] = max(target + 1 - dealt[0], 0ll);
    block_scan<kThreads, 2>(dealt, dealt_all, sm->sums);
    skipped = dealt_all[0];
    if (tid == cta)
      for (int f = waves; f < fit; ++f) sm->cut[f] = Cut{s.batch, 0, 0, 0};
  }
  // ---- the rest of the line ----
  const long long rest = total - skipped;
  const int parts = rest < static_cast<long long>(s.min_share) * n ? max(static_cast<int>(rest) / s.min_share, 1) : n;
  if (waves > 0 && parts == n) {
    // (in double: the product of two lengths may pass 2^63, and rounding keeps the borders' order)
    if (tid == cta || tid == cta + 1)
      sm->x[tid - cta] = skipped + static_cast<long long>(static_cast<double>(rest) * (static_cast<double>(dealt[1]) / static_cast<double>(dealt_all[1])));
    if (tid == cta && cta == n - 1) sm->x[1] = total;
  } else if (tid < 2 && cta < parts && rest > 0) {
    sm->x[tid] = skipped + quotient(rest * (cta + tid), parts);
  }
  if (tid == 0) sm->waves = waves;
  __syncthreads();
  const long long x0 = sm->x[0], x1 = sm->x[1];
  auto place = [&](int b, long long at, long long cost, long long head) {
    if (x0 >= at && x0 < at + cost) sm->cut[waves] = resolve(s, b, x0 - at, head);
    if (x1 >= at && x1 < at + cost) sm->cut[waves + 1] = resolve(s, b, x1 - at, head);
  };
  if (one_pass) {
    if (mine > 0) place(tid, before[0], mine, per_head);
  } else {
    long long carry = 0;
    for (int base = 0; base < s.batch; base += kThreads) {
      const int b = base + tid;
      per_head = b < s.batch ? head_cost(s, seq_info(s, b)) : 0;
      mine = per_head * s.kv_heads;
      long long at[1] = {mine}, chunk[1];
      block_scan<kThreads, 1>(at, chunk, sm->sums);
      if (mine > 0) place(b, carry + at[0], mine, per_head);
      carry += chunk[0];
    }
  }
  __syncthreads();
  if (tid == 0) {
    const Cut c = sm->cut[waves], e = sm->cut[waves + 1];
    const bool empty = same_tile(c, e) && c.blk == e.blk;  // its whole tiles were as long as its share
    borders[cta] = x0 >= 0 && c.blk > 0 ? make_int4(c.b, c.h, c.i, empty ? -1 : c.blk) : make_int4(-1, 0, 0, 0);
  }
}

// A CTA's work walked tile by tile (every role warp walks it by itself).
struct Walk {
  Cut at, end;
  SeqInfo q;
  TileInfo t;
  int from, to;  // blocks of the current tile in this CTA's work, relative to its first
  int wave;
  __device__ __forceinline__ bool start(const Sched &s, const SchedSmem *sm) {
    wave = -1;
    return open(s, sm);
  }
  // the next whole tile, or the stretch
  __device__ __forceinline__ bool open(const Sched &s, const SchedSmem *sm) {
    if (++wave > sm->waves) return false;
    at = sm->cut[wave];
    if (at.b >= s.batch) return false;
    if (wave == sm->waves) {
      end = sm->cut[wave + 1];
      if (same_tile(at, end) && at.blk == end.blk) return false;
    }
    else end = Cut{s.batch, 0, 0, 0};
    q = seq_info(s, at.b);
    load(s);
    if (wave < sm->waves) end = Cut{at.b, at.h, at.i, to};
    return true;
  }
  __device__ __forceinline__ void load(const Sched &s) {
    t = tile_info(s, q, at.i);
    from = at.blk;
    to = same_tile(at, end) ? end.blk : t.n;
  }
  __device__ __forceinline__ bool next(const Sched &s, const SchedSmem *sm) {
    if (same_tile(at, end)) return open(s, sm);
    next_tile(s, at, q);
    if (at.b >= s.batch || (same_tile(at, end) && end.blk == 0)) return open(s, sm);
    load(s);
    return true;
  }
  __device__ __forceinline__ bool whole() const { return from == 0 && to == t.n; }
  // which of the partial results: a CTA has two, for the tile that its stretch begins in and the one that it ends in
  __device__ __forceinline__ long long slot() const { return static_cast<long long>(blockIdx.x) * 2 + (from > 0 ? 0 : 1); }
};

// ---- joining the parts of cut tiles --------------------------------------------------------------------------------
struct JoinParams {
  Sched s;
  const int4 *borders;  // [ctas]
  const float4 *part;   // [ctas][2][D / 4][rows]: four columns of a row together, rows next to each other
  const float2 *ml;     // [ctas][2][rows]: maximum (log2 units) and sum
  void *out;
  float *m_out;
  long long out_stride[2];
  int32_t ctas, rows, heads, head_dim;
};

// The joined value of 16 columns of a row: o = sum_i 2^(m_i - M) o_i / sum_i 2^(m_i - M) l_i.
struct Joined {
  float acc[16], top, sum;
  __device__ __forceinline__ void clear() {
    top = -INFINITY;
    sum = 0.f;
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[e] = 0.f;
  }
  __device__ __forceinline__ void scale_to(float m) {  // a common reference of this and what comes next
    const float next = fmaxf(top, m);
    if (next == top) return;
    const float f = fast_exp2(top - next);
    top = next;
    sum *= f;
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[e] *= f;
  }
};

// The parts of a tile are those of consecutive CTAs; the block of a tile's first border does the tile. A thread joins 16
// columns of a row (32 bytes of output, a whole sector), the threads of a warp are rows, which the parts are laid out for.
// What it costs is loads that wait for one another, so a warp takes 32 borders at once, and the loads of several parts are
// under way together.
// kRows (16 or 32: the rows of the streaming kernel's tiles; single tokens may have a few dozen parts): a block has a tile,
// a warp 16 of its columns, and at 16 rows the half-warps take every second part. 0 (256 rows, two or three parts): a warp
// has 32 rows and 16 columns, bound by reading them. (A thread that walked borders and parts one after another: 12 to 16 us
// of 2 x 131071 or 64 ragged single tokens; all eight warps of a block on 16 columns: 8 us.)
template <typename T, int D, int kRows>
__global__ void __launch_bounds__(kRows ? D * 2 : 256) paged_join_kernel(const __grid_constant__ JoinParams p) {
  constexpr int kColGroups = D / 16, kAtOnce = kRows ? 4 : 2, kSplit = kRows == 16 ? 2 : 1;
  const int c = static_cast<int>(blockIdx.x) + 1, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int unit = kRows ? static_cast<int>(blockIdx.y) * kColGroups + warp : static_cast<int>(blockIdx.y) * 8 + warp;
  const int row = unit / kColGroups * 32 + (kRows == 16 ? lane & 15 : lane), col = unit % kColGroups * 16;
  grid_dep_wait();
  // lane i: the border that CTA c - 1 + i starts at, so part i of the tile that is cut there
  int4 at = make_int4(-1, 0, 0, 0);
  if (c - 1 + lane < p.ctas) at = p.borders[c - 1 + lane];
  const int b = __shfl_sync(0xffffffffu, at.x, 1), h = __shfl_sync(0xffffffffu, at.y, 1), tile = __shfl_sync(0xffffffffu, at.z, 1);
  uint32_t same = __ballot_sync(0xffffffffu, at.x == b && at.y == h && at.z == tile);
  if (b < 0 || (same & 1u)) return;  // no tile is cut here, or it has been cut before
  uint32_t there = __ballot_sync(0xffffffffu, at.w > 0) | 1u;  // an empty stretch has left nothing
  const SeqInfo q = seq_info(p.s, b);
  const int t0 = tile * p.s.tile_tokens, t1 = min(t0 + p.s.tile_tokens, q.q);
  const int rows = (t1 - t0) * p.s.group;
  if (unit / kColGroups * 32 >= rows || col >= p.head_dim) return;  // for the whole warp
  same |= 1u;
  Joined j;
  j.clear();
  for (int base = 0;; base += 32) {
    const int run = same == 0xffffffffu ? 32 : __ffs(~same) - 1;  // parts base .. base + run - 1
    for (int i = kSplit == 2 ? lane >> 4 : 0; i < run; i += kSplit * kAtOnce) {
      float2 ml[kAtOnce];
      float4 x[kAtOnce][4];
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) {
        const int k = i + u * kSplit;
        ml[u] = make_float2(-INFINITY, 0.f);
        if (k < run && (there >> k & 1u) && row < rows) {
          const long long slot = (static_cast<long long>(c - 1 + base) + k) * 2 + (base + k == 0 ? 1 : 0);
          ml[u] = p.ml[slot * p.rows + row];
          const float4 *o = p.part + (slot * (D / 4) + col / 4) * p.rows + row;
#pragma unroll
          for (int e = 0; e < 4; ++e) x[u][e] = o[static_cast<long long>(e) * p.rows];
        }
      }
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u) {
        if (ml[u].x == -INFINITY) continue;  // nothing there, or nothing seen: no output was left
        j.scale_to(ml[u].x);
        const float w = fast_exp2(ml[u].x - j.top);
        j.sum += w * ml[u].y;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          j.acc[4 * e] += w * x[u][e].x;
          j.acc[4 * e + 1] += w * x[u][e].y;
          j.acc[4 * e + 2] += w * x[u][e].z;
          j.acc[4 * e + 3] += w * x[u][e].w;
        }
      }
    }
    if (run < 32) break;
    at = make_int4(-1, 0, 0, 0);
    const int k = c - 1 + base + 32 + lane;
    if (k < p.ctas) at = p.borders[k];
    same = __ballot_sync(0xffffffffu, at.x == b && at.y == h && at.z == tile);
    there = __ballot_sync(0xffffffffu, at.w > 0);
  }
  if (kSplit == 2) {  // the other half-warp's parts; both halves come to the same
    const float m = __shfl_xor_sync(0xffffffffu, j.top, 16);
    const float next = fmaxf(j.top, m), ref = next == -INFINITY ? 0.f : next;
    const float f = fast_exp2(j.top - ref);
    j.top = next;
    j.sum *= f;
    j.sum += __shfl_xor_sync(0xffffffffu, j.sum, 16);
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      j.acc[e] *= f;
      j.acc[e] += __shfl_xor_sync(0xffffffffu, j.acc[e], 16);
    }
  }
  if (row >= rows || (kSplit == 2 && lane >= 16)) return;
  const float inv = j.sum > 0.f ? 1.f / j.sum : 0.f;
  const int tok = q.q0 + t0 + row / p.s.group, head = h * p.s.group + row % p.s.group;
  struct alignas(16) Eight { T x[8]; } y[2];
#pragma unroll
  for (int e = 0; e < 16; ++e) y[e / 8].x[e % 8] = static_cast<T>(j.acc[e] * inv);  // rounded once, to nearest
  Eight *out = reinterpret_cast<Eight *>(static_cast<T *>(p.out) + tok * p.out_stride[0] + head * p.out_stride[1] + col);
  out[0] = y[0];
  out[1] = y[1];
  if (p.m_out && col == 0)
    p.m_out[static_cast<long long>(tok) * p.heads + head] = j.sum > 0.f ? j.top + log2f(j.sum) : -INFINITY;
}

}  // namespace txp
