// How the work of one paged-attention call is shared out, on the device and without the host knowing any length.
//
// The work is a line of tiles, in order of sequence, key head and query tile (T new tokens with the G query heads of one key
// head: T * G rows); a tile is as long as the KV blocks that its rows see, plus a constant for what a tile costs besides.
// CTA c of n takes the stretch [total * c / n, total * (c + 1) / n) of that line, so ragged batches, causal triangles and
// a single sequence over a long cache are all shared evenly. A tile that a border cuts is attended to in parts: each part leaves
// its unnormalised output, maximum and sum in the workspace (at most two parts of a CTA are not whole tiles: its first and
// its last), and a second kernel joins them in order. Nothing waits for another CTA, nothing is counted with atomics, and
// the order of every sum depends on the lengths alone.
//
// Every CTA finds its borders itself, from the lengths: one pass over the batch for the total and one for the places.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "paged_host.h"
#include "sm100_ptx.cuh"

namespace txp {

using namespace txd;

struct Sched {
  const int32_t *kv_lens, *cu_q;
  int32_t batch, tokens, kv_heads, group;
  int32_t tile_tokens;         // T
  int32_t causal, window;      // window 0: none
  int32_t max_kv;              // what the page table has room for
  int32_t block_shift;         // log2 of the KV block
  int32_t tile_cost;           // of a tile besides its blocks, in blocks
  int32_t min_part;            // no part is shorter, in blocks
  int32_t min_share;           // no CTA's share is shorter (fewer CTAs work then)
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

// The place at distance r along the tiles of sequence b, moved to a tile's start where a part would be too short.
__device__ __forceinline__ Cut resolve(const Sched &s, int b, long long r, long long per_head) {
  SeqInfo q = seq_info(s, b);
  Cut c = {b, static_cast<int>(r / per_head), 0, 0};
  r -= c.h * per_head;
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

template <int kThreads>
__device__ __forceinline__ long long block_sum_scan(long long x, long long *total, long long *sums) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long long sum = x;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const long long y = __shfl_up_sync(0xffffffffu, sum, d);
    if (lane >= d) sum += y;
  }
  if (lane == 31) sums[warp] = sum;
  __syncthreads();
  long long before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w < warp) before += sums[w];
    all += sums[w];
  }
  *total = all;
  __syncthreads();
  return before + sum - x;
}

struct SchedSmem {
  long long sums[32];
  Cut cut[2];
};

// For all threads of a CTA: its stretch goes to sm->cut[0], sm->cut[1]; false when there is nothing for it. Its first
// border is also written to `borders` (b = -1 where no tile is cut), for the joining kernel.
template <int kThreads>
__device__ __forceinline__ bool find_stretch(const Sched &s, SchedSmem *sm, int4 *borders) {
  const int cta = blockIdx.x;
  const bool one_pass = s.batch <= kThreads;
  long long mine = 0, per_head = 0, total;
  for (int b = threadIdx.x; b < s.batch; b += kThreads) {
    const SeqInfo q = seq_info(s, b);
    if (cta == 0 && s.kv_lens[b] > s.max_kv) atomicOr(s.status, kNoRoomInRow);
    per_head = head_cost(s, q);
    mine += per_head * s.kv_heads;
  }
  const long long before = block_sum_scan<kThreads>(mine, &total, sm->sums);
  const long long most = total / s.min_share;
  const int n = most < static_cast<int>(gridDim.x) ? max(static_cast<int>(most), 1) : gridDim.x;
  const long long x0 = total * cta / n, x1 = total * (cta + 1) / n;
  if (threadIdx.x == 0) sm->cut[0] = sm->cut[1] = Cut{s.batch, 0, 0, 0};
  __syncthreads();
  if (cta < n) {
    if (one_pass) {
      if (threadIdx.x < s.batch) {
        if (x0 >= before && x0 < before + mine) sm->cut[0] = resolve(s, threadIdx.x, x0 - before, per_head);
        if (x1 >= before && x1 < before + mine) sm->cut[1] = resolve(s, threadIdx.x, x1 - before, per_head);
      }
    } else {
      long long carry = 0;
      for (int base = 0; base < s.batch; base += kThreads) {
        const int b = base + threadIdx.x;
        long long chunk;
        per_head = b < s.batch ? head_cost(s, seq_info(s, b)) : 0;
        mine = per_head * s.kv_heads;
        const long long at = carry + block_sum_scan<kThreads>(mine, &chunk, sm->sums);
        if (x0 >= at && x0 < at + mine) sm->cut[0] = resolve(s, b, x0 - at, per_head);
        if (x1 >= at && x1 < at + mine) sm->cut[1] = resolve(s, b, x1 - at, per_head);
        carry += chunk;
      }
    }
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    const Cut c = sm->cut[0];
    borders[cta] = cta < n && c.blk > 0 ? make_int4(c.b, c.h, c.i, c.blk) : make_int4(-1, 0, 0, 0);
  }
  const Cut a = sm->cut[0], b = sm->cut[1];
  return cta < n && !(same_tile(a, b) && a.blk == b.blk);
}

// A stretch walked tile by tile (every role warp walks it by itself).
struct Walk {
  Cut at, end;
  SeqInfo q;
  TileInfo t;
  int from, to;  // blocks of the current tile in this stretch, relative to its first
  __device__ __forceinline__ bool start(const Sched &s, const SchedSmem *sm) {
    at = sm->cut[0];
    end = sm->cut[1];
    if (at.b >= s.batch || (same_tile(at, end) && at.blk == end.blk)) return false;
    q = seq_info(s, at.b);
    load(s);
    return true;
  }
  __device__ __forceinline__ void load(const Sched &s) {
    t = tile_info(s, q, at.i);
    from = at.blk;
    to = same_tile(at, end) ? end.blk : t.n;
  }
  __device__ __forceinline__ bool next(const Sched &s) {
    if (same_tile(at, end)) return false;
    next_tile(s, at, q);
    if (at.b >= s.batch || (same_tile(at, end) && end.blk == 0)) return false;
    load(s);
    return true;
  }
  __device__ __forceinline__ bool whole() const { return from == 0 && to == t.n; }
  __device__ __forceinline__ int slot() const { return from > 0 ? 0 : 1; }  // of this CTA's two partial results
};

// ---- joining the parts of cut tiles --------------------------------------------------------------------------------
struct JoinParams {
  Sched s;
  const int4 *borders;  // [ctas]
  const float *part;    // [ctas][2][rows][D], then
  const float2 *ml;     // [ctas][2][rows]: maximum (log2 units) and sum
  void *out;
  float *m_out;
  long long out_stride[2];
  int32_t ctas, rows, heads, head_dim;
};

// One warp joins one row: o = sum_i 2^(m_i - M) o_i / sum_i 2^(m_i - M) l_i. The parts of a tile are those of consecutive
// CTAs; the block of a tile's first border does the tile. Bound by latency when there are few rows and by reading the
// parts when there are many (L2 holds them).
template <typename T, int D>
__global__ void __launch_bounds__(256) paged_join_kernel(const __grid_constant__ JoinParams p) {
  constexpr int kVec = D / 32;  // columns of a lane
  grid_dep_wait();
  const int c = static_cast<int>(blockIdx.x) + 1, lane = threadIdx.x & 31;
  const int4 cut = p.borders[c], prev = p.borders[c - 1];
  if (cut.x < 0 || (prev.x == cut.x && prev.y == cut.y && prev.z == cut.z)) return;
  const SeqInfo q = seq_info(p.s, cut.x);
  const int t0 = cut.z * p.s.tile_tokens, t1 = min(t0 + p.s.tile_tokens, q.q);
  const int row = static_cast<int>(blockIdx.y) * 8 + static_cast<int>(threadIdx.x >> 5);
  if (row >= (t1 - t0) * p.s.group) return;
  int parts = 2;  // of CTAs c - 1 and c, and of those behind whose border lies in the tile as well
  for (bool more = true; more; ) {
    const int k = c + parts - 1 + lane;
    int4 x = make_int4(-1, 0, 0, 0);
    if (k < p.ctas) x = p.borders[k];
    const uint32_t in = __ballot_sync(0xffffffffu, x.x == cut.x && x.y == cut.y && x.z == cut.z);
    const int run = in == 0xffffffffu ? 32 : __ffs(~in) - 1;
    parts += run;
    more = run == 32;
  }
  auto place = [&](int i) { return (static_cast<long long>(c - 1 + i) * 2 + (i == 0 ? 1 : 0)) * p.rows + row; };
  float top = -INFINITY;
  for (int i = lane; i < parts; i += 32) top = fmaxf(top, p.ml[place(i)].x);
#pragma unroll
  for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
  const float ref = top == -INFINITY ? 0.f : top;
  float acc[kVec], sum = 0.f;
#pragma unroll
  for (int e = 0; e < kVec; ++e) acc[e] = 0.f;
  for (int base = 0; base < parts; base += 32) {
    float2 ml = make_float2(-INFINITY, 0.f);
    if (base + lane < parts) ml = p.ml[place(base + lane)];
    const float mine = fast_exp2(ml.x - ref);
    const int count = min(parts - base, 32);
#pragma unroll 4
    for (int i = 0; i < count; ++i) {
      const float w = __shfl_sync(0xffffffffu, mine, i), l = __shfl_sync(0xffffffffu, ml.y, i);
      // a part that saw nothing has left no output
      if (w > 0.f) {
        sum += w * l;
        const float *o = p.part + place(base + i) * D + lane * kVec;
#pragma unroll
        for (int e = 0; e < kVec; e += 2) {
          const float2 x = *reinterpret_cast<const float2 *>(o + e);
          acc[e] += w * x.x;
          acc[e + 1] += w * x.y;
        }
      }
    }
  }
  const float inv = sum > 0.f ? 1.f / sum : 0.f;
  const int tok = q.q0 + t0 + row / p.s.group, head = cut.y * p.s.group + row % p.s.group;
  T *out = static_cast<T *>(p.out) + tok * p.out_stride[0] + head * p.out_stride[1] + lane * kVec;
#pragma unroll
  for (int e = 0; e < kVec; ++e)
    if (lane * kVec + e < p.head_dim) out[e] = static_cast<T>(acc[e] * inv);  // rounded once, to nearest
  if (p.m_out && lane == 0) p.m_out[static_cast<long long>(tok) * p.heads + head] = sum > 0.f ? top + log2f(sum) : -INFINITY;
}

}  // namespace txp
