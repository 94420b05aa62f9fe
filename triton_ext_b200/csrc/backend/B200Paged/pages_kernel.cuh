// The handling of a cache's pages on the device: who holds which page (table, lens, refs), and copies of page contents.
//
// The bookkeeping is small whole-number work; what it costs is launches and latency, so a reserve or a compaction is
// planned by ONE block (prefix sums over the listed rows and over the reference counts in shared memory, no grid-wide
// step) and its plan, a list of (source, destination) pages in the workspace, is carried out by a second kernel over the
// whole GPU. Copies are bound by HBM: every byte moved is read once and written once (a compaction that moves 214 MB: 67 us,
// 6.4 TB/s); a plan is 5 to 9 us of loads that depend on one another.
//
// Every result is the same from run to run: free pages are taken in ascending order, by the order of the list. Where
// integer atomics are used (reference counts), their order does not matter.
#pragma once

#include "paged_host.h"
#include "sm100_ptx.cuh"

namespace txp {

using namespace txd;

struct PagesParams {
  uint4 *k, *v;
  long long page_vecs;  // 16-byte vectors of one page of one layer
  int32_t *table, *lens, *refs;
  int32_t *ws;          // workspace
  uint32_t *status;
  int32_t layers, num_pages, page_shift, rows, width;
};

// Workspace of a plan: [0] pairs, [1] first moved page, pairs from kPlanPairs on.
constexpr int kPlanPairs = 4;
constexpr int kPlanThreads = 1024;

__global__ void __launch_bounds__(256) pages_free_kernel(const __grid_constant__ PagesParams p, const int32_t *rows) {
  grid_dep_wait();
  const int row = rows[blockIdx.x];
  if (row < 0 || row >= p.rows) {
    if (threadIdx.x == 0) atomicOr(p.status, kBadRow);
    return;
  }
  for (int c = threadIdx.x; c < p.width; c += 256) {
    int32_t *cell = p.table + static_cast<long long>(row) * p.width + c;
    // a row may be listed twice: the exchange hands each page to one of the two only
    const int page = *cell < 0 ? -1 : atomicExch(cell, -1);
    if (page >= 0) {
      if (page < p.num_pages) atomicSub(&p.refs[page], 1);
      else atomicOr(p.status, kBadPage);
    }
  }
  if (threadIdx.x == 0) p.lens[row] = 0;
}

// Rows are cut to keep[i] tokens (drafts that were not accepted); a row listed twice ends at the lesser, whatever the order
// of the blocks: the length is a minimum, and the exchange hands each page to one of the two only.
__global__ void __launch_bounds__(256) pages_truncate_kernel(const __grid_constant__ PagesParams p, const int32_t *rows,
                                                             const int32_t *keep) {
  grid_dep_wait();
  const int row = rows[blockIdx.x], tokens = keep[blockIdx.x];
  if (row < 0 || row >= p.rows || tokens < 0) {
    if (threadIdx.x == 0) atomicOr(p.status, row < 0 || row >= p.rows ? kBadRow : kBadLength);
    return;
  }
  const long long first = (static_cast<long long>(tokens) + (1ll << p.page_shift) - 1) >> p.page_shift;
  for (long long c = first + threadIdx.x; c < p.width; c += 256) {
    int32_t *cell = p.table + row * static_cast<long long>(p.width) + c;
    const int page = *cell < 0 ? -1 : atomicExch(cell, -1);
    if (page >= 0) {
      if (page < p.num_pages) atomicSub(&p.refs[page], 1);
      else atomicOr(p.status, kBadPage);
    }
  }
  if (threadIdx.x == 0) atomicMin(&p.lens[row], tokens);
}

// A fork runs as two kernels: the first takes the source rows as they are and counts the new holders, the second gives
// up what the destinations held and writes them. Between them every source has been read, so rows may be both.
__device__ __forceinline__ bool fork_listed_later(const int32_t *dst, int n, int i) {
  // true for the whole block when destination i appears again further on (the last one holds)
  bool later = false;
  const int row = dst[i];
  for (int j = i + 1 + static_cast<int>(threadIdx.x); j < n; j += 256) later |= dst[j] == row;
  return __syncthreads_or(later) != 0;
}

__global__ void __launch_bounds__(256) pages_fork_take_kernel(const __grid_constant__ PagesParams p, const int32_t *dst,
                                                              const int32_t *src, int n) {
  grid_dep_wait();
  const int i = blockIdx.x;
  const int to = dst[i], from = src[i];
  int32_t *keep = p.ws + kPlanPairs + static_cast<long long>(i) * (p.width + 1);
  const bool bad = to < 0 || to >= p.rows || from < 0 || from >= p.rows;
  if (bad || fork_listed_later(dst, n, i)) {
    if (threadIdx.x == 0) {
      keep[p.width] = -1;
      if (bad) atomicOr(p.status, kBadRow);
    }
    return;
  }
  for (int c = threadIdx.x; c < p.width; c += 256) {
    const int page = p.table[static_cast<long long>(from) * p.width + c];
    keep[c] = page;
    if (page >= 0) {
      if (page < p.num_pages) atomicAdd(&p.refs[page], 1);
      else atomicOr(p.status, kBadPage);
    }
  }
  if (threadIdx.x == 0) keep[p.width] = p.lens[from];
}

__global__ void __launch_bounds__(256) pages_fork_put_kernel(const __grid_constant__ PagesParams p, const int32_t *dst) {
  grid_dep_wait();
  const int32_t *keep = p.ws + kPlanPairs + static_cast<long long>(blockIdx.x) * (p.width + 1);
  const int len = keep[p.width];
  if (len < 0) return;
  const int row = dst[blockIdx.x];
  for (int c = threadIdx.x; c < p.width; c += 256) {
    int32_t *cell = p.table + static_cast<long long>(row) * p.width + c;
    const int old = *cell;
    if (old >= 0 && old < p.num_pages) atomicSub(&p.refs[old], 1);
    *cell = keep[c];
  }
  if (threadIdx.x == 0) p.lens[row] = len;
}

// Exclusive prefix sum of one value per thread over a block of 1024 threads; `total` for everyone.
__device__ __forceinline__ int block_scan(int x, int *total, int *warp_sums) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int sum = x;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, sum, d);
    if (lane >= d) sum += y;
  }
  if (lane == 31) warp_sums[warp] = sum;
  __syncthreads();
  int w = warp_sums[lane];
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, w, d);
    if (lane >= d) w += y;
  }
  *total = __shfl_sync(0xffffffffu, w, 31);
  const int before = warp ? __shfl_sync(0xffffffffu, w, warp - 1) : 0;
  __syncthreads();  // the sums may be written again
  return before + sum - x;
}

__device__ __forceinline__ void load_refs(const PagesParams &p, int first, int (&r)[16]) {
#pragma unroll
  for (int i = 0; i < 16; i += 4) {
    if (first + i + 4 <= p.num_pages) {
      const int4 q = *reinterpret_cast<const int4 *>(p.refs + first + i);
      r[i] = q.x; r[i + 1] = q.y; r[i + 2] = q.z; r[i + 3] = q.w;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) r[i + e] = first + i + e < p.num_pages ? p.refs[first + i + e] : INT32_MIN;
    }
  }
}

// A reserve is done for all of its rows or for none. step_lens (may be NULL) carries that to the kernels behind it, which are
// launched without the host knowing: the rows' new lengths, or kRefused. Without it an append behind a reserve that found no
// free pages would take the last old tokens' places, in pages that other rows may hold as well.
constexpr int32_t kRefused = TX_PAGES_REFUSED;

// Dynamic shared memory: end[n], last[n] (last page of the row if it is partly filled, else -1), row[n], len[n],
// seen[rows / 32]. What takes the time is loads that wait for one another, so each is made once and the first step's
// reference counts are loaded before anything else.
constexpr int kFreshShared = 2048;  // free pages that are handed on in shared memory

__global__ void __launch_bounds__(kPlanThreads) pages_reserve_plan_kernel(const __grid_constant__ PagesParams p,
                                                                          const int32_t *rows, const int32_t *counts, int n,
                                                                          int32_t *step_lens) {
  extern __shared__ int32_t plan_smem[];
  __shared__ int warp_sums[32], s_fresh[kFreshShared];
  __shared__ int s_bad, s_pairs;
  int32_t *end = plan_smem, *last = plan_smem + n, *s_row = plan_smem + 2 * n, *s_len = plan_smem + 3 * n;
  uint32_t *seen = reinterpret_cast<uint32_t *>(plan_smem + 4 * n);
  int32_t *pairs = p.ws + kPlanPairs, *fresh = pairs + 2 * n;
  const int tid = threadIdx.x;
  const int slots = 1 << p.page_shift;
  if (tid == 0) s_bad = 0, s_pairs = 0;
  for (int i = tid; i < (p.rows + 31) / 32; i += kPlanThreads) seen[i] = 0;
  grid_dep_wait();
  int r0[16];
  load_refs(p, tid * 16, r0);
  __syncthreads();
  for (int i = tid; i < n; i += kPlanThreads) {
    const int row = rows[i], count = counts[i];
    int need = 0, page = -1, len_now = 0;
    uint32_t bad = 0;
    if (row < 0 || row >= p.rows || count < 0 || (atomicOr(&seen[row >> 5], 1u << (row & 31)) >> (row & 31) & 1u)) {
      bad = kBadRow;
    } else {
      len_now = p.lens[row];
      const long long len = max(len_now, 0), want = (len + count + slots - 1) >> p.page_shift;
      const long long have = (len + slots - 1) >> p.page_shift;
      if (len_now < 0) {
        bad = kBadLength;
      } else if (want > p.width || len + count > INT32_MAX) {
        bad = kNoRoomInRow;
      } else {
        need = static_cast<int>(want - have);
        if (count > 0 && (len & (slots - 1))) {
          page = p.table[static_cast<long long>(row) * p.width + have - 1];
          if (page < 0 || page >= p.num_pages) bad = kBadPage, page = -1;
        }
      }
    }
    if (bad) atomicOr(&s_bad, static_cast<int>(bad));
    end[i] = need;
    last[i] = page;
    s_row[i] = row;
    s_len[i] = len_now;
  }
  __syncthreads();
  // a shared last page is copied by its holder i if somebody holds it after those listed before i have left it
  const int per = (n + kPlanThreads - 1) / kPlanThreads;  // consecutive rows of a thread
  int mine = 0;
  uint32_t copies = 0;  // bit e: row tid * per + e copies its last page (per <= 4)
  for (int e = 0; e < per; ++e) {
    const int i = tid * per + e;
    if (i >= n) break;
    if (last[i] >= 0) {
      const int holders = p.refs[last[i]];
      if (holders > 1) {
        int earlier = 0;
        for (int j = 0; j < i; ++j) earlier += last[j] == last[i];
        if (holders - earlier > 1) copies |= 1u << e;
      }
    }
    mine += end[i] + static_cast<int>(copies >> e & 1u);
  }
  int need_all;
  int start = block_scan(mine, &need_all, warp_sums);
  for (int e = 0; e < per; ++e) {
    const int i = tid * per + e;
    if (i >= n) break;
    const int copy = static_cast<int>(copies >> e & 1u);
    start += end[i] + copy;
    end[i] = start;
    if (!copy) last[i] = -1;  // from here on: the page to copy
  }
  // the first need_all free pages, ascending
  const bool shared = need_all <= kFreshShared;
  int found = 0;
  for (int base = 0; base < p.num_pages && found < need_all; base += kPlanThreads * 16) {
    if (base) load_refs(p, base + tid * 16, r0);
    int zeros = 0, total;
#pragma unroll
    for (int i = 0; i < 16; ++i) zeros += r0[i] == 0;
    int at = found + block_scan(zeros, &total, warp_sums);
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (r0[i] == 0) {
        if (at < need_all) (shared ? s_fresh : fresh)[at] = base + tid * 16 + i;
        ++at;
      }
    found += total;
  }
  __syncthreads();
  if (s_bad || found < need_all) {
    if (tid == 0) {
      atomicOr(p.status, static_cast<uint32_t>(s_bad) | (found < need_all ? kNoFreePages : 0u));
      p.ws[0] = 0;
    }
    if (step_lens)
      for (int i = tid; i < n; i += kPlanThreads) step_lens[i] = kRefused;
    return;
  }
  for (int r = tid; r < need_all; r += kPlanThreads) {
    int lo = 0, hi = n - 1;  // the first row whose end is past r
    while (lo < hi) {
      const int mid = (lo + hi) / 2;
      if (end[mid] > r) hi = mid;
      else lo = mid + 1;
    }
    const int page = (shared ? s_fresh : fresh)[r];
    const int off = r - (lo ? end[lo - 1] : 0), copy = last[lo] >= 0;
    const int have = static_cast<int>((static_cast<long long>(s_len[lo]) + slots - 1) >> p.page_shift);
    p.table[static_cast<long long>(s_row[lo]) * p.width + have + off - copy] = page;
    p.refs[page] = 1;
    if (copy && off == 0) {
      const int slot = atomicAdd(&s_pairs, 1);
      pairs[2 * slot] = last[lo];
      pairs[2 * slot + 1] = page;
      atomicSub(&p.refs[last[lo]], 1);
    }
  }
  for (int i = tid; i < n; i += kPlanThreads) {
    const int len = s_len[i] + counts[i];
    p.lens[s_row[i]] = len;
    if (step_lens) step_lens[i] = len;
  }
  __syncthreads();
  if (tid == 0) p.ws[0] = s_pairs;
}

// Copies pairs[0 .. ws[0]) in every layer of both pools. A piece is 16 KB (4 vectors a thread in flight) of one page of
// one pool; with about 8 blocks an SM that keeps 128 KB on their way per SM.
constexpr int kCopyVecs = 4;
__device__ __forceinline__ void copy_pages(const PagesParams &p, const int32_t *pairs, long long count) {
  const long long pieces = (p.page_vecs + 256 * kCopyVecs - 1) / (256 * kCopyVecs);
  const long long all = count * p.layers * 2 * pieces;
  for (long long w = blockIdx.x; w < all; w += gridDim.x) {
    const long long piece = w % pieces, rest = w / pieces;
    const int which = static_cast<int>(rest & 1), layer = static_cast<int>((rest >> 1) % p.layers);
    const long long pair = (rest >> 1) / p.layers;
    const long long src = pairs[2 * pair], dst = pairs[2 * pair + 1];
    uint4 *pool = (which ? p.v : p.k) + static_cast<long long>(layer) * p.num_pages * p.page_vecs;
    const uint4 *from = pool + src * p.page_vecs;
    uint4 *to = pool + dst * p.page_vecs;
    const long long at = piece * 256 * kCopyVecs + threadIdx.x;
    uint4 x[kCopyVecs];
#pragma unroll
    for (int i = 0; i < kCopyVecs; ++i)
      if (at + i * 256 < p.page_vecs) x[i] = __ldcs(from + at + i * 256);
#pragma unroll
    for (int i = 0; i < kCopyVecs; ++i)
      if (at + i * 256 < p.page_vecs) __stcs(to + at + i * 256, x[i]);
  }
}

__global__ void __launch_bounds__(256) pages_copy_kernel(const __grid_constant__ PagesParams p) {
  grid_dep_wait();
  copy_pages(p, p.ws + kPlanPairs, p.ws[0]);
}

// Pairs from the host ride in the launch's parameters: no copy to the device that a stream or a graph would have to order.
constexpr int kParamPairs = 1024;
struct ParamPairs {
  int32_t pair[2 * kParamPairs];
};
__global__ void __launch_bounds__(256) pages_copy_listed_kernel(const __grid_constant__ PagesParams p,
                                                                const __grid_constant__ ParamPairs pairs, int count) {
  grid_dep_wait();
  copy_pages(p, pairs.pair, count);
}

// With U pages in use, hole number i below U takes the used page number i at or above U: the fewest pages that can move,
// and no page is both source and destination. Workspace: pairs, then where every page at or above U went.
__global__ void __launch_bounds__(kPlanThreads) pages_compact_plan_kernel(const __grid_constant__ PagesParams p) {
  __shared__ int warp_sums[32];
  const int tid = threadIdx.x;
  int32_t *pairs = p.ws + kPlanPairs, *went = pairs + p.num_pages + 1;
  constexpr int kStep = kPlanThreads * 16;
  grid_dep_wait();
  int r[16], used = 0;
  for (int base = 0; base < p.num_pages; base += kStep) {
    load_refs(p, base + tid * 16, r);
#pragma unroll
    for (int i = 0; i < 16; ++i) used += r[i] > 0;
  }
  int live;
  block_scan(used, &live, warp_sums);
  int holes = 0, movers = 0;
  for (int base = 0; base < p.num_pages; base += kStep) {
    const int first = base + tid * 16;
    if (p.num_pages > kStep) load_refs(p, first, r);  // a single step's counts are still here
    // holes below the border, used pages above it: a step has at most 16384 of either, so both fit one sum
    int mine = 0, total;
#pragma unroll
    for (int i = 0; i < 16; ++i) mine += first + i < live ? (r[i] == 0) : (r[i] > 0) << 16;
    const int before = block_scan(mine, &total, warp_sums);
    int hole = holes + (before & 0xffff), mover = movers + (before >> 16);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int page = first + i;
      if (page < live) {
        if (r[i] == 0) pairs[2 * hole++ + 1] = page;
      } else if (page < p.num_pages) {
        if (r[i] > 0) pairs[2 * mover++] = page;
        went[page] = page;
      }
    }
    holes += total & 0xffff;
    movers += total >> 16;
  }
  __syncthreads();
  for (int i = tid; i < holes; i += kPlanThreads) {
    const int src = pairs[2 * i], dst = pairs[2 * i + 1];
    went[src] = dst;
    p.refs[dst] = p.refs[src];
    p.refs[src] = 0;
  }
  if (tid == 0) {
    p.ws[0] = holes;
    p.ws[1] = live;
  }
}

__global__ void __launch_bounds__(256) pages_compact_move_kernel(const __grid_constant__ PagesParams p) {
  grid_dep_wait();
  const int32_t *pairs = p.ws + kPlanPairs, *went = pairs + p.num_pages + 1;
  const int count = p.ws[0], live = p.ws[1];
  if (!count) return;
  const long long cells = static_cast<long long>(p.rows) * p.width;
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < cells; i += gridDim.x * 256ll) {
    const int page = p.table[i];
    if (page >= live && page < p.num_pages) p.table[i] = went[page];
  }
  copy_pages(p, pairs, count);
}

}  // namespace txp
