// Paged attention for many rows (chunks of a prompt): bound by the tensor pipe and the softmax's exponentials.
//
// The pipeline is the fused attention forward's (attn_fwd_kernel.cuh: two 128-row sub-tiles with a softmax warpgroup and
// an S and an O accumulator in tensor memory each, a TMA producer warp, a tcgen05.mma warp that serves the sub-tiles in
// turn), made persistent and fed from pages:
//   * a sub-tile's 128 rows are T new tokens x the G query heads of one key head (T = 128 / G, rows left over are zero), so
//     that a group reads its keys and values once; one TMA box {64, G, T} brings them. The two sub-tiles take every second
//     token each, so that under a causal mask both see the same blocks: with the earlier tokens in one and the later ones
//     in the other, the one was done a block before the other in every tile and waited for it from then on (12 prompts of
//     1024 tokens, 12 heads of 64: 84 us, this 76 us)
//   * K and V tiles of 128 tokens arrive as one TMA copy per page and 64 columns, page coordinates from the page table
//   * a CTA walks its share of the work (paged_schedule.cuh), so the barriers' phases run on from tile to tile; a scheduler
//     warp works the next tiles out ahead of the others (each role doing that by itself took over 1 us a tile); a tile of
//     which the CTA has only some blocks leaves fp32 partial results to the joining kernel
//   * rows of V that no row of the tile sees may hold anything: the MMA warp zeroes them in shared memory before the
//     product (0 * NaN must not reach O); scores of keys that a row does not see are replaced, not added to
// Every wait on an mbarrier is bounded in time, as there.
//
// What it takes: 2.2 us a block of 128 keys for 256 rows at D = 128, 1.9 us at D = 64 (the softmax warps issue in 43 % of
// their cycles, two to a scheduler, and the exponentials take half of theirs), 2.5 to 3 us from a tile to the next, 5 us to
// share the work out (few dozen tiles a sequence; see head_cost for many more). A chunk of 2048 tokens over 32768, 32 + 8 heads of 128: 0.98 ms alone, 1.09 PFLOP/s (1.09 ms under the
// power cap). Computing a part of the exponentials by a polynomial on the FMA pipe made it slower (1 of 8: +2 %, 3 of 8:
// +10 %): instructions, not the special-function unit, are what these warps are short of.
#pragma once

#include "paged_row_kernel.cuh"
#include "attn_fwd_kernel.cuh"

namespace txp {

constexpr int kSchedulerWarp = 10;
constexpr int kTileThreads = 352;
constexpr int kItems = 4;  // tiles that the scheduler warp may be ahead

// One tile of a CTA's work, as its roles take it.
struct TileItem {
  int tok0, tokens;    // new tokens [tok0, tok0 + tokens) of the batch
  int pos0;            // position of the first in its sequence
  int head, seq;
  int lo, hi, kv;      // keys that some row sees: [lo, hi); the sequence's keys
  int block, blocks;   // KV blocks [block, block + blocks) of the sequence
  int whole;           // not a part of a cut tile
  int slot;            // of the partial result
  int more;            // 0: the work is done
  int pad[3];
};

struct TileParams {
  CUtensorMap tmap_q, tmap_q2; // {head_dim, heads, tokens}, box {64, G, T} of consecutive tokens and of every second one
  CUtensorMap tmap_k, tmap_v;  // {64 columns, slots, column groups, heads, pages}, box {64, rows, 1, 1, 1}
  Sched s;
  void *out;
  float *m_out;
  long long out_stride[2];
  const int32_t *table;
  long long table_stride;
  int4 *borders;
  float4 *part;
  float2 *ml;
  unsigned long long wait_limit_ns;
  float qk_scale;
  uint32_t idesc_qk, idesc_pv;
  int32_t num_pages, page_shift, box_shift;  // box: rows of one TMA copy, min(page_size, 128)
  int32_t sub_tokens;                        // T
  int32_t heads, head_dim, part_rows;
  int32_t inject_stall;
};

template <int D>
struct TileShape {
  static constexpr uint32_t kTileBytes = 128 * D * 2;
  static constexpr int kAtoms = D / 64;
  static constexpr uint32_t kStages = D == 128 ? 3 : 6;
  static constexpr int kSmem = static_cast<int>(2 * kTileBytes + 2 * txa::kPBytes + kStages * kTileBytes + 1024);
};

struct TileCtl {
  uint64_t q_full, q_empty;
  uint64_t kv_full[6], kv_empty[6];
  uint64_t s_full[2], s_free[2], p_full[2], o_done[2];
  uint64_t item_full[kItems], item_empty[kItems];
  uint64_t drain;
  TileItem item[kItems];
  uint32_t tmem_base;
  volatile uint32_t abort_flag;
};

template <bool kBf16, int D>
__global__ void __launch_bounds__(kTileThreads, 1) paged_tile_kernel(const __grid_constant__ TileParams p) {
  using Shape = TileShape<D>;
  constexpr uint32_t tile_bytes = Shape::kTileBytes;
  constexpr uint32_t kStages = Shape::kStages;
  constexpr int kAtoms = Shape::kAtoms;
  constexpr uint32_t kAtomBytes = txa::kAtomBytes;
  extern __shared__ uint8_t tile_smem_raw[];
  __shared__ SchedSmem sched;
  __shared__ TileCtl ctl;
  const uint32_t q_addr0 = (smem_u32(tile_smem_raw) + 1023u) & ~1023u;
  const uint32_t p_addr0 = q_addr0 + 2 * tile_bytes;
  const uint32_t kv_addr0 = p_addr0 + 2 * txa::kPBytes;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    mbar_init(smem_u32(&ctl.q_full), 1);
    mbar_init(smem_u32(&ctl.q_empty), 1);
    for (uint32_t i = 0; i < kStages; ++i) {
      mbar_init(smem_u32(&ctl.kv_full[i]), 1);
      mbar_init(smem_u32(&ctl.kv_empty[i]), 1);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(smem_u32(&ctl.s_full[t]), 1);
      mbar_init(smem_u32(&ctl.s_free[t]), 128);
      mbar_init(smem_u32(&ctl.p_full[t]), 128);
      mbar_init(smem_u32(&ctl.o_done[t]), 1);
    }
    for (int i = 0; i < kItems; ++i) {
      mbar_init(smem_u32(&ctl.item_full[i]), 1);
      mbar_init(smem_u32(&ctl.item_empty[i]), 10);  // every warp but the scheduler
    }
    mbar_init(smem_u32(&ctl.drain), 1);
    ctl.abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&p.tmap_q);
    tma_prefetch_desc(&p.tmap_q2);
    tma_prefetch_desc(&p.tmap_k);
    tma_prefetch_desc(&p.tmap_v);
  }
  if (warp == txa::kMmaWarp) {
    tmem_alloc(smem_u32(&ctl.tmem_base), txa::kTmemCols);
    tmem_relinquish();
  }
  {  // the rows of Q that no token and head falls on stay zero
    const int rows = p.sub_tokens * p.s.group;
    const int vecs = (128 - rows) * 8;
    for (int i = threadIdx.x; i < 2 * kAtoms * vecs; i += kTileThreads) {
      const int block = i / vecs;
      st_shared_v4(q_addr0 + block * kAtomBytes + rows * 128 + (i - block * vecs) * 16, 0u, 0u, 0u, 0u);
    }
    fence_proxy_async();
  }
  grid_dep_wait();
  tc_fence_before();
  find_work<kTileThreads, true>(p.s, &sched, p.borders, reinterpret_cast<int *>(tile_smem_raw + (p_addr0 - smem_u32(tile_smem_raw))));
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = ctl.tmem_base;

  AbortCtl ac;
  ac.flag = &ctl.abort_flag;
  ac.status = p.s.status;
  ac.limit_ns = p.wait_limit_ns;

  // The next tile, read into registers; false when there is none (or the wait for it ran out).
  TileItem w;
  uint32_t item_count = 0;
  auto next_item = [&]() -> bool {
    const uint32_t i = item_count % kItems;
    if (!warp_mbar_poll(smem_u32(&ctl.item_full[i]), (item_count / kItems) & 1u, ac, kWaitRanOut, lane)) return false;
    w = ctl.item[i];
    __syncwarp();
    if (lane == 0) mbar_arrive(smem_u32(&ctl.item_empty[i]));
    ++item_count;
    return w.more != 0;
  };

  if (warp == kSchedulerWarp) {
    // ------------------------------ scheduler: walks the CTA's work ahead of the others ------------------------------
    Walk walk;
    uint32_t count = 0;
    for (bool more = walk.start(p.s, &sched), last = false; !last; more = more && walk.next(p.s, &sched), ++count) {
      last = !more;
      const uint32_t i = count % kItems;
      if (!warp_mbar_wait(smem_u32(&ctl.item_empty[i]), ((count / kItems) & 1u) ^ 1u, ac, kWaitRanOut, lane)) break;
      if (lane == 0) {
        TileItem x = {};
        if (more) {
          x.tok0 = walk.q.q0 + walk.t.t0;
          x.tokens = walk.t.t1 - walk.t.t0;
          x.pos0 = walk.t.off + walk.t.t0;
          x.head = walk.at.h;
          x.seq = walk.at.b;
          x.lo = walk.t.lo;
          x.hi = walk.t.hi;
          x.kv = walk.q.kv;
          x.block = walk.t.blk0 + walk.from;
          x.blocks = walk.to - walk.from;
          x.whole = walk.whole();
          x.slot = static_cast<int>(walk.slot());
          x.more = 1;
        }
        ctl.item[i] = x;
        mbar_arrive(smem_u32(&ctl.item_full[i]));
      }
      __syncwarp();
    }
  } else if (warp == txa::kProducerWarp) {
    // ------------------------------ TMA producer ------------------------------
    const bool issuer = elect_one();
    uint32_t issued = 0, items = 0;
    bool ok = true;
    const int boxes = 128 >> p.box_shift;  // copies of one atom of a tile
    const uint32_t box_bytes = 128u << p.box_shift;
    while (ok && next_item()) {
      const int nb = w.blocks;
      if (nb <= 0) continue;
      if (!warp_mbar_poll(smem_u32(&ctl.q_empty), (items & 1u) ^ 1u, ac, kWaitRanOut, lane)) {
        ok = false;
        break;
      }
      if (issuer) {
        const uint32_t bar = smem_u32(&ctl.q_full);
        const int active = w.tokens > p.sub_tokens ? 2 : 1;
        mbar_arrive_expect_tx(bar, active * kAtoms * p.sub_tokens * p.s.group * 128);
        for (int t = 0; t < active; ++t)
          for (int a = 0; a < kAtoms; ++a)
            tma_load_3d(q_addr0 + t * tile_bytes + a * kAtomBytes, active == 2 ? &p.tmap_q2 : &p.tmap_q, a * 64,
                        w.head * p.s.group, w.tok0 + t, bar);
      }
      __syncwarp();
      ++items;
      const int32_t *row = p.table + w.seq * p.table_stride;
      const int first_page = w.lo >> p.page_shift, last_page = (w.hi - 1) >> p.page_shift;
      // The page table, 32 entries (one a lane) at a time: the window that K is in, the one before it (V follows one block
      // behind) and the one after it, whose load is under way long before it is needed.
      auto entries = [&](int win) {
        const int at = win * 32 + lane;
        return at >= first_page && at <= last_page ? row[at] : 0;
      };
      int window = (w.block * 128 >> p.page_shift) >> 5;
      int before = 0, cur = entries(window), after = entries(window + 1);
      auto check = [&] {
        if (cur < 0 || cur >= p.num_pages) atomicOr(p.s.status, kBadPage);
      };
      check();
      // All lanes walk the copies of a tile together and one issues them; what a copy needs is at hand before the wait for its
      // slot, because at D = 128 the ring's three slots leave a load little time.
      auto load_tile = [&](int j, bool is_v) {
        const int tok0 = (w.block + j) * 128;
        const int want = (tok0 >> p.page_shift) >> 5;
        if (want > window) {  // by K only, one at a time
          window = want;
          before = cur;
          cur = after;
          after = entries(window + 1);
          check();
        }
        const int ids = want == window ? cur : before;
        const int b0 = max(w.lo - tok0, 0) >> p.box_shift;  // copies [b0, b1) hold keys that are seen
        const int b1 = min((w.hi - tok0 + (1 << p.box_shift) - 1) >> p.box_shift, boxes);
        const uint32_t slot = issued % kStages;
        const uint32_t bar = smem_u32(&ctl.kv_full[slot]);
        const CUtensorMap *map = is_v ? &p.tmap_v : &p.tmap_k;
        const uint32_t dst = kv_addr0 + slot * tile_bytes;
        const uint32_t bytes = (b1 - b0) * kAtoms * box_bytes;
        const int in_mask = (1 << p.page_shift) - 1;
        int id = __shfl_sync(0xffffffffu, ids, ((tok0 + (b0 << p.box_shift)) >> p.page_shift) & 31);
        if (!warp_mbar_poll(smem_u32(&ctl.kv_empty[slot]), ((issued / kStages) & 1u) ^ 1u, ac, kWaitRanOut, lane)) {
          ok = false;
          return;
        }
        if (issuer) mbar_arrive_expect_tx(bar, bytes);
        for (int b = b0;;) {
          const int tok = tok0 + (b << p.box_shift);
          if (issuer) {
#pragma unroll
            for (int a = 0; a < kAtoms; ++a)
              tma_load_5d(dst + a * kAtomBytes + b * box_bytes, map, 0, tok & in_mask, a, w.head, id, bar);
          }
          if (++b >= b1) break;
          id = __shfl_sync(0xffffffffu, ids, ((tok0 + (b << p.box_shift)) >> p.page_shift) & 31);
        }
        __syncwarp();
        ++issued;
      };
      if (p.inject_stall) {
        ok = false;
        break;
      }
      load_tile(0, false);
      for (int j = 0; ok && j < nb; ++j) {
        if (j + 1 < nb) load_tile(j + 1, false);
        if (ok) load_tile(j, true);
      }
    }
    if (!ok || ctl.abort_flag) {  // copies in flight land before the shared memory goes away
      if (lane == 0) {
        const unsigned long long t0 = global_timer_ns();
        if (items)
          while (!mbar_try_wait(smem_u32(&ctl.q_full), (items - 1) & 1u))
            if (global_timer_ns() - t0 > ac.limit_ns) break;
        for (uint32_t i = issued > kStages ? issued - kStages : 0u; i < issued; ++i)
          while (!mbar_try_wait(smem_u32(&ctl.kv_full[i % kStages]), (i / kStages) & 1u))
            if (global_timer_ns() - t0 > 2 * ac.limit_ns) break;
      }
      __syncwarp();
    }
  } else if (warp == txa::kMmaWarp) {
    // ------------------------------ tcgen05.mma issuer ------------------------------
    const bool issuer = elect_one();
    auto desc64 = [](uint32_t hi, uint32_t lo) { return (static_cast<uint64_t>(hi) << 32) | lo; };
    const uint32_t desc_hi = ((1024u >> 4) & 0x3FFFu) | (1u << 14) | (2u << 29);  // SBO 1024, sm_100, SWIZZLE_128B
    const uint32_t kmajor_lbo = 1u << 16;
    const uint32_t v_lbo = ((kAtomBytes >> 4) & 0x3FFFu) << 16;  // between 64-column chunks
    auto lo_of = [](uint32_t addr) { return (addr & 0x3FFFFu) >> 4; };
    uint32_t taken = 0, items = 0, s_count[2] = {0, 0}, p_count[2] = {0, 0};
    bool ok = true;
    auto take = [&]() -> uint32_t {
      const uint32_t slot = taken % kStages;
      if (!warp_mbar_poll(smem_u32(&ctl.kv_full[slot]), (taken / kStages) & 1u, ac, kWaitRanOut, lane)) ok = false;
      ++taken;
      return slot;
    };
    // A V tile: its rows that nobody sees are zeroed before they are multiplied (only a tile's first and last block have any).
    int fix_first = -1, fix_last = -1;
    auto take_v = [&](int j) -> uint32_t {
      const uint32_t slot = take();
      if (ok && (j == fix_first || j == fix_last)) {
        const int tok0 = (w.block + j) * 128;
        const int a = max(w.lo - tok0, 0), b = min(w.hi - tok0, 128);
        for (int at = 0; at < kAtoms; ++at) {
          const uint32_t base = kv_addr0 + slot * tile_bytes + at * kAtomBytes;
          for (int i = lane; i < a * 8; i += 32) st_shared_v4(base + i * 16, 0u, 0u, 0u, 0u);
          for (int i = b * 8 + lane; i < 1024; i += 32) st_shared_v4(base + i * 16, 0u, 0u, 0u, 0u);
        }
        fence_proxy_async();
        __syncwarp();
      }
      return slot;
    };
    auto release = [&](uint32_t slot) {
      if (issuer) tc_commit(smem_u32(&ctl.kv_empty[slot]));
      __syncwarp();
    };
    const uint32_t idesc_qk = p.idesc_qk, idesc_pv = p.idesc_pv;
    auto issue_qk = [&](int t, uint32_t k_slot) {  // S_t = Q_t K^T: D / 16 MMAs of 128 x 128 x 16
      const uint32_t qa = lo_of(q_addr0 + t * tile_bytes) | kmajor_lbo;
      const uint32_t ka = lo_of(kv_addr0 + k_slot * tile_bytes) | kmajor_lbo;
      const uint32_t d_tmem = tmem_base + static_cast<uint32_t>(t) * 128u;
      if (issuer) {
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          const uint32_t step = static_cast<uint32_t>(i >> 2) * (kAtomBytes >> 4) + static_cast<uint32_t>(i & 3) * 2u;
          if (i == 0) umma<false, false>(d_tmem, desc64(desc_hi, qa + step), desc64(desc_hi, ka + step), idesc_qk, 0u);
          else umma_acc<false, false>(d_tmem, desc64(desc_hi, qa + step), desc64(desc_hi, ka + step), idesc_qk);
        }
        tc_commit(smem_u32(&ctl.s_full[t]));
      }
      __syncwarp();
      ++s_count[t];
    };
    auto issue_pv = [&](int t, uint32_t v_slot, bool accumulate) {  // O_t += P_t V: 8 MMAs of 128 x D x 16
      const uint32_t pa = lo_of(p_addr0 + t * txa::kPBytes) | kmajor_lbo;
      const uint32_t va = lo_of(kv_addr0 + v_slot * tile_bytes) | v_lbo;
      const uint32_t d_tmem = tmem_base + 256u + static_cast<uint32_t>(t) * 128u;
      if (issuer) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint32_t pstep = static_cast<uint32_t>(i >> 2) * (kAtomBytes >> 4) + static_cast<uint32_t>(i & 3) * 2u;
          const uint32_t vstep = static_cast<uint32_t>(i) * (16u * 128u >> 4);
          if (i == 0) umma<false, false>(d_tmem, desc64(desc_hi, pa + pstep), desc64(desc_hi, va + vstep), idesc_pv, accumulate ? 1u : 0u);
          else umma_acc<false, false>(d_tmem, desc64(desc_hi, pa + pstep), desc64(desc_hi, va + vstep), idesc_pv);
        }
        tc_commit(smem_u32(&ctl.o_done[t]));
      }
      __syncwarp();
      ++p_count[t];
    };

    while (ok && next_item()) {
      const int nb = w.blocks;
      if (nb <= 0) continue;
      const int n_blk[2] = {nb, w.tokens > p.sub_tokens ? nb : 0};
      fix_first = w.block * 128 < w.lo ? 0 : -1;
      fix_last = (w.block + nb) * 128 > w.hi ? nb - 1 : -1;
      // S of block j: after the accumulator's last S has been read into registers (one tile's last before the next one's first)
      auto next_s = [&](int t, int j, uint32_t k_slot) {
        if (j >= n_blk[t]) return;
        if (s_count[t] > 0 && !warp_mbar_poll(smem_u32(&ctl.s_free[t]), (s_count[t] - 1) & 1u, ac, kWaitRanOut, lane)) {
          ok = false;
          return;
        }
        tc_fence_after();
        issue_qk(t, k_slot);
      };
      auto update_o = [&](int t, int j, uint32_t v_slot) {
        if (j >= n_blk[t]) return;
        if (!warp_mbar_poll(smem_u32(&ctl.p_full[t]), p_count[t] & 1u, ac, kWaitRanOut, lane)) {
          ok = false;
          return;
        }
        tc_fence_after();
        issue_pv(t, v_slot, j > 0);
      };
      if (!warp_mbar_poll(smem_u32(&ctl.q_full), items & 1u, ac, kWaitRanOut, lane)) {
        ok = false;
        break;
      }
      ++items;
      const uint32_t k_slot = take();
      if (!ok) break;
      next_s(0, 0, k_slot);
      if (ok) next_s(1, 0, k_slot);
      if (!ok) break;
      release(k_slot);
      if (nb == 1) {  // Q has been multiplied for the last time
        if (issuer) tc_commit(smem_u32(&ctl.q_empty));
        __syncwarp();
      }
      constexpr bool kVAhead = kStages >= 6;  // see the forward kernel: tiles are taken off the ring one step early
      uint32_t k_ahead = 0, v_ahead = 0;
      if (nb > 1) k_ahead = take();
      if (ok && kVAhead) v_ahead = take_v(0);
      for (int j = 0; ok && j < nb; ++j) {
        const bool have_next = j + 1 < nb;
        const uint32_t kn_slot = k_ahead;
        const uint32_t v_slot = kVAhead ? v_ahead : take_v(j);
        if (!ok) break;
        if (have_next) next_s(0, j + 1, kn_slot);
        if (ok) update_o(0, j, v_slot);
        if (ok && have_next) next_s(1, j + 1, kn_slot);
        if (!ok) break;
        if (have_next) {
          release(kn_slot);
          if (j + 2 == nb) {
            if (issuer) tc_commit(smem_u32(&ctl.q_empty));
            __syncwarp();
          }
        }
        if (j + 2 < nb) {
          k_ahead = take();
          if (!ok) break;
        }
        if (kVAhead && have_next) {
          v_ahead = take_v(j + 1);
          if (!ok) break;
        }
        update_o(1, j, v_slot);
        if (!ok) break;
        release(v_slot);
      }
    }
    // every MMA issued above has completed before tensor and shared memory are given back
    if (issuer) tc_commit(smem_u32(&ctl.drain));
    __syncwarp();
    if (lane == 0) {
      const unsigned long long t0 = global_timer_ns();
      while (!mbar_try_wait(smem_u32(&ctl.drain), 0u)) {
        if (global_timer_ns() - t0 > ac.limit_ns) {
          ctl.abort_flag = 1;
          atomicOr(ac.status, static_cast<uint32_t>(kTimeout));
          break;
        }
      }
    }
    __syncwarp();
  } else {
    // ------------------------------ softmax warpgroups ------------------------------
    constexpr int kElt = kBf16 ? 1 : 0;
    const int t = warp >> 2, quarter = warp & 3;
    const int r = quarter * 32 + lane;  // row of the sub-tile
    const uint32_t lane_base = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16);
    const uint32_t s_tmem = lane_base + static_cast<uint32_t>(t) * 128u;
    const uint32_t o_tmem = lane_base + 256u + static_cast<uint32_t>(t) * 128u;
    const uint32_t p_row = p_addr0 + t * txa::kPBytes + static_cast<uint32_t>((r >> 3) * 1024 + (r & 7) * 128);
    const int row_xor = r & 7;
    const int sub_rows = p.sub_tokens * p.s.group;
    const int tok_in_sub = r / p.s.group, g = r - tok_in_sub * p.s.group;
    uint32_t count = 0;  // blocks of this sub-tile so far
    bool ok = true;
    while (ok && next_item()) {
      const bool both = w.tokens > p.sub_tokens;  // a tile of few tokens is sub-tile 0's alone
      const int n = t == 0 || both ? w.blocks : 0;
      const int rel = both ? t + 2 * tok_in_sub : tok_in_sub;  // this row's token of the tile's
      const bool valid = r < sub_rows && rel < w.tokens && (t == 0 || both);
      const int pos = w.pos0 + rel;
      const int hi_r = !valid ? 0 : p.s.causal ? pos + 1 : w.kv;
      const int lo_r = p.s.window ? pos + 1 - p.s.window : 0;
      // blocks [seen_lo, seen_hi) of the part are seen whole by every row: the loop's unmasked part
      const int seen_hi = ((p.s.causal ? w.pos0 + t + 1 : w.kv) >> 7) - w.block;
      const int seen_lo = ((p.s.window ? max(w.pos0 + w.tokens - p.s.window, 0) : 0) + 127 >> 7) - w.block;
      float m_i = -INFINITY, l_i = 0.f;
      for (int j = 0; j < n; ++j, ++count) {
        if (!warp_mbar_poll(smem_u32(&ctl.s_full[t]), count & 1u, ac, kWaitRanOut, lane)) {
          ok = false;
          break;
        }
        tc_fence_after();
        uint32_t s[128];
        tmem_ld_32x32(s_tmem, *reinterpret_cast<uint32_t(*)[32]>(&s[0]));
        tmem_ld_32x32(s_tmem + 32, *reinterpret_cast<uint32_t(*)[32]>(&s[32]));
        tmem_ld_32x32(s_tmem + 64, *reinterpret_cast<uint32_t(*)[32]>(&s[64]));
        tmem_ld_32x32(s_tmem + 96, *reinterpret_cast<uint32_t(*)[32]>(&s[96]));
        tmem_ld_wait();
        tc_fence_before();
        mbar_arrive(smem_u32(&ctl.s_free[t]));
        if (j >= seen_hi || j < seen_lo) {
          const int col0 = (w.block + j) * 128;
          // by one word of bits for 32 columns: a third of the instructions of two compares for each score, and what this
          // code takes is mostly its own fetching (12 prompts, of 150 to 1500 tokens: 112 us with compares, 102)
          const int hi = hi_r - col0, lo = lo_r - col0;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const int h = min(max(hi - c * 32, 0), 32), l = min(max(lo - c * 32, 0), 32);
            const uint32_t seen = (h == 32 ? 0xffffffffu : (1u << h) - 1u) & (l == 32 ? 0u : 0xffffffffu << l);
#pragma unroll
            for (int i = 0; i < 32; ++i) s[c * 32 + i] = (seen & (1u << i)) ? s[c * 32 + i] : 0xff800000u;  // -inf
          }
        }
        const float mx = txa::row_block_max<false>(s, 0, 0);
        // the reference moves only when the block's maximum passes it by 2^8 (see the forward kernel)
        const float m_cand = fmaxf(m_i, mx * p.qk_scale);
        const float m_next = (m_cand - m_i > txa::kRescaleThreshold) ? m_cand : m_i;
        const float ref = m_next == -INFINITY ? 0.f : m_next;  // a row that has seen nothing yet
        const float alpha = fast_exp2(m_i - ref);
        if (count > 0) {
          // the last O update of this sub-tile has completed: P may be overwritten and O rescaled
          if (!warp_mbar_poll(smem_u32(&ctl.o_done[t]), (count - 1) & 1u, ac, kWaitRanOut, lane)) {
            ok = false;
            break;
          }
          tc_fence_after();
          if (j > 0 && __any_sync(0xffffffffu, alpha != 1.0f)) {
#pragma unroll 1
            for (int c = 0; c < D / 32; ++c) {
              uint32_t o[32];
              tmem_ld_32x32(o_tmem + c * 32, o);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
              tmem_st_32x32(o_tmem + c * 32, o);
            }
            tmem_st_wait();
          }
        }
        // P goes to shared memory rounded to the cache's type, the sum takes the unrounded values (see the row kernel)
        const float sum = txa::row_block_exp_store<false, kElt>(s, p.qk_scale, -ref, 0, 0, p_row, row_xor);
        l_i = l_i * alpha + sum;
        m_i = m_next;
        fence_proxy_async();  // P is read by the tensor core through the async proxy
        tc_fence_before();
        mbar_arrive(smem_u32(&ctl.p_full[t]));
      }
      if (!ok) break;
      // ---- the tile's end ----
      if (n > 0) {
        ok = warp_mbar_poll(smem_u32(&ctl.o_done[t]), (count - 1) & 1u, ac, kWaitRanOut, lane);
        if (!ok) break;
        tc_fence_after();
      }
      if (t == 1 && !both) continue;
      const float inv_l = l_i > 0.f ? 1.0f / l_i : 0.f;
      const bool whole = w.whole != 0;
      const int head = w.head * p.s.group + g, tok = w.tok0 + rel;
      const int part_row = rel * p.s.group + g;
      using T = typename std::conditional<kBf16, __nv_bfloat16, __half>::type;
      const long long o_row = tok * p.out_stride[0] + head * p.out_stride[1];
      const uint32_t stage = p_row - static_cast<uint32_t>((r & 7) * 128 + (r >> 3) * 1024);  // this sub-tile's P
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        uint32_t o[32];
        if (n > 0) {
          tmem_ld_32x32(o_tmem + c * 32, o);
          tmem_ld_wait();
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = 0u;
        }
        if (whole) {
          // rows go out through P's place in shared memory, so that a store instruction covers whole rows
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            uint32_t x[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
              x[i] = txa::pack_pair<kElt>(__uint_as_float(o[q * 8 + 2 * i]) * inv_l, __uint_as_float(o[q * 8 + 2 * i + 1]) * inv_l);
            st_shared_v4(stage + (c >> 1) * kAtomBytes + txa::swz_off(r, (c & 1) * 4 + q), x[0], x[1], x[2], x[3]);
          }
        } else if (valid) {
          float4 *dst = p.part + (static_cast<long long>(w.slot) * (D / 4) + c * 8) * p.part_rows + part_row;
#pragma unroll
          for (int q = 0; q < 8; ++q)
            dst[static_cast<long long>(q) * p.part_rows] =
                make_float4(__uint_as_float(o[4 * q]), __uint_as_float(o[4 * q + 1]), __uint_as_float(o[4 * q + 2]), __uint_as_float(o[4 * q + 3]));
        }
        __syncwarp();
      }
      if (whole) {
        constexpr int kLanes = D / 8;  // lanes of a row, 16 bytes each
        const uint32_t valid_rows = __ballot_sync(0xffffffffu, valid);
#pragma unroll 4
        for (int i = 0; i < kLanes; ++i) {
          const int rr = i * (32 / kLanes) + lane / kLanes, c16 = lane % kLanes;
          const long long at = __shfl_sync(0xffffffffu, o_row, rr);
          uint4 x;
          const uint32_t from = stage + (c16 >> 3) * kAtomBytes + txa::swz_off(quarter * 32 + rr, c16 & 7);
          asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w) : "r"(from) : "memory");
          if ((valid_rows >> rr & 1u) && c16 * 8 < p.head_dim) *reinterpret_cast<uint4 *>(static_cast<T *>(p.out) + at + c16 * 8) = x;
        }
        __syncwarp();
      }
      if (valid) {
        if (!whole) p.ml[static_cast<long long>(w.slot) * p.part_rows + part_row] = make_float2(m_i, l_i);
        else if (p.m_out) p.m_out[static_cast<long long>(tok) * p.heads + head] = l_i > 0.f ? m_i + log2f(l_i) : -INFINITY;
      }
    }
  }

  grid_dep_launch();
  tc_fence_before();
  __syncthreads();
  if (warp == txa::kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem_base, txa::kTmemCols);
  }
}

}  // namespace txp
