// Paged attention for many rows (chunks of a prompt): bound by the tensor pipe and the softmax's exponentials.
//
// The pipeline is the fused attention forward's (attn_fwd_kernel.cuh: two 128-row sub-tiles with a softmax warpgroup and
// an S and an O accumulator in tensor memory each, a TMA producer warp, a tcgen05.mma warp that serves the sub-tiles in
// turn), made persistent and fed from pages:
//   * a sub-tile's 128 rows are T new tokens x the G query heads of one key head (T = 128 / G, rows left over are zero), so
//     that a group reads its keys and values once; one TMA box {64, G, T} brings them
//   * K and V tiles of 128 tokens arrive as one TMA copy per page and 64 columns, page coordinates from the page table
//   * a CTA walks its stretch of the work line (paged_schedule.cuh), so the barriers' phases run on from tile to tile; a
//     tile of which it has only some blocks leaves fp32 partial results to the joining kernel
//   * rows of V that no row of the tile sees may hold anything: the MMA warp zeroes them in shared memory before the
//     product (0 * NaN must not reach O); scores of keys that a row does not see are replaced, not added to
// Every wait on an mbarrier is bounded in time, as there.
#pragma once

#include "paged_row_kernel.cuh"
#include "attn_fwd_kernel.cuh"

namespace txp {

constexpr int kTileThreads = txa::kAttnThreads;

struct TileParams {
  CUtensorMap tmap_q;          // {head_dim, heads, tokens}, box {64, G, T}
  CUtensorMap tmap_k, tmap_v;  // {64 columns, slots, column groups, heads, pages}, box {64, rows, 1, 1, 1}
  Sched s;
  void *out;
  float *m_out;
  long long out_stride[2];
  const int32_t *table;
  long long table_stride;
  int4 *borders;
  float *part;
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
  uint64_t drain;
  uint32_t tmem_base;
  volatile uint32_t abort_flag;
};

// Blocks [0, n) of a walk's part that sub-tile t takes: its rows see fewer keys than the tile's last ones.
__device__ __forceinline__ int sub_blocks(const Sched &s, const Walk &w, int t, int sub_tokens) {
  const int a = w.t.t0 + t * sub_tokens, b = min(a + sub_tokens, w.t.t1);
  if (a >= w.t.t1) return 0;
  const int hi = s.causal ? max(w.t.off + b, 0) : w.q.kv;
  const int end = min(((hi + 127) >> 7) - w.t.blk0, w.to);
  return max(end - w.from, 0);
}

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
    mbar_init(smem_u32(&ctl.drain), 1);
    ctl.abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&p.tmap_q);
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
  const bool work = find_stretch<kTileThreads>(p.s, &sched, p.borders);  // syncs the CTA
  tc_fence_after();
  const uint32_t tmem_base = ctl.tmem_base;

  AbortCtl ac;
  ac.flag = &ctl.abort_flag;
  ac.status = p.s.status;
  ac.limit_ns = p.wait_limit_ns;
  Walk w;

  if (!work) {
    // nothing to do but to give the tensor memory back
  } else if (warp == txa::kProducerWarp) {
    // ------------------------------ TMA producer ------------------------------
    const bool issuer = elect_one();
    uint32_t issued = 0, items = 0;
    bool ok = true;
    const int boxes = 128 >> p.box_shift;  // copies of one atom of a tile
    const uint32_t box_bytes = 128u << p.box_shift;
    for (bool more = w.start(p.s, &sched); more && ok; more = w.next(p.s)) {
      const int nb = w.to - w.from;
      if (nb <= 0) continue;
      if (!warp_mbar_poll(smem_u32(&ctl.q_empty), (items & 1u) ^ 1u, ac, kTimeout, lane)) {
        ok = false;
        break;
      }
      if (issuer) {
        const uint32_t bar = smem_u32(&ctl.q_full);
        const int active = w.t.t1 - w.t.t0 > p.sub_tokens ? 2 : 1;
        mbar_arrive_expect_tx(bar, active * kAtoms * p.sub_tokens * p.s.group * 128);
        for (int t = 0; t < active; ++t)
          for (int a = 0; a < kAtoms; ++a)
            tma_load_3d(q_addr0 + t * tile_bytes + a * kAtomBytes, &p.tmap_q, a * 64, w.at.h * p.s.group,
                        w.q.q0 + w.t.t0 + t * p.sub_tokens, bar);
      }
      __syncwarp();
      ++items;
      const int32_t *row = p.table + w.at.b * p.table_stride;
      const int first_page = w.t.lo >> p.page_shift, last_page = (w.t.hi - 1) >> p.page_shift;
      int window[2] = {-1, -1}, page_reg[2] = {0, 0};  // for K and V: 32 entries of the page table, one a lane
      // lane: box and atom of the tile
      const int box = lane & (boxes - 1), atom = lane >> (7 - p.box_shift);
      auto load_tile = [&](int j, int is_v) {
        const int tok0 = (w.t.blk0 + w.from + j) * 128;
        const int tok = tok0 + (box << p.box_shift), page = tok >> p.page_shift;
        const int want_window = (tok0 >> p.page_shift) >> 5;
        if (window[is_v] != want_window) {
          window[is_v] = want_window;
          const int at = want_window * 32 + lane;
          page_reg[is_v] = at >= first_page && at <= last_page ? row[at] : 0;
          if (page_reg[is_v] < 0 || page_reg[is_v] >= p.num_pages) atomicOr(p.s.status, kBadPage);
        }
        const int id = __shfl_sync(0xffffffffu, page_reg[is_v], page & 31);
        const bool wanted = atom < kAtoms && tok < w.t.hi && tok + (1 << p.box_shift) > w.t.lo;
        const uint32_t count = __popc(__ballot_sync(0xffffffffu, wanted));
        const uint32_t slot = issued % kStages;
        if (!warp_mbar_poll(smem_u32(&ctl.kv_empty[slot]), ((issued / kStages) & 1u) ^ 1u, ac, kTimeout, lane)) {
          ok = false;
          return;
        }
        const uint32_t bar = smem_u32(&ctl.kv_full[slot]);
        if (lane == 0) mbar_arrive_expect_tx(bar, count * box_bytes);
        __syncwarp();
        if (wanted)
          tma_load_5d(kv_addr0 + slot * tile_bytes + atom * kAtomBytes + box * box_bytes, is_v ? &p.tmap_v : &p.tmap_k, 0,
                      tok & ((1 << p.page_shift) - 1), atom, w.at.h, id, bar);
        __syncwarp();
        ++issued;
      };
      if (p.inject_stall) {
        ok = false;
        break;
      }
      load_tile(0, 0);
      for (int j = 0; ok && j < nb; ++j) {
        if (j + 1 < nb) load_tile(j + 1, 0);
        if (ok) load_tile(j, 1);
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
      if (!warp_mbar_poll(smem_u32(&ctl.kv_full[slot]), (taken / kStages) & 1u, ac, kTimeout, lane)) ok = false;
      ++taken;
      return slot;
    };
    // A V tile: its rows that nobody sees are zeroed before they are multiplied.
    auto take_v = [&](int j) -> uint32_t {
      const uint32_t slot = take();
      const int tok0 = (w.t.blk0 + w.from + j) * 128;
      const int a = max(w.t.lo - tok0, 0), b = min(w.t.hi - tok0, 128);
      if (ok && (a > 0 || b < 128)) {
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

    for (bool more = w.start(p.s, &sched); more && ok; more = w.next(p.s)) {
      const int nb = w.to - w.from;
      if (nb <= 0) continue;
      const int n_blk[2] = {sub_blocks(p.s, w, 0, p.sub_tokens), sub_blocks(p.s, w, 1, p.sub_tokens)};
      // S of block j: after the accumulator's last S has been read into registers (one tile's last before the next one's first)
      auto next_s = [&](int t, int j, uint32_t k_slot) {
        if (j >= n_blk[t]) return;
        if (s_count[t] > 0 && !warp_mbar_poll(smem_u32(&ctl.s_free[t]), (s_count[t] - 1) & 1u, ac, kTimeout, lane)) {
          ok = false;
          return;
        }
        tc_fence_after();
        issue_qk(t, k_slot);
      };
      auto update_o = [&](int t, int j, uint32_t v_slot) {
        if (j >= n_blk[t]) return;
        if (!warp_mbar_poll(smem_u32(&ctl.p_full[t]), p_count[t] & 1u, ac, kTimeout, lane)) {
          ok = false;
          return;
        }
        tc_fence_after();
        issue_pv(t, v_slot, j > 0);
      };
      if (!warp_mbar_poll(smem_u32(&ctl.q_full), items & 1u, ac, kTimeout, lane)) {
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
    for (bool more = w.start(p.s, &sched); more && ok; more = w.next(p.s)) {
      const int n = sub_blocks(p.s, w, t, p.sub_tokens);
      const int first = w.t.t0 + t * p.sub_tokens;  // the sub-tile's tokens: [first, last)
      const int last = min(first + p.sub_tokens, w.t.t1);
      const int tok = first + tok_in_sub;
      const bool valid = r < sub_rows && tok < last;
      const int pos = w.t.off + tok;
      const int hi_r = !valid ? 0 : p.s.causal ? pos + 1 : w.q.kv;
      const int lo_r = p.s.window ? pos + 1 - p.s.window : 0;
      // blocks inside [inner_lo, inner_hi) are seen whole by every row: the loop's unmasked part
      const int inner_hi = p.s.causal ? w.t.off + first + 1 : w.q.kv;
      const int inner_lo = p.s.window ? w.t.off + last - p.s.window : 0;
      float m_i = -INFINITY, l_i = 0.f;
      for (int j = 0; j < n; ++j, ++count) {
        if (!warp_mbar_poll(smem_u32(&ctl.s_full[t]), count & 1u, ac, kTimeout, lane)) {
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
        const int col0 = (w.t.blk0 + w.from + j) * 128;
        if (col0 + 128 > inner_hi || col0 < inner_lo) {
#pragma unroll
          for (int i = 0; i < 128; ++i) s[i] = col0 + i < hi_r && col0 + i >= lo_r ? s[i] : 0xff800000u;  // -inf
        }
        const float mx = txa::row_block_max<false>(s, 0, 0);
        // the reference moves only when the block's maximum passes it by 2^8 (see the forward kernel)
        const float m_cand = fmaxf(m_i, mx * p.qk_scale);
        const float m_next = (m_cand - m_i > txa::kRescaleThreshold) ? m_cand : m_i;
        const float ref = m_next == -INFINITY ? 0.f : m_next;  // a row that has seen nothing yet
        const float alpha = fast_exp2(m_i - ref);
        if (count > 0) {
          // the last O update of this sub-tile has completed: P may be overwritten and O rescaled
          if (!warp_mbar_poll(smem_u32(&ctl.o_done[t]), (count - 1) & 1u, ac, kTimeout, lane)) {
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
        ok = warp_mbar_poll(smem_u32(&ctl.o_done[t]), (count - 1) & 1u, ac, kTimeout, lane);
        if (!ok) break;
        tc_fence_after();
      }
      if (first >= w.t.t1) continue;
      const float inv_l = l_i > 0.f ? 1.0f / l_i : 0.f;
      const bool whole = w.whole();
      const int head = w.at.h * p.s.group + g;
      const long long part_row = (static_cast<long long>(blockIdx.x) * 2 + w.slot()) * p.part_rows + t * sub_rows + r;
      using T = typename std::conditional<kBf16, __nv_bfloat16, __half>::type;
      T *o_row = static_cast<T *>(p.out) + (w.q.q0 + tok) * p.out_stride[0] + head * p.out_stride[1];
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
        if (valid && whole) {
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            uint32_t x[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
              x[i] = txa::pack_pair<kElt>(__uint_as_float(o[q * 8 + 2 * i]) * inv_l, __uint_as_float(o[q * 8 + 2 * i + 1]) * inv_l);
            if (c * 32 + q * 8 < p.head_dim) *reinterpret_cast<uint4 *>(o_row + c * 32 + q * 8) = make_uint4(x[0], x[1], x[2], x[3]);
          }
        } else if (valid) {
          float *dst = p.part + part_row * D + c * 32;
#pragma unroll
          for (int q = 0; q < 8; ++q)
            *reinterpret_cast<uint4 *>(dst + q * 4) = make_uint4(o[4 * q], o[4 * q + 1], o[4 * q + 2], o[4 * q + 3]);
        }
        __syncwarp();
      }
      if (valid) {
        if (!whole) p.ml[part_row] = make_float2(m_i, l_i);
        else if (p.m_out) p.m_out[static_cast<long long>(w.q.q0 + tok) * p.heads + head] = l_i > 0.f ? m_i + log2f(l_i) : -INFINITY;
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
