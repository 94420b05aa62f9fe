// Paged attention for few rows (single tokens, drafted tokens): bound by reading K and V once from HBM.
//
// A CTA walks its stretch of the work line (paged_schedule.cuh). One warp walks it and streams KV blocks of BS tokens through a ring in
// shared memory by TMA, one copy per page and tensor (page coordinate from the page table, so a bad entry reads zeros); the
// other warps are MT groups of 16 rows x KS shares of a block's tokens. Each keeps a running maximum, a running sum and its
// output in registers through the whole tile (one pass over the keys), on m16n8k16 tensor instructions: at 16 rows per
// 32 KB of K and V these need a tenth of the time the bytes take, so 128-row tcgen05 tiles would only add empty rows and
// their softmax. At a tile's end the KS warps of a row group are joined through a ring slot that the producer leaves empty.
//
// The share of a tile that HBM has to deliver is all there is to wait for: the ring holds 96 KB a CTA, two CTAs an SM
// (at 16 rows), which covers HBM's latency several times. 64 ragged sequences of up to 8192 tokens, 32 + 8 heads of 128:
// 212 us, 6.4 TB/s. At 32 rows a warp's own chain (products, exponentials, products) is as long as its share of the bytes
// takes, about 0.9 us for 16 tokens, so a warp takes 32 tokens at a time there (8 drafted tokens over up to 4100: 51 us with
// 16, 47 with 32). Short calls are latency: 2.2 us to share the work out, 2 to 3 us to the first block, 2.5 us to join.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "paged_schedule.cuh"

namespace txp {

constexpr int kRowItems = 4;   // tiles that the producer may be ahead

// One tile of a CTA's work, as the consumers take it.
struct RowItem {
  int tok0, tokens;   // new tokens [tok0, tok0 + tokens) of the batch
  int pos0;           // position of the first in its sequence
  int head;
  int lo, hi, kv;     // keys that some row sees: [lo, hi); the sequence's keys
  int first_key;      // of the first block of this part
  int blocks;
  int whole, slot;    // not a part of a cut tile; else the place of the partial result
  int more;           // 0: the work is done
};

struct RowParams {
  CUtensorMap tmap_k, tmap_v;  // {64 columns, slots, column groups, heads, pages}
  Sched s;
  const void *q;
  void *out;
  float *m_out;
  long long q_stride[2], out_stride[2];
  const int32_t *table;
  long long table_stride;
  int4 *borders;
  float4 *part;
  float2 *ml;
  unsigned long long wait_limit_ns;
  float qk_scale;  // sm_scale * log2(e)
  int32_t num_pages, page_shift, box_shift;  // box: rows of one TMA copy, min(page_size, BS)
  int32_t heads, head_dim;
  int32_t inject_stall;
};

template <bool kBf16>
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (kBf16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldmatrix_x4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <bool kBf16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if (kBf16) {
    __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t *>(&h);
  }
  __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<uint32_t *>(&h);
}
__device__ __forceinline__ void tma_load_5d(uint32_t dst, const CUtensorMap *m, int x, int y, int z, int w, int v, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(m)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(v), "r"(bar)
      : "memory");
}

// Whether it holds for any of kThreads threads, which meet at named barrier 1.
template <int kThreads>
__device__ __forceinline__ bool any_of(bool x) {
  uint32_t r;
  asm volatile(
      "{\n"
      ".reg .pred p, q;\n"
      "setp.ne.u32 p, %1, 0;\n"
      "bar.red.or.pred q, 1, %2, p;\n"
      "selp.u32 %0, 1, 0, q;\n"
      "}\n"
      : "=r"(r)
      : "r"(x ? 1u : 0u), "n"(kThreads)
      : "memory");
  return r != 0;
}

template <int D, int BS, int kStages>
constexpr int row_smem_bytes() { return kStages * 2 * BS * D * 2 + 1024; }

template <bool kBf16, int D, int BS, int MT, int KS, int kStages, int kBlocksPerSm>
__global__ void __launch_bounds__((MT * KS + 1) * 32, kBlocksPerSm) paged_row_kernel(const __grid_constant__ RowParams p) {
  constexpr int kConsumers = MT * KS;
  constexpr int kThreads = (kConsumers + 1) * 32;
  constexpr int kTok = BS / KS;             // tokens of a block that one warp takes
  constexpr int kSlabs = kTok / 16;
  constexpr int kGroups = D / 64;           // column groups of 128 bytes
  constexpr uint32_t kTensorBytes = BS * D * 2;
  constexpr uint32_t kStageBytes = 2 * kTensorBytes;
  constexpr int kRounds = MT * KS * 16 / BS;  // of the join: a ring slot holds BS rows of D fp32 values
  constexpr int kJoinCols = D / kRounds;
  static_assert(kJoinCols >= 32, "a round has whole groups of columns");

  extern __shared__ uint8_t row_smem_raw[];
  __shared__ SchedSmem sched;
  __shared__ uint64_t full[kStages], empty[kStages], item_full[kRowItems], item_empty[kRowItems];
  __shared__ RowItem items[kRowItems];
  __shared__ float2 s_ml[KS][MT * 16];
  __shared__ uint32_t abort_flag;
  const uint32_t ring = (smem_u32(row_smem_raw) + 1023u) & ~1023u;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(smem_u32(&full[i]), 1);
      mbar_init(smem_u32(&empty[i]), kConsumers);
    }
    for (int i = 0; i < kRowItems; ++i) {
      mbar_init(smem_u32(&item_full[i]), 1);
      mbar_init(smem_u32(&item_empty[i]), kConsumers);
    }
    abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&p.tmap_k);
    tma_prefetch_desc(&p.tmap_v);
  }
  grid_dep_wait();
  find_work<kThreads, false>(p.s, &sched, p.borders, nullptr);
  __syncthreads();

  AbortCtl ac;
  ac.flag = &abort_flag;
  ac.status = p.s.status;
  ac.limit_ns = p.wait_limit_ns;

  if (warp == kConsumers) {
    // ------------------------------ producer: walks the work, hands the tiles on, loads their blocks ------------------------------
    Walk w;
    uint32_t issued = 0, count = 0;
    bool ok = true;
    const int boxes = BS >> p.box_shift;           // copies of a tensor per block
    const uint32_t box_bytes = (128u << p.box_shift) * kGroups;
    auto hand_on = [&](bool more) {
      const uint32_t i = count % kRowItems;
      if (!warp_mbar_poll(smem_u32(&item_empty[i]), ((count / kRowItems) & 1u) ^ 1u, ac, kWaitRanOut, lane)) {
        ok = false;
        return;
      }
      if (lane == 0) {
        RowItem x = {};
        if (more) {
          x.tok0 = w.q.q0 + w.t.t0;
          x.tokens = w.t.t1 - w.t.t0;
          x.pos0 = w.t.off + w.t.t0;
          x.head = w.at.h;
          x.lo = w.t.lo;
          x.hi = w.t.hi;
          x.kv = w.q.kv;
          x.first_key = (w.t.blk0 + w.from) * BS;
          x.blocks = w.to - w.from;
          x.whole = w.whole();
          x.slot = static_cast<int>(w.slot());
          x.more = 1;
        }
        items[i] = x;
        mbar_arrive(smem_u32(&item_full[i]));
      }
      __syncwarp();
      ++count;
    };
    for (bool more = w.start(p.s, &sched); more && ok; more = w.next(p.s, &sched)) {
      hand_on(true);
      const int32_t *row = p.table + w.at.b * p.table_stride;
      const int first_page = w.t.lo >> p.page_shift, last_page = (w.t.hi - 1) >> p.page_shift;
      int window = -1, page_reg = 0;  // 32 entries of the page table, one a lane
      for (int j = w.from; j < w.to && ok; ++j) {
        const uint32_t slot = issued % kStages, pass = issued / kStages;
        const int tok0 = (w.t.blk0 + j) * BS;
        // lane: tensor (K first) and box
        const int box = lane < boxes ? lane : lane - boxes;
        const int tok = tok0 + (box << p.box_shift), page = tok >> p.page_shift;
        if (window != (tok0 >> p.page_shift) >> 5) {
          window = (tok0 >> p.page_shift) >> 5;
          const int at = window * 32 + lane;
          page_reg = at >= first_page && at <= last_page ? row[at] : 0;
          if (page_reg < 0 || page_reg >= p.num_pages) atomicOr(p.s.status, kBadPage);
        }
        const int id = __shfl_sync(0xffffffffu, page_reg, page & 31);
        const bool wanted = lane < 2 * boxes && tok < w.t.hi && tok + (1 << p.box_shift) > w.t.lo;
        const uint32_t count = __popc(__ballot_sync(0xffffffffu, wanted));
        if (!warp_mbar_poll(smem_u32(&empty[slot]), (pass & 1u) ^ 1u, ac, kWaitRanOut, lane)) {
          ok = false;
          break;
        }
        const uint32_t bar = smem_u32(&full[slot]);
        if (lane == 0) mbar_arrive_expect_tx(bar, count * box_bytes);
        __syncwarp();
        if (wanted) {
          const uint32_t dst = ring + slot * kStageBytes + (lane < boxes ? 0u : kTensorBytes) + box * box_bytes;
          tma_load_5d(dst, lane < boxes ? &p.tmap_k : &p.tmap_v, 0, tok & ((1 << p.page_shift) - 1), 0, w.at.h, id, bar);
        }
        __syncwarp();
        ++issued;
        if (p.inject_stall) ok = false;
      }
      if (ok && w.to > w.from) {  // the slot that the tile's warps are joined in
        const uint32_t slot = issued % kStages, pass = issued / kStages;
        if (!warp_mbar_poll(smem_u32(&empty[slot]), (pass & 1u) ^ 1u, ac, kWaitRanOut, lane)) ok = false;
        else if (lane == 0) mbar_arrive(smem_u32(&full[slot]));
        __syncwarp();
        ++issued;
      }
    }
    if (ok) hand_on(false);
    if (!ok) {  // copies in flight land before the shared memory goes away
      if (lane == 0)
        for (uint32_t i = issued > kStages ? issued - kStages : 0u; i < issued; ++i) {
          const unsigned long long t0 = global_timer_ns();
          while (!mbar_try_wait(smem_u32(&full[i % kStages]), (i / kStages) & 1u))
            if (global_timer_ns() - t0 > ac.limit_ns) break;
        }
      __syncwarp();
    }
  } else {
    // ------------------------------ consumers ------------------------------
    using T = typename std::conditional<kBf16, __nv_bfloat16, __half>::type;
    const int mt = warp / KS, ks = warp % KS;
    const int g4 = lane >> 2, l4 = lane & 3;
    uint32_t taken = 0;
    // After a wait that ran out a warp goes through the tile's end without waiting, so that every warp still meets the
    // others at the barriers below; what it computes then is reported as undefined.
    bool ok = true;
    auto take = [&]() -> uint32_t {
      const uint32_t slot = taken % kStages;
      if (ok && !warp_mbar_poll(smem_u32(&full[slot]), (taken / kStages) & 1u, ac, kWaitRanOut, lane)) ok = false;
      ++taken;
      return slot;
    };
    auto give = [&](uint32_t slot) {
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&empty[slot]));
    };
    // this warp's tokens of a block: where their rows start in a tensor's part of a stage
    const uint32_t group_bytes = 128u << p.box_shift;  // one column group of one copy
    uint32_t slab[kSlabs];
#pragma unroll
    for (int i = 0; i < kSlabs; ++i) {
      const int t = ks * kTok + i * 16;
      slab[i] = static_cast<uint32_t>((t >> p.box_shift)) * group_bytes * kGroups +
                static_cast<uint32_t>(t & ((1 << p.box_shift) - 1)) * 128u;
    }
    const uint32_t x7 = lane & 7;
    const uint32_t k_row = ((lane >> 4) * 8 + x7) * 128u, k_chunk = (lane >> 3) & 1;
    const uint32_t v_row = (((lane >> 3) & 1) * 8 + x7) * 128u, v_chunk = lane >> 4;

    for (uint32_t count = 0;; ++count) {
      const uint32_t item = count % kRowItems;
      if (ok && !warp_mbar_poll(smem_u32(&item_full[item]), (count / kRowItems) & 1u, ac, kWaitRanOut, lane)) ok = false;
      if (any_of<kConsumers * 32>(!ok)) break;  // all of them leave, or none
      const RowItem w = items[item];
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&item_empty[item]));
      if (!w.more) break;
      const int rows = w.tokens * p.s.group;
      // ---- Q: the A fragments of this warp's 16 rows, straight from memory ----
      uint32_t qf[D / 16][4];
      int hi_r[2], lo_r[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = mt * 16 + g4 + e * 8;
        const int tok = r / p.s.group;
        const int head = w.head * p.s.group + r % p.s.group;
        const bool valid = r < rows;
        const T *src = static_cast<const T *>(p.q) + (w.tok0 + tok) * p.q_stride[0] + head * p.q_stride[1] + l4 * 2;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const bool in = valid && (D > 64 || kk * 16 < p.head_dim);
          qf[kk][e] = in ? *reinterpret_cast<const uint32_t *>(src + kk * 16) : 0u;
          qf[kk][2 + e] = in ? *reinterpret_cast<const uint32_t *>(src + kk * 16 + 8) : 0u;
        }
        const int pos = w.pos0 + tok;
        hi_r[e] = !valid ? 0 : p.s.causal ? pos + 1 : w.kv;
        lo_r[e] = p.s.window ? max(pos + 1 - p.s.window, 0) : 0;
      }
      // blocks outside [inner_lo, inner_hi) have keys that some row of the tile does not see
      const int inner_hi = p.s.causal ? w.pos0 + 1 : w.kv;
      const int inner_lo = p.s.window ? w.pos0 + w.tokens - p.s.window : 0;
      float o[D / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
      for (int i = 0; i < D / 8; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i][e] = 0.f;

      for (int j = 0; j < w.blocks; ++j) {
        const uint32_t slot = take();
        const uint32_t k_base = ring + slot * kStageBytes, v_base = k_base + kTensorBytes;
        const int blk_tok = w.first_key + j * BS;
        const bool edge = blk_tok + BS > inner_hi || blk_tok < inner_lo;
        // ---- S = Q K^T ----
        float s[kSlabs * 2][4];
#pragma unroll
        for (int i = 0; i < kSlabs * 2; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[i][e] = 0.f;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
          for (int i = 0; i < kSlabs; ++i) {
            uint32_t b[4];
            ldmatrix_x4(k_base + slab[i] + (kk >> 2) * group_bytes + k_row + ((((kk & 3) * 2 + k_chunk) ^ x7) << 4), b);
            mma_16816<kBf16>(s[2 * i], qf[kk], b[0], b[1]);
            mma_16816<kBf16>(s[2 * i + 1], qf[kk], b[2], b[3]);
          }
        if (edge) {
          // V at keys that no row of the tile sees may be anything, NaN included: 0 * NaN must not reach O. (Warps of other
          // rows write the same zeros.)
#pragma unroll
          for (int i = 0; i < kSlabs; ++i) {
            const int key = blk_tok + ks * kTok + i * 16;
            if (key >= w.lo && key + 16 <= w.hi) continue;
            for (int x = lane; x < 16 * 8 * kGroups; x += 32) {
              const int tok = (x >> 3) & 15;
              if (key + tok < w.lo || key + tok >= w.hi)
                st_shared_v4(v_base + slab[i] + (x >> 7) * group_bytes + tok * 128u + (x & 7) * 16u, 0u, 0u, 0u, 0u);
            }
          }
          fence_proxy_async();  // TMA writes the slot next
          __syncwarp();
          // scores of keys that the row does not see
#pragma unroll
          for (int i = 0; i < kSlabs * 2; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int key = blk_tok + ks * kTok + i * 8 + l4 * 2 + (e & 1);
              s[i][e] = key < hi_r[e >> 1] && key >= lo_r[e >> 1] ? s[i][e] : -INFINITY;
            }
        }
        // ---- softmax, in log2 units, against the running maximum ----
        float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < kSlabs * 2; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) mx[e >> 1] = fmaxf(mx[e >> 1], s[i][e]);
        float ref[2];
        bool grow = false;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 1));
          mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 2)) * p.qk_scale;
          // the reference moves only when a score passes it by 2^8 (values stay below 2^8 times the exact ones: nothing is
          // lost in fp32)
          grow |= mx[e] > m[e] + 8.f;
        }
        if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float next = mx[e] > m[e] + 8.f ? mx[e] : m[e];
            const float a = next != m[e] ? fast_exp2(m[e] - next) : 1.f;
            m[e] = next;
            l[e] *= a;
#pragma unroll
            for (int i = 0; i < D / 8; ++i) {
              o[i][2 * e] *= a;
              o[i][2 * e + 1] *= a;
            }
          }
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) ref[e] = m[e] == -INFINITY ? 0.f : -m[e];
        // P is rounded to the cache's type for its product, as in the dense forward: the tensor instructions take 16-bit
        // values, and a second product for what is rounded off would double the work. The sum takes the unrounded values.
        // Outputs are off by 1.25 to 1.45 times what their own rounding costs (bf16: 0.0023 of their size against 0.0017).
        uint32_t pf[kSlabs][4];
#pragma unroll
        for (int i = 0; i < kSlabs * 2; ++i) {
          const float e0 = fast_exp2(fmaf(s[i][0], p.qk_scale, ref[0])), e1 = fast_exp2(fmaf(s[i][1], p.qk_scale, ref[0]));
          const float e2 = fast_exp2(fmaf(s[i][2], p.qk_scale, ref[1])), e3 = fast_exp2(fmaf(s[i][3], p.qk_scale, ref[1]));
          l[0] += e0 + e1;
          l[1] += e2 + e3;
          pf[i >> 1][(i & 1) * 2] = pack2<kBf16>(e0, e1);
          pf[i >> 1][(i & 1) * 2 + 1] = pack2<kBf16>(e2, e3);
        }
        // ---- O += P V ----
#pragma unroll
        for (int i = 0; i < kSlabs; ++i)
#pragma unroll
          for (int dd = 0; dd < D / 16; ++dd) {
            uint32_t b[4];
            ldmatrix_x4_trans(v_base + slab[i] + (dd >> 2) * group_bytes + v_row + ((((dd & 3) * 2 + v_chunk) ^ x7) << 4), b);
            mma_16816<kBf16>(o[2 * dd], pf[i], b[0], b[1]);
            mma_16816<kBf16>(o[2 * dd + 1], pf[i], b[2], b[3]);
          }
        give(slot);
      }

      // ---- the tile's end: the KS warps of each row group become one ----
      const bool any = w.blocks > 0;
      if (any) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          l[e] += __shfl_xor_sync(0xffffffffu, l[e], 1);
          l[e] += __shfl_xor_sync(0xffffffffu, l[e], 2);
          if (l4 == 0) s_ml[ks][mt * 16 + g4 + e * 8] = make_float2(m[e], l[e]);
        }
      } else if (ks == 0) {  // a tile without keys
        if (l4 == 0) s_ml[0][mt * 16 + g4] = s_ml[0][mt * 16 + g4 + 8] = make_float2(-INFINITY, 0.f);
      }
      const uint32_t slot = any ? take() : 0;
      asm volatile("bar.sync 1, %0;" ::"n"(kConsumers * 32) : "memory");
      const uint32_t buf = ring + slot * kStageBytes;
      float f[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < KS; ++i) top = fmaxf(top, s_ml[i][mt * 16 + g4 + e * 8].x);
        f[e] = top == -INFINITY ? 0.f : fast_exp2(m[e] - top);
      }
      const bool whole = w.whole != 0;
#pragma unroll 1
      for (int round = 0; round < kRounds; ++round) {
        // rows are kJoinCols fp32 values; groups of 8 columns are exchanged by the row's last bits against bank conflicts
        if (any) {
#pragma unroll
          for (int i = 0; i < D / 8; ++i) {
            if (i / (kJoinCols / 8) != round) continue;
            const int c8 = i % (kJoinCols / 8);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int r = ks * MT * 16 + mt * 16 + g4 + e * 8;
              const uint32_t addr = buf + static_cast<uint32_t>(r * kJoinCols + ((c8 ^ (r & (kJoinCols / 8 - 1) & 7)) * 8) + l4 * 2) * 4u;
              st_shared_v2(addr, __float_as_uint(o[i][2 * e] * f[e]), __float_as_uint(o[i][2 * e + 1] * f[e]));
            }
          }
          asm volatile("bar.sync 1, %0;" ::"n"(kConsumers * 32) : "memory");
        }
        for (int idx = threadIdx.x; idx < MT * 16 * (kJoinCols / 4); idx += kConsumers * 32) {
          // neighbouring threads take neighbouring columns of the output, or neighbouring rows of a partial result
          const int r = whole ? idx / (kJoinCols / 4) : idx % (MT * 16);
          const int c = (whole ? idx % (kJoinCols / 4) : idx / (MT * 16)) * 4, col = round * kJoinCols + c;
          if (r >= rows) continue;
          float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
          float top = -INFINITY, sum = 0.f;
          if (any) {
#pragma unroll
            for (int i = 0; i < KS; ++i) top = fmaxf(top, s_ml[i][r].x);
#pragma unroll
            for (int i = 0; i < KS; ++i) {
              const int rr = i * MT * 16 + r;
              float4 y;
              const uint32_t addr = buf + static_cast<uint32_t>(rr * kJoinCols + (((c >> 3) ^ (rr & (kJoinCols / 8 - 1) & 7)) * 8) + (c & 7)) * 4u;
              asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(y.x), "=f"(y.y), "=f"(y.z), "=f"(y.w) : "r"(addr) : "memory");
              x.x += y.x;
              x.y += y.y;
              x.z += y.z;
              x.w += y.w;
              const float2 ml = s_ml[i][r];
              if (ml.x != -INFINITY) sum += ml.y * fast_exp2(ml.x - top);
            }
          }
          if (whole) {
            const float inv = sum > 0.f ? 1.f / sum : 0.f;
            const int tok = w.tok0 + r / p.s.group, head = w.head * p.s.group + r % p.s.group;
            if (col < p.head_dim) {
              T *dst = static_cast<T *>(p.out) + tok * p.out_stride[0] + head * p.out_stride[1] + col;
              *reinterpret_cast<uint2 *>(dst) = make_uint2(pack2<kBf16>(x.x * inv, x.y * inv), pack2<kBf16>(x.z * inv, x.w * inv));
            }
            if (p.m_out && col == 0) p.m_out[static_cast<long long>(tok) * p.heads + head] = sum > 0.f ? top + log2f(sum) : -INFINITY;
          } else {
            p.part[(static_cast<long long>(w.slot) * (D / 4) + col / 4) * (MT * 16) + r] = x;
            if (col == 0) p.ml[static_cast<long long>(w.slot) * (MT * 16) + r] = make_float2(top, sum);
          }
        }
        asm volatile("bar.sync 1, %0;" ::"n"(kConsumers * 32) : "memory");
      }
      if (any) {
        fence_proxy_async();  // the slot was written by these threads, and is written by TMA next
        give(slot);
      }
    }
  }
  grid_dep_launch();
}

}  // namespace txp
