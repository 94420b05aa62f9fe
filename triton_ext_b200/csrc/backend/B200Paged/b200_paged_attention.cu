// Host side of paged attention (include/b200_paged.h): argument checks, the choice of kernel, TMA descriptors, launches.
// There is no CPU path here: without an sm_100 device every compute entry point fails.
#include <atomic>
#include <climits>
#include <cstdlib>
#include <mutex>

#include "paged_tile_kernel.cuh"

namespace txp {
namespace {

typedef CUresult (*EncodeTiledFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                  const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_fn() {
  static EncodeTiledFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void *p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiledFn>(p);
  });
  return fn;
}

// One pool as {64 columns, slots, column groups, heads, pages}; a box is `box_rows` slots of one page and head, with
// `box_groups` column groups. Columns past head_dim (16 and 32) are out of bounds and arrive as zeros.
int encode_pool(CUtensorMap *map, const void *ptr, const tx_paged_view &c, const int64_t *stride, int box_rows,
                int box_groups) {
  EncodeTiledFn enc = encode_fn();
  if (!enc) return fail(TXD_ERR_NO_DEVICE, "cuTensorMapEncodeTiled is not available from the CUDA driver");
  const int groups = c.head_dim > 64 ? c.head_dim / 64 : 1;
  const cuuint64_t dims[5] = {static_cast<cuuint64_t>(c.head_dim < 64 ? c.head_dim : 64), static_cast<cuuint64_t>(c.page_size),
                              static_cast<cuuint64_t>(groups), static_cast<cuuint64_t>(c.kv_heads), static_cast<cuuint64_t>(c.num_pages)};
  const cuuint64_t strides[4] = {static_cast<cuuint64_t>(stride[1]) * 2, 128, static_cast<cuuint64_t>(stride[2]) * 2,
                                 static_cast<cuuint64_t>(stride[0]) * 2};
  const cuuint32_t box[5] = {64, static_cast<cuuint32_t>(box_rows), static_cast<cuuint32_t>(box_groups), 1, 1};
  const cuuint32_t estr[5] = {1, 1, 1, 1, 1};
  const CUresult r = enc(map, c.dtype == TXD_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 5,
                         const_cast<void *>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(TXD_ERR_CUDA, "cuTensorMapEncodeTiled (pool) failed with code %d", static_cast<int>(r));
  return TXD_OK;
}

// Queries as {head_dim, heads, tokens}; a box is the heads of one key head of a sub-tile's tokens, every `every`-th one.
int encode_queries(CUtensorMap *map, const void *ptr, const tx_paged_view &c, const int64_t *stride, int heads, int tokens,
                   int group, int sub_tokens, int every) {
  EncodeTiledFn enc = encode_fn();
  if (!enc) return fail(TXD_ERR_NO_DEVICE, "cuTensorMapEncodeTiled is not available from the CUDA driver");
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(c.head_dim), static_cast<cuuint64_t>(heads), static_cast<cuuint64_t>(tokens)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(stride[1]) * 2, static_cast<cuuint64_t>(stride[0]) * 2};
  const cuuint32_t box[3] = {64, static_cast<cuuint32_t>(group), static_cast<cuuint32_t>(sub_tokens * every)};
  const cuuint32_t estr[3] = {1, 1, static_cast<cuuint32_t>(every)};
  const CUresult r = enc(map, c.dtype == TXD_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
                         const_cast<void *>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(TXD_ERR_CUDA, "cuTensorMapEncodeTiled (queries) failed with code %d", static_cast<int>(r));
  return TXD_OK;
}

constexpr int kRowBlock32 = 128;  // KV tokens of a block where a tile has 32 rows

// Which kernel takes a call of few rows: a function of the group, the bound on a sequence's new tokens and the head dimension.
struct RowShape {
  int rows, block, per_sm;  // rows of a tile, KV tokens of a block, CTAs per SM
};

RowShape row_shape(int kernel_d, long long rows) {
  if (kernel_d == 256) return {rows <= 16 ? 16 : rows <= 32 ? 32 : 64, 64, 1};
  if (rows <= 16) return {16, 64, 2};
  return {32, kRowBlock32, 1};
}

int sm_count() {
  static std::atomic<int> cached[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) {
    cudaGetLastError();
    return 148;  // no device: only sizes are asked for
  }
  int n = cached[dev].load(std::memory_order_relaxed);
  if (!n) {
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 148;
    cached[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}

struct Plan {
  tx_paged_view view;
  int kernel_d, group, rows, ctas;
  bool tiled;  // the kernel for many rows
  bool cuts;   // tiles may be cut, and joined by a second kernel
  RowShape shape;
  size_t borders_bytes, part_bytes, ml_bytes;
  int64_t bytes() const { return static_cast<int64_t>(borders_bytes + part_bytes + ml_bytes); }
};

int make_plan(const tx_paged_view *cache, const tx_paged_attn_problem *pr, Plan *plan) {
  int rc = check_view(cache, &plan->view);
  if (rc) return rc;
  if (!pr) return fail(TXD_ERR_INVALID, "null problem");
  const tx_paged_view &c = plan->view;
  if (pr->tokens < 0 || pr->q_heads < 1) return fail(TXD_ERR_INVALID, "tokens must be >= 0 and q_heads >= 1");
  if (pr->q_heads % c.kv_heads) return fail(TXD_ERR_INVALID, "q_heads %d is not a multiple of kv_heads %d", pr->q_heads, c.kv_heads);
  plan->group = pr->q_heads / c.kv_heads;
  if (plan->group > 64) return fail(TXD_ERR_UNSUPPORTED, "%d query heads to a key head: at most 64 are built", plan->group);
  if (pr->tokens > 0 && pr->max_q < 1) return fail(TXD_ERR_INVALID, "max_q must be >= 1");
  if (pr->window < 0 || (pr->window > 0 && !pr->causal)) return fail(TXD_ERR_INVALID, "a window is >= 0 and goes with causal");
  if (!(pr->sm_scale > 0.f) || pr->sm_scale > 1e30f) return fail(TXD_ERR_INVALID, "sm_scale must be positive and finite");
  if (static_cast<long long>(c.table_width) * c.page_size > (1ll << 30)) return fail(TXD_ERR_UNSUPPORTED, "a row of the page table holds more than 2^30 tokens");
  if (c.cu_q == nullptr && pr->tokens != c.batch) return fail(TXD_ERR_INVALID, "without cu_q there is one new token for each of the %d sequences", c.batch);
  plan->kernel_d = c.head_dim <= 64 ? 64 : c.head_dim;
  int max_q = pr->max_q;
  if (max_q > pr->tokens) max_q = pr->tokens;
  plan->shape = row_shape(plan->kernel_d, static_cast<long long>(plan->group) * (max_q > 0 ? max_q : 1));
  // 128-row tiles on tcgen05 for head dimensions up to 128 (256 columns of O for two sub-tiles do not fit tensor memory
  // next to S); up to 32 rows the streaming kernel. Measured, 16 sequences of up to 4100 tokens, 32 + 8 heads of 128, tiles
  // against streams: 32 rows 71 us and 57, 64 rows 66 us and 84.
  plan->tiled = plan->kernel_d <= 128 && static_cast<long long>(plan->group) * max_q > 32;
  plan->rows = plan->tiled ? 256 : plan->shape.rows;
  plan->ctas = sm_count() * (plan->tiled ? 1 : plan->shape.per_sm);
  // Single tokens over at most 8 blocks: a tile is over sooner than a second kernel has joined its parts (1 sequence of 512
  // tokens, 16 + 4 heads of 64: 10.2 us cut or whole, and a launch less; of 256 tokens: 7.9 us whole). The host knows what
  // the table has room for and no length, so short sequences under a wide table are cut.
  plan->cuts = plan->tiled || static_cast<long long>(c.table_width) * c.page_size > 8 * plan->shape.block;
  plan->borders_bytes = (static_cast<size_t>(plan->ctas) * 16 + 255) / 256 * 256;
  const size_t rows = static_cast<size_t>(plan->ctas) * 2 * plan->rows;
  plan->part_bytes = rows * plan->kernel_d * 4;
  plan->ml_bytes = rows * 8;
  return TXD_OK;
}

// The kernel's shared-memory limit is raised once per device.
template <typename P>
cudaError_t allow_smem(void (*kernel)(P), int bytes, std::atomic<uint64_t> *done) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (done->load(std::memory_order_acquire) >> dev & 1) return cudaSuccess;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) done->fetch_or(1ull << dev, std::memory_order_acq_rel);
  return e;
}

template <bool kBf16, int D, int BS, int MT, int KS, int kStages, int kPerSm>
int launch_row(const RowParams &prm, int ctas, cudaStream_t stream) {
  static std::atomic<uint64_t> done{0};
  auto kernel = paged_row_kernel<kBf16, D, BS, MT, KS, kStages, kPerSm>;
  constexpr int smem = row_smem_bytes<D, BS, kStages>();
  TXP_CUDA(allow_smem(kernel, smem, &done));
  TXP_CUDA(launch(kernel, dim3(ctas), dim3((MT * KS + 1) * 32), smem, stream, prm));
  return TXD_OK;
}

template <bool kBf16>
int launch_row_any(const RowShape &shape, int kernel_d, const RowParams &prm, int ctas, cudaStream_t s) {
  // ring: 96 KB a CTA where two share an SM, 192 KB where one has it
  if (kernel_d == 64) {
    if (shape.rows == 16) return launch_row<kBf16, 64, 64, 1, 4, 6, 2>(prm, ctas, s);
    return launch_row<kBf16, 64, kRowBlock32, 2, 4, 768 / kRowBlock32, 1>(prm, ctas, s);
  }
  if (kernel_d == 128) {
    if (shape.rows == 16) return launch_row<kBf16, 128, 64, 1, 4, 3, 2>(prm, ctas, s);
    return launch_row<kBf16, 128, kRowBlock32, 2, 4, 384 / kRowBlock32, 1>(prm, ctas, s);
  }
  if (shape.rows == 16) return launch_row<kBf16, 256, 64, 1, 4, 3, 1>(prm, ctas, s);
  if (shape.rows == 32) return launch_row<kBf16, 256, 64, 2, 4, 3, 1>(prm, ctas, s);
  return launch_row<kBf16, 256, 64, 4, 2, 3, 1>(prm, ctas, s);
}

template <bool kBf16, int D>
int launch_tile(const TileParams &prm, int ctas, cudaStream_t stream) {
  static std::atomic<uint64_t> done{0};
  auto kernel = paged_tile_kernel<kBf16, D>;
  TXP_CUDA(allow_smem(kernel, TileShape<D>::kSmem, &done));
  TXP_CUDA(launch(kernel, dim3(ctas), dim3(kTileThreads), TileShape<D>::kSmem, stream, prm));
  return TXD_OK;
}

template <bool kBf16>
int launch_tile_any(const Plan &plan, const TileParams &prm, cudaStream_t s) {
  return plan.kernel_d == 64 ? launch_tile<kBf16, 64>(prm, plan.ctas, s) : launch_tile<kBf16, 128>(prm, plan.ctas, s);
}

// tcgen05 instruction descriptor: fp32 accumulator, A and B f16 or bf16, B n-major or k-major, 128 x n
uint32_t mma_idesc(bool bf16, bool b_mn_major, int n) {
  const uint32_t type = bf16 ? 1u : 0u;
  return 1u << 4 | type << 7 | type << 10 | (b_mn_major ? 1u : 0u) << 16 | static_cast<uint32_t>(n >> 3) << 17 | (128u >> 4) << 24;
}

template <typename T, int D>
int launch_join_d(const Plan &plan, const JoinParams &j, cudaStream_t s) {
  const unsigned borders = static_cast<unsigned>(j.ctas - 1), row_groups = static_cast<unsigned>(plan.rows + 31) / 32;
  if (plan.rows == 16) TXP_CUDA(launch(paged_join_kernel<T, D, 16>, dim3(borders), dim3(D * 2), 0, s, j));
  else if (plan.rows <= 64) TXP_CUDA(launch(paged_join_kernel<T, D, 32>, dim3(borders, row_groups), dim3(D * 2), 0, s, j));
  else TXP_CUDA(launch(paged_join_kernel<T, D, 0>, dim3(borders, (row_groups * (D / 16) + 7) / 8), dim3(256), 0, s, j));
  return TXD_OK;
}

template <typename T>
int launch_join(const Plan &plan, const JoinParams &j, cudaStream_t s) {
  if (j.ctas < 2) return TXD_OK;
  if (plan.kernel_d == 64) return launch_join_d<T, 64>(plan, j, s);
  if (plan.kernel_d == 128) return launch_join_d<T, 128>(plan, j, s);
  return launch_join_d<T, 256>(plan, j, s);
}

unsigned long long wait_limit() {
  unsigned long long ns = 2000ull * 1000 * 1000;
  if (const char *e = getenv("TXD_WAIT_LIMIT_MS")) {
    const long ms = atol(e);
    if (ms > 0) ns = static_cast<unsigned long long>(ms) * 1000 * 1000;
  }
  return ns;
}

}  // namespace
}  // namespace txp

using namespace txp;

extern "C" {

int64_t tx_paged_attention_workspace(const tx_paged_view *cache, const tx_paged_attn_problem *pr) {
  Plan plan;
  if (make_plan(cache, pr, &plan)) return 0;
  return plan.bytes();
}

int tx_paged_attention(const tx_paged_view *cache, const tx_paged_attn_problem *pr, void *workspace, int64_t workspace_bytes,
                       void *stream_v) {
  Plan plan;
  int rc = make_plan(cache, pr, &plan);
  if (rc) return rc;
  if (pr->tokens == 0 || plan.view.batch == 0) return TXD_OK;
  if (!pr->q || !pr->out) return fail(TXD_ERR_INVALID, "null tensor pointer");
  if ((reinterpret_cast<uintptr_t>(pr->q) | reinterpret_cast<uintptr_t>(pr->out)) & 15)
    return fail(TXD_ERR_INVALID, "q and out must be 16-byte aligned");
  int64_t q_stride[2], o_stride[2];
  for (int i = 0; i < 2; ++i) {
    const bool one = (i == 0 ? pr->tokens : pr->q_heads) == 1;
    q_stride[i] = one ? plan.view.head_dim : pr->q_stride[i];
    o_stride[i] = one ? plan.view.head_dim : pr->out_stride[i];
    if (q_stride[i] < 1 || o_stride[i] < 1 || q_stride[i] % 8 || o_stride[i] % 8)
      return fail(TXD_ERR_UNSUPPORTED, "strides of q and out must be positive multiples of 16 bytes");
  }
  uint32_t *status = nullptr;
  if ((rc = device_ready(&status))) return rc;
  if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15) || workspace_bytes < plan.bytes())
    return fail(TXD_ERR_INVALID, "a 16-byte aligned workspace of %lld bytes is wanted", static_cast<long long>(plan.bytes()));
  const tx_paged_view &c = plan.view;
  char *ws = static_cast<char *>(workspace);

  Sched sched = {};
  sched.kv_lens = c.kv_lens;
  sched.cu_q = c.cu_q;
  sched.batch = c.batch;
  sched.tokens = pr->tokens;
  sched.kv_heads = c.kv_heads;
  sched.group = plan.group;
  sched.tile_tokens = plan.rows / plan.group;
  sched.causal = pr->causal ? 1 : 0;
  sched.window = pr->window > (1 << 30) ? 1 << 30 : pr->window;
  sched.max_kv = c.table_width * c.page_size;
  sched.block_shift = shift_of(plan.shape.block);
  sched.tile_cost = 2;
  sched.min_part = plan.cuts ? 1 : 1 << 30;  // at two, 8 drafts over ragged lengths take 27.7 us, not 27.2, and 16 37.5, not 35.7
  sched.min_share = 3;
  sched.waves = kMaxWaves;
  sched.status = status;

  if (plan.tiled) {
    sched.tile_tokens = 2 * (128 / plan.group);
    sched.block_shift = 7;
  }
  cudaStream_t stream = static_cast<cudaStream_t>(stream_v);
  const bool bf16 = c.dtype == TXD_BF16;
  int4 *borders = reinterpret_cast<int4 *>(ws);
  float4 *part = reinterpret_cast<float4 *>(ws + plan.borders_bytes);
  float2 *ml = reinterpret_cast<float2 *>(ws + plan.borders_bytes + plan.part_bytes);
  const float qk_scale = pr->sm_scale * 1.44269504f;  // 1 / ln 2
  int32_t inject_stall = 0;
  if (const char *e = getenv("TXD_INJECT_STALL")) inject_stall = atoi(e) != 0;
  auto fill = [&](auto &prm, int box_rows) {
    prm.s = sched;
    prm.out = pr->out;
    prm.m_out = pr->m;
    for (int i = 0; i < 2; ++i) prm.out_stride[i] = o_stride[i];
    prm.table = c.table;
    prm.table_stride = c.table_stride;
    prm.borders = borders;
    prm.part = part;
    prm.ml = ml;
    prm.wait_limit_ns = wait_limit();
    prm.qk_scale = qk_scale;
    prm.num_pages = c.num_pages;
    prm.page_shift = shift_of(c.page_size);
    prm.box_shift = shift_of(box_rows);
    prm.heads = pr->q_heads;
    prm.head_dim = c.head_dim;
    prm.inject_stall = inject_stall;
  };
  if (plan.tiled) {
    TileParams prm = {};
    const int box_rows = c.page_size < 128 ? c.page_size : 128;
    prm.sub_tokens = 128 / plan.group;
    prm.part_rows = plan.rows;
    for (int i = 0; i < 2; ++i)
      if ((rc = encode_queries(i ? &prm.tmap_q2 : &prm.tmap_q, pr->q, c, q_stride, pr->q_heads, pr->tokens, plan.group, prm.sub_tokens, i + 1))) return rc;
    if ((rc = encode_pool(&prm.tmap_k, c.k, c, c.k_stride, box_rows, 1))) return rc;
    if ((rc = encode_pool(&prm.tmap_v, c.v, c, c.v_stride, box_rows, 1))) return rc;
    fill(prm, box_rows);
    prm.idesc_qk = mma_idesc(bf16, false, 128);
    prm.idesc_pv = mma_idesc(bf16, true, plan.kernel_d);
    if ((rc = bf16 ? launch_tile_any<true>(plan, prm, stream) : launch_tile_any<false>(plan, prm, stream))) return rc;
  } else {
    RowParams prm = {};
    const int box_rows = c.page_size < plan.shape.block ? c.page_size : plan.shape.block;
    const int groups = plan.kernel_d / 64;
    if ((rc = encode_pool(&prm.tmap_k, c.k, c, c.k_stride, box_rows, groups))) return rc;
    if ((rc = encode_pool(&prm.tmap_v, c.v, c, c.v_stride, box_rows, groups))) return rc;
    fill(prm, box_rows);
    prm.q = pr->q;
    for (int i = 0; i < 2; ++i) prm.q_stride[i] = q_stride[i];
    if ((rc = bf16 ? launch_row_any<true>(plan.shape, plan.kernel_d, prm, plan.ctas, stream)
                   : launch_row_any<false>(plan.shape, plan.kernel_d, prm, plan.ctas, stream))) return rc;
  }

  if (!plan.cuts) {
    count_launches(1);
    return TXD_OK;
  }
  JoinParams join = {};
  join.s = sched;
  join.borders = borders;
  join.part = part;
  join.ml = ml;
  join.out = pr->out;
  join.m_out = pr->m;
  join.out_stride[0] = o_stride[0];
  join.out_stride[1] = o_stride[1];
  join.ctas = plan.ctas;
  join.rows = plan.rows;
  join.heads = pr->q_heads;
  join.head_dim = c.head_dim;
  if ((rc = bf16 ? launch_join<__nv_bfloat16>(plan, join, stream) : launch_join<__half>(plan, join, stream))) return rc;
  count_launches(2);
  return TXD_OK;
}

}  // extern "C"
