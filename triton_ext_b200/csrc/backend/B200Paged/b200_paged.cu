// Host side of the rotary, append and page-handling entry points (include/b200_paged.h): argument checks and launches.
// There is no CPU path here: without an sm_100 device every compute entry point fails.
#include <atomic>
#include <climits>
#include <cstdarg>
#include <cstdio>
#include <cstdlib>
#include <mutex>

#include "pages_kernel.cuh"
#include "rotary_kernel.cuh"

namespace txp {

namespace {
thread_local char g_error[512] = "";
std::atomic<uint64_t> g_launches{0};
__device__ uint32_t g_status_word;
__device__ uint32_t g_found_word;  // what the check under way has taken from it
std::mutex g_check_mutex[64];      // one check a device at a time
std::atomic<uint32_t *> g_status_ptr[64];
std::atomic<bool> g_attr_set[64];

// Reads and clears in one step: what a kernel on another stream reports meanwhile is in this check's report or stays for the
// next one. (A copy to the host and a clearing after it lost 84 of 300 such reports.)
__global__ void take_status_kernel(uint32_t *status) { g_found_word = atomicExch(status, 0u); }
}  // namespace

int fail(int code, const char *fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_error, sizeof g_error, fmt, ap);
  va_end(ap);
  return code;
}

void count_launches(int n) { g_launches.fetch_add(static_cast<uint64_t>(n)); }

int device_ready(uint32_t **status) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) {
    cudaGetLastError();
    return fail(TXD_ERR_NO_DEVICE, "no CUDA device");
  }
  uint32_t *s = g_status_ptr[dev].load(std::memory_order_acquire);
  if (!s) {
    int major = 0, minor = 0;
    TXP_CUDA(cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev));
    TXP_CUDA(cudaDeviceGetAttribute(&minor, cudaDevAttrComputeCapabilityMinor, dev));
    if (major != 10)
      return fail(TXD_ERR_NO_DEVICE, "device %d is sm_%d%d; these kernels are built for sm_100a only", dev, major, minor);
    void *p = nullptr;
    TXP_CUDA(cudaGetSymbolAddress(&p, g_status_word));
    s = static_cast<uint32_t *>(p);
    g_status_ptr[dev].store(s, std::memory_order_release);
  }
  *status = s;
  return TXD_OK;
}

int check_view(const tx_paged_view *c, tx_paged_view *out) {
  if (!c) return fail(TXD_ERR_INVALID, "null cache");
  if (c->dtype != TXD_F16 && c->dtype != TXD_BF16) return fail(TXD_ERR_UNSUPPORTED, "cache dtype must be f16 or bf16");
  if (c->batch < 0 || c->table_width < 0 || c->num_pages < 1 || c->kv_heads < 1)
    return fail(TXD_ERR_INVALID, "batch, table_width must be >= 0 and num_pages, kv_heads >= 1");
  if (c->page_size != 16 && c->page_size != 32 && c->page_size != 64 && c->page_size != 128 && c->page_size != 256)
    return fail(TXD_ERR_UNSUPPORTED, "page_size %d: 16, 32, 64, 128 and 256 are built", c->page_size);
  if (c->head_dim != 16 && c->head_dim != 32 && c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256)
    return fail(TXD_ERR_UNSUPPORTED, "head_dim %d: 16, 32, 64, 128 and 256 are built", c->head_dim);
  if (!c->k || !c->v) return fail(TXD_ERR_INVALID, "null cache pointer");
  if ((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v)) & 15)
    return fail(TXD_ERR_INVALID, "cache pointers must be 16-byte aligned");
  // a stride over one element says nothing: give it a value that every use can take
  *out = *c;
  const int32_t extent[3] = {c->num_pages, c->page_size, c->kv_heads};
  for (int i = 0; i < 3; ++i)
    if (extent[i] == 1) out->k_stride[i] = out->v_stride[i] = c->head_dim;
  c = out;
  for (int i = 0; i < 3; ++i)
    if (c->k_stride[i] < 1 || c->v_stride[i] < 1 || c->k_stride[i] % 8 || c->v_stride[i] % 8)
      return fail(TXD_ERR_UNSUPPORTED, "cache strides must be positive multiples of 16 bytes");
  if (c->batch > 0 && (!c->table || !c->kv_lens)) return fail(TXD_ERR_INVALID, "null table or kv_lens");
  if (c->table_stride < 0) return fail(TXD_ERR_INVALID, "negative table stride");
  return TXD_OK;
}

namespace {

int check_rope(const tx_rope *r, int head_dim) {
  if (r->rotary_dim < 2 || r->rotary_dim % 2 || r->rotary_dim > head_dim || r->rotary_dim > 2 * TX_ROPE_MAX_PAIRS)
    return fail(TXD_ERR_INVALID, "rotary_dim %d must be even, 2 .. min(head_dim, %d)", r->rotary_dim, 2 * TX_ROPE_MAX_PAIRS);
  return TXD_OK;
}

// The widest vector (in elements) that divides what a unit touches and keeps every access aligned.
struct Widest {
  int v;
  void divide(long long x) { while (v > 1 && x % v) v >>= 1; }
  void align(const void *p, int size) { while (v > 1 && reinterpret_cast<uintptr_t>(p) % (v * size)) v >>= 1; }
};

template <typename T>
int launch_rotary_t(const RotaryParams &prm, int v, cudaStream_t stream) {
  const long long warps = static_cast<long long>(prm.total) * prm.slices;
  const unsigned grid = static_cast<unsigned>((warps + kRotaryThreads / 32 - 1) / (kRotaryThreads / 32));
  constexpr int kWide = 16 / static_cast<int>(sizeof(T));
  auto kernel = v == kWide ? rotary_kernel<T, kWide> : v >= 2 ? rotary_kernel<T, 2> : rotary_kernel<T, 1>;
  TXP_CUDA(launch(kernel, dim3(grid), dim3(kRotaryThreads), 0, stream, prm));
  count_launches(1);
  return TXD_OK;
}

// Vector width, lanes of a head, warps of a token; then the launch.
int launch_rotary(RotaryParams &prm, long long total, int head_dim, int dtype, cudaStream_t stream) {
  if (total > INT_MAX) return fail(TXD_ERR_UNSUPPORTED, "%lld tokens: at most 2^31 - 1 in one launch", total);
  const int size = dtype == TXD_F32 ? 4 : 2;
  const int rd = prm.rope.rotary_dim;
  Widest w{16 / size};
  for (int i = 0; i < prm.parts; ++i) {
    const RotaryPart &q = prm.part[i];
    w.align(q.in, size);
    w.align(q.out, size);
    for (int j = 0; j < 3; ++j) {
      w.divide(q.in_stride[j]);
      w.divide(q.out_stride[j]);
    }
  }
  w.divide(rd / 2);  // pairs of a unit
  w.divide(head_dim - rd);
  w.divide(head_dim);
  if (w.v != 16 / size && w.v > 2) w.v = 2;
  prm.turned = rd / 2 / w.v;
  int most = 1;  // steps over the heads of the part that takes the most
  for (int i = 0; i < prm.parts; ++i) {
    RotaryPart &q = prm.part[i];
    // in place, the columns behind the turned ones stand where they belong already
    const bool same = q.kind == kTurn && q.in == q.out && q.in_stride[0] == q.out_stride[0] &&
                      q.in_stride[1] == q.out_stride[1] && q.in_stride[2] == q.out_stride[2];
    q.pass = q.kind == kCopyToPage ? head_dim / w.v : same ? 0 : (head_dim - rd) / w.v;
    const int units = (q.kind == kCopyToPage ? 0 : prm.turned) + q.pass;
    while ((1 << q.lanes_shift) < units && q.lanes_shift < 5) ++q.lanes_shift;
    const int steps = (q.heads * (1 << q.lanes_shift) + 31) / 32;
    if (steps > most) most = steps;
  }
  // A warp takes a whole token where there are tokens enough to fill the SMs (32 warps each); fewer tokens are shared.
  long long slices = total > 0 ? 148ll * 32 * 2 / total : 1;
  if (slices > most) slices = most;
  if (slices < 1) slices = 1;
  prm.slices = static_cast<uint32_t>(slices);
  prm.total = static_cast<uint32_t>(total);
  if (dtype == TXD_F32) return launch_rotary_t<float>(prm, w.v, stream);
  if (dtype == TXD_BF16) return launch_rotary_t<__nv_bfloat16>(prm, w.v, stream);
  return launch_rotary_t<__half>(prm, w.v, stream);
}

}  // namespace

int shift_of(int page_size) {
  int s = 0;
  while ((1 << s) < page_size) ++s;
  return s;
}

namespace {

int check_pages(const tx_pages_state *st) {
  if (!st) return fail(TXD_ERR_INVALID, "null state");
  if (!st->k || !st->v || !st->table || !st->lens || !st->refs) return fail(TXD_ERR_INVALID, "null state pointer");
  if (st->layers < 1 || st->num_pages < 1 || st->rows < 1 || st->width < 1)
    return fail(TXD_ERR_INVALID, "layers, num_pages, rows and width must be >= 1");
  if (st->page_size < 1 || (st->page_size & (st->page_size - 1)))
    return fail(TXD_ERR_UNSUPPORTED, "page_size %d must be a power of two", st->page_size);
  if (st->page_bytes < 16 || st->page_bytes % 16) return fail(TXD_ERR_UNSUPPORTED, "page_bytes must be a multiple of 16");
  if (st->rows > (1 << 20) || st->num_pages > (1 << 30) - 16) return fail(TXD_ERR_UNSUPPORTED, "at most 2^20 rows and 2^30 - 16 pages");
  if ((reinterpret_cast<uintptr_t>(st->k) | reinterpret_cast<uintptr_t>(st->v) | reinterpret_cast<uintptr_t>(st->refs)) & 15)
    return fail(TXD_ERR_INVALID, "k, v and refs must be 16-byte aligned");
  return TXD_OK;
}

int pages_params(const tx_pages_state *st, void *workspace, PagesParams *p) {
  int rc = device_ready(&p->status);
  if (rc) return rc;
  p->k = static_cast<uint4 *>(st->k);
  p->v = static_cast<uint4 *>(st->v);
  p->page_vecs = st->page_bytes / 16;
  p->table = st->table;
  p->lens = st->lens;
  p->refs = st->refs;
  p->ws = static_cast<int32_t *>(workspace);
  p->layers = st->layers;
  p->num_pages = st->num_pages;
  p->page_shift = shift_of(st->page_size);
  p->rows = st->rows;
  p->width = st->width;
  return TXD_OK;
}

int check_workspace(const void *ws) {
  if (!ws || (reinterpret_cast<uintptr_t>(ws) & 15)) return fail(TXD_ERR_INVALID, "the workspace must be a 16-byte aligned device buffer");
  return TXD_OK;
}

// Blocks for copies of at most `pages` pages.
unsigned copy_grid(const tx_pages_state *st, long long pages) {
  const long long pieces = (st->page_bytes / 16 + 256 * kCopyVecs - 1) / (256 * kCopyVecs);
  const double all = static_cast<double>(pages) * st->layers * 2 * pieces;
  return all < 148 * 8 ? static_cast<unsigned>(all < 1 ? 1 : all) : 148 * 8;
}

int set_plan_smem() {
  int dev = 0;
  TXP_CUDA(cudaGetDevice(&dev));
  if (!g_attr_set[dev].load(std::memory_order_acquire)) {
    TXP_CUDA(cudaFuncSetAttribute(pages_reserve_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024));
    g_attr_set[dev].store(true, std::memory_order_release);
  }
  return TXD_OK;
}

}  // namespace
}  // namespace txp

using namespace txp;

extern "C" {

const char *tx_paged_last_error(void) { return g_error; }
uint64_t tx_paged_kernel_launches(void) { return g_launches.load(); }

int tx_rotary(const tx_rope *rope, const tx_rotary_problem *pr, const void *positions, void *stream) {
  if (!rope || !pr) return fail(TXD_ERR_INVALID, "null argument");
  if (pr->dtype != TXD_F16 && pr->dtype != TXD_BF16 && pr->dtype != TXD_F32)
    return fail(TXD_ERR_UNSUPPORTED, "rotary takes f16, bf16 or f32");
  if (pr->head_dim > 1024) return fail(TXD_ERR_UNSUPPORTED, "head_dim %d: at most 1024", pr->head_dim);
  if (pr->batch < 0 || pr->tokens < 0 || pr->head_dim < 1 || pr->parts < 1 || pr->parts > 2)
    return fail(TXD_ERR_INVALID, "batch, tokens must be >= 0, head_dim >= 1, parts 1 or 2");
  int rc = check_rope(rope, pr->head_dim);
  if (rc) return rc;
  RotaryParams prm = {};
  int heads = 0;
  for (int i = 0; i < pr->parts; ++i) {
    const tx_rotary_part &q = pr->part[i];
    if (q.heads < 0) return fail(TXD_ERR_INVALID, "negative heads");
    heads |= q.heads;
    prm.part[i].heads = q.heads;
    prm.part[i].in = q.in;
    prm.part[i].out = q.out;
    for (int j = 0; j < 3; ++j) {
      prm.part[i].in_stride[j] = q.in_stride[j];
      prm.part[i].out_stride[j] = q.out_stride[j];
    }
    prm.part[i].kind = kTurn;
  }
  const long long total = static_cast<long long>(pr->batch) * pr->tokens;
  if (total == 0 || heads == 0) return TXD_OK;
  if (!positions) return fail(TXD_ERR_INVALID, "null positions");
  for (int i = 0; i < pr->parts; ++i)
    if (pr->part[i].heads > 0 && (!pr->part[i].in || !pr->part[i].out)) return fail(TXD_ERR_INVALID, "null tensor pointer");
  if ((rc = device_ready(&prm.status))) return rc;
  prm.rope = *rope;
  prm.positions = positions;
  prm.positions_64 = pr->positions_64;
  prm.position_stride[0] = pr->position_stride[0];
  prm.position_stride[1] = pr->position_stride[1];
  prm.inverse = pr->inverse;
  prm.tokens = static_cast<uint32_t>(pr->tokens);
  prm.parts = pr->parts;
  return launch_rotary(prm, total, pr->head_dim, pr->dtype, static_cast<cudaStream_t>(stream));
}

int tx_paged_append(const tx_paged_view *cache, const tx_rope *rope, const tx_append_problem *pr, void *stream) {
  tx_paged_view view;
  int rc = check_view(cache, &view);
  if (rc) return rc;
  const tx_paged_view *c = &view;
  if (!pr) return fail(TXD_ERR_INVALID, "null problem");
  if (pr->tokens < 0 || pr->q_heads < 0) return fail(TXD_ERR_INVALID, "tokens and q_heads must be >= 0");
  if (rope && (rc = check_rope(rope, c->head_dim))) return rc;
  if (pr->tokens == 0) return TXD_OK;
  if (!pr->k || !pr->v || (pr->q_heads > 0 && (!pr->q || !pr->q_out))) return fail(TXD_ERR_INVALID, "null tensor pointer");
  RotaryParams prm = {};
  if ((rc = device_ready(&prm.status))) return rc;
  if (rope) prm.rope = *rope;
  else prm.rope.rotary_dim = 0, prm.rope.magnitude = 1.f;
  int n = 0;
  auto part = [&](const void *in, const int64_t *in_s, void *out, const int64_t *out_s, int kind, int h) {
    RotaryPart &q = prm.part[n];
    q.in = in;
    q.out = out;
    q.in_stride[1] = in_s[1];
    q.in_stride[2] = in_s[0];
    if (kind == kTurn) q.out_stride[1] = out_s[1], q.out_stride[2] = out_s[0];
    else for (int j = 0; j < 3; ++j) q.out_stride[j] = out_s[j];
    q.kind = kind;
    q.heads = h;
    ++n;
  };
  // without a rotation, a q that is its own output has nothing to be done to it
  const bool idle_q = !rope && pr->q == pr->q_out && pr->q_stride[0] == pr->q_out_stride[0] && pr->q_stride[1] == pr->q_out_stride[1];
  if (pr->q_heads > 0 && !idle_q) part(pr->q, pr->q_stride, pr->q_out, pr->q_out_stride, kTurn, pr->q_heads);
  part(pr->k, pr->k_stride, c->k, c->k_stride, rope ? kTurnToPage : kCopyToPage, c->kv_heads);
  part(pr->v, pr->v_stride, c->v, c->v_stride, kCopyToPage, c->kv_heads);
  prm.parts = n;
  prm.table = c->table;
  prm.table_stride = c->table_stride;
  prm.kv_lens = c->kv_lens;
  prm.cu_q = c->cu_q;
  prm.batch = c->batch;
  prm.table_width = c->table_width;
  prm.num_pages = c->num_pages;
  prm.page_shift = shift_of(c->page_size);
  prm.tokens = static_cast<uint32_t>(pr->tokens);
  return launch_rotary(prm, pr->tokens, c->head_dim, c->dtype, static_cast<cudaStream_t>(stream));
}

int64_t tx_pages_workspace(const tx_pages_state *st, int32_t n) {
  if (!st || n < 0) return 0;
  const int64_t fork = static_cast<int64_t>(n) * (static_cast<int64_t>(st->width) + 1);
  const int64_t reserve = 2 * static_cast<int64_t>(n) + st->num_pages;
  const int64_t compact = 2 * (static_cast<int64_t>(st->num_pages) + 1);
  int64_t most = fork > reserve ? fork : reserve;
  if (compact > most) most = compact;
  return (most + kPlanPairs) * 4 + 16;
}

int tx_pages_free(const tx_pages_state *st, const int32_t *rows, int32_t n, void *stream) {
  int rc = check_pages(st);
  if (rc) return rc;
  if (n < 0 || (n > 0 && !rows)) return fail(TXD_ERR_INVALID, "a list of n >= 0 rows is wanted");
  if (n == 0) return TXD_OK;
  PagesParams p = {};
  if ((rc = pages_params(st, nullptr, &p))) return rc;
  TXP_CUDA(launch(pages_free_kernel, dim3(n), dim3(256), 0, static_cast<cudaStream_t>(stream), p, rows));
  count_launches(1);
  return TXD_OK;
}

int tx_pages_truncate(const tx_pages_state *st, const int32_t *rows, const int32_t *keep, int32_t n, void *stream) {
  int rc = check_pages(st);
  if (rc) return rc;
  if (n < 0 || (n > 0 && (!rows || !keep))) return fail(TXD_ERR_INVALID, "lists of n >= 0 rows and lengths are wanted");
  if (n == 0) return TXD_OK;
  PagesParams p = {};
  if ((rc = pages_params(st, nullptr, &p))) return rc;
  TXP_CUDA(launch(pages_truncate_kernel, dim3(n), dim3(256), 0, static_cast<cudaStream_t>(stream), p, rows, keep));
  count_launches(1);
  return TXD_OK;
}

int tx_pages_fork(const tx_pages_state *st, const int32_t *dst, const int32_t *src, int32_t n, void *workspace, void *stream) {
  int rc = check_pages(st);
  if (rc) return rc;
  if (n < 0 || (n > 0 && (!dst || !src))) return fail(TXD_ERR_INVALID, "lists of n >= 0 rows are wanted");
  if (n == 0) return TXD_OK;
  if ((rc = check_workspace(workspace))) return rc;
  PagesParams p = {};
  if ((rc = pages_params(st, workspace, &p))) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  TXP_CUDA(launch(pages_fork_take_kernel, dim3(n), dim3(256), 0, s, p, dst, src, n));
  TXP_CUDA(launch(pages_fork_put_kernel, dim3(n), dim3(256), 0, s, p, dst));
  count_launches(2);
  return TXD_OK;
}

int tx_pages_reserve(const tx_pages_state *st, const int32_t *rows, const int32_t *counts, int32_t n, void *workspace,
                     void *stream) {
  return tx_pages_reserve_lens(st, rows, counts, n, nullptr, workspace, stream);
}

int tx_pages_reserve_lens(const tx_pages_state *st, const int32_t *rows, const int32_t *counts, int32_t n, int32_t *step_lens,
                          void *workspace, void *stream) {
  int rc = check_pages(st);
  if (rc) return rc;
  if (n < 0 || (n > 0 && (!rows || !counts))) return fail(TXD_ERR_INVALID, "lists of n >= 0 rows and counts are wanted");
  if (n > TX_PAGES_MAX_LIST) return fail(TXD_ERR_UNSUPPORTED, "at most %d rows in one reserve", TX_PAGES_MAX_LIST);
  if (static_cast<long long>(n) * (st->width + 1ll) > INT_MAX) return fail(TXD_ERR_UNSUPPORTED, "too many pages in one reserve");
  if (n == 0) return TXD_OK;
  if ((rc = check_workspace(workspace))) return rc;
  PagesParams p = {};
  if ((rc = pages_params(st, workspace, &p))) return rc;
  if ((rc = set_plan_smem())) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const size_t smem = (4 * static_cast<size_t>(n) + (st->rows + 31) / 32) * 4;
  TXP_CUDA(launch(pages_reserve_plan_kernel, dim3(1), dim3(kPlanThreads), smem, s, p, rows, counts, n, step_lens));
  TXP_CUDA(launch(pages_copy_kernel, dim3(copy_grid(st, n)), dim3(256), 0, s, p));
  count_launches(2);
  return TXD_OK;
}

int tx_pages_compact(const tx_pages_state *st, void *workspace, void *stream) {
  int rc = check_pages(st);
  if (rc) return rc;
  if ((rc = check_workspace(workspace))) return rc;
  PagesParams p = {};
  if ((rc = pages_params(st, workspace, &p))) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  TXP_CUDA(launch(pages_compact_plan_kernel, dim3(1), dim3(kPlanThreads), 0, s, p));
  TXP_CUDA(launch(pages_compact_move_kernel, dim3(copy_grid(st, st->num_pages)), dim3(256), 0, s, p));
  count_launches(2);
  return TXD_OK;
}

int tx_pages_copy(const tx_pages_state *st, const int32_t *src, const int32_t *dst, int32_t n, void *stream) {
  int rc = check_pages(st);
  if (rc) return rc;
  if (n < 0 || (n > 0 && (!src || !dst))) return fail(TXD_ERR_INVALID, "lists of n >= 0 pages are wanted");
  for (int i = 0; i < n; ++i)
    if (src[i] < 0 || src[i] >= st->num_pages || dst[i] < 0 || dst[i] >= st->num_pages)
      return fail(TXD_ERR_INVALID, "pair %d (%d to %d) is outside the %d pages", i, src[i], dst[i], st->num_pages);
  if (n == 0) return TXD_OK;
  unsigned char *seen = static_cast<unsigned char *>(calloc(static_cast<size_t>(st->num_pages), 1));
  if (!seen) return fail(TXD_ERR_INVALID, "out of host memory");
  int clash = -1;
  for (int i = 0; i < n; ++i) {
    if (seen[dst[i]]) clash = dst[i];
    seen[dst[i]] = 1;
  }
  for (int i = 0; i < n; ++i)
    if (seen[src[i]]) clash = src[i];
  free(seen);
  if (clash >= 0) return fail(TXD_ERR_INVALID, "page %d is a destination twice, or source and destination", clash);
  PagesParams p = {};
  if ((rc = pages_params(st, nullptr, &p))) return rc;
  for (int at = 0; at < n; at += kParamPairs) {
    ParamPairs pp;
    const int count = n - at < kParamPairs ? n - at : kParamPairs;
    for (int i = 0; i < count; ++i) {
      pp.pair[2 * i] = src[at + i];
      pp.pair[2 * i + 1] = dst[at + i];
    }
    TXP_CUDA(launch(pages_copy_listed_kernel, dim3(copy_grid(st, count)), dim3(256), 0, static_cast<cudaStream_t>(stream), p, pp, count));
    count_launches(1);
  }
  return TXD_OK;
}

int tx_paged_check(void *stream_v) {
  uint32_t *status = nullptr;
  int rc = device_ready(&status);
  if (rc) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream_v);
  TXP_CUDA(cudaStreamSynchronize(s));
  int dev = 0;
  TXP_CUDA(cudaGetDevice(&dev));
  uint32_t found = 0;
  {
    std::lock_guard<std::mutex> lock(g_check_mutex[dev]);
    take_status_kernel<<<1, 1, 0, s>>>(status);
    TXP_CUDA(cudaGetLastError());
    TXP_CUDA(cudaMemcpyFromSymbolAsync(&found, g_found_word, sizeof found, 0, cudaMemcpyDeviceToHost, s));
    TXP_CUDA(cudaStreamSynchronize(s));
  }
  if (!found) return TXD_OK;
  return fail(found & kTimeout ? TXD_ERR_DEVICE_TIMEOUT : TXD_ERR_INVALID, "on the device:%s%s%s%s%s%s%s",
              found & kTimeout ? " a bounded wait inside the paged attention kernel ran out;" : "",
              found & kBadPage ? " a page-table entry outside the cache;" : "",
              found & kBadRow ? " a row outside the table, listed twice or with a negative count;" : "",
              found & kNoRoomInRow ? " a position past the width of the page table;" : "",
              found & kNoFreePages ? " no free pages;" : "",
              found & kBadLength ? " a length below zero or below the number of new tokens;" : "",
              found & kBadOffsets ? " offsets in cu_q that fall or lie outside the new tokens;" : "");
}

}  // extern "C"
