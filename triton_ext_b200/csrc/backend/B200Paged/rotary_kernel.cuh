// Rotary positions, and the append of new tokens to a paged cache.
//
// Pair i of a head is the complex number x1 + i x2; a position p turns it by the angle 2 pi p f_i, where f_i is kept as
// a 64-bit fraction of a turn. p * f_i in 64-bit wrap-around arithmetic IS the angle modulo whole turns, so no range
// reduction loses anything at far positions (a product in fp32 is off by 0.06 rad at position 2^20 already); its upper
// 32 bits go through sincospi. The cosines and sines of a token are computed once per block and used by all heads.
//
// The work is one read and one write of every value: HBM bound when there are many tokens, launch bound when there are
// few. A block takes a few tokens, so that every thread has up to kUnroll pairs of vectors in flight before the block
// looks at positions and computes angles; the loads do not depend on either.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "paged_host.h"

namespace txp {

constexpr int kRotaryThreads = 256;
constexpr int kMaxBlockTokens = 8;
constexpr int kUnroll = 4;

enum RotaryKind : int32_t { kTurn = 0, kTurnToPage = 1, kCopyToPage = 2 };

struct RotaryPart {
  const void *in;
  void *out;               // kTurn: the tensor; else the pool
  long long in_stride[3];  // batch, head, token
  long long out_stride[3]; // kTurn: batch, head, token; else page, slot, head
  int32_t kind, first_unit;
  int32_t turned, units;   // units of a head: `turned` pairs of vectors, then single vectors that pass
};

struct RotaryParams {
  tx_rope rope;
  RotaryPart part[3];
  const void *positions;   // NULL in an append
  long long position_stride[2];
  const int32_t *table, *kv_lens, *cu_q;
  long long table_stride;
  uint32_t *status;
  long long total;         // tokens of all batch entries
  int32_t tokens, parts, units, block_tokens, positions_64, inverse;
  int32_t batch, table_width, num_pages, page_shift;
};

template <typename T, int V>
struct alignas(sizeof(T) * V) Pack {
  T x[V];
};

__device__ __forceinline__ float rot_f32(float x) { return x; }
__device__ __forceinline__ float rot_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float rot_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T rot_from(float x);
template <>
__device__ __forceinline__ float rot_from<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half rot_from<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 rot_from<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

template <typename T, int V>
__global__ void __launch_bounds__(kRotaryThreads) rotary_kernel(const __grid_constant__ RotaryParams p) {
  extern __shared__ float2 turn[];  // [block_tokens][rotary_dim / 2]: cosine, sine
  __shared__ long long s_pos[kMaxBlockTokens];
  __shared__ int s_page[kMaxBlockTokens], s_seq[kMaxBlockTokens];
  const long long t0 = static_cast<long long>(blockIdx.x) * p.block_tokens;
  const int here = static_cast<int>(min(static_cast<long long>(p.block_tokens), p.total - t0));
  const int all = here * p.units;
  const int half_dim = p.rope.rotary_dim / 2;
  const bool append = p.positions == nullptr;
  const int slots = 1 << p.page_shift;

  for (int base = 0; base < all; base += kRotaryThreads * kUnroll) {
    Pack<T, V> a[kUnroll], b[kUnroll];
    int where[kUnroll], head[kUnroll];  // where: part | token << 2 | unit << 8
#pragma unroll
    for (int j = 0; j < kUnroll; ++j) {
      const int u = base + j * kRotaryThreads + static_cast<int>(threadIdx.x);
      where[j] = -1;
      if (u >= all) continue;
      const int tok = u / p.units;
      int rest = u - tok * p.units;
      int part = 0;
      if (p.parts > 1 && rest >= p.part[1].first_unit) part = 1;
      if (p.parts > 2 && rest >= p.part[2].first_unit) part = 2;
      const RotaryPart &q = p.part[part];
      rest -= q.first_unit;
      const int h = rest / q.units, k = rest - h * q.units;
      where[j] = part | tok << 2 | k << 8;
      head[j] = h;
      const long long t = t0 + tok;
      const long long z = append ? 0 : t / p.tokens;
      const T *src = static_cast<const T *>(q.in) + z * q.in_stride[0] + h * q.in_stride[1] + (t - z * p.tokens) * q.in_stride[2];
      if (k < q.turned) {
        const int c1 = p.rope.interleaved ? 2 * k * V : k * V;
        const int c2 = p.rope.interleaved ? c1 + V : c1 + half_dim;
        a[j] = *reinterpret_cast<const Pack<T, V> *>(src + c1);
        b[j] = *reinterpret_cast<const Pack<T, V> *>(src + c2);
      } else {
        a[j] = *reinterpret_cast<const Pack<T, V> *>(src + (q.turned ? p.rope.rotary_dim : 0) + (k - q.turned) * V);
      }
    }
    if (base == 0) {
      if (append) {
        // the sequence of each token, found by all threads at once; tokens behind the last sequence keep -1
        if (threadIdx.x < kMaxBlockTokens) s_seq[threadIdx.x] = -1;
        __syncthreads();
        if (p.cu_q) {
          for (int s = threadIdx.x; s < p.batch; s += kRotaryThreads) {
            const long long lo = p.cu_q[s], hi = p.cu_q[s + 1];
            for (int i = 0; i < here; ++i)
              if (t0 + i >= lo && t0 + i < hi) s_seq[i] = s;
          }
        } else if (threadIdx.x < here) {
          s_seq[threadIdx.x] = t0 + threadIdx.x < p.batch ? static_cast<int>(t0 + threadIdx.x) : -1;
        }
        __syncthreads();
        if (threadIdx.x < here) {
          const int s = s_seq[threadIdx.x];
          int page = -1;
          if (s >= 0) {
            const long long t = t0 + threadIdx.x;
            const long long pos = p.cu_q ? p.kv_lens[s] - (p.cu_q[s + 1] - t) : p.kv_lens[s] - 1;
            s_pos[threadIdx.x] = pos;
            if (pos < 0) {
              atomicOr(p.status, kBadLength);
            } else if ((pos >> p.page_shift) >= p.table_width) {
              atomicOr(p.status, kNoRoomInRow);
            } else {
              page = p.table[s * p.table_stride + (pos >> p.page_shift)];
              if (page < 0 || page >= p.num_pages) {
                atomicOr(p.status, kBadPage);
                page = -1;
              }
            }
          } else {
            s_pos[threadIdx.x] = 0;
          }
          s_page[threadIdx.x] = page;
        }
      } else if (threadIdx.x < here) {
        const long long t = t0 + threadIdx.x, z = t / p.tokens;
        const long long at = z * p.position_stride[0] + (t - z * p.tokens) * p.position_stride[1];
        s_pos[threadIdx.x] = p.positions_64 ? static_cast<const long long *>(p.positions)[at]
                                            : static_cast<long long>(static_cast<const int32_t *>(p.positions)[at]);
      }
      __syncthreads();
      for (int i = threadIdx.x; i < here * half_dim; i += kRotaryThreads) {
        const int tok = i / half_dim, pair = i - tok * half_dim;
        const unsigned long long angle = static_cast<unsigned long long>(s_pos[tok]) * p.rope.turns[pair];
        float s, c;
        sincospif(static_cast<float>(static_cast<int32_t>(angle >> 32)) * 0x1p-31f, &s, &c);
        turn[i] = make_float2(c * p.rope.magnitude, (p.inverse ? -s : s) * p.rope.magnitude);
      }
      __syncthreads();
    }
#pragma unroll
    for (int j = 0; j < kUnroll; ++j) {
      if (where[j] < 0) continue;
      const int part = where[j] & 3, tok = (where[j] >> 2) & 63, k = where[j] >> 8;
      const RotaryPart &q = p.part[part];
      T *dst = static_cast<T *>(q.out);
      const long long t = t0 + tok;
      if (q.kind == kTurn) {
        if (append && s_seq[tok] < 0) continue;
        const long long z = append ? 0 : t / p.tokens;
        dst += z * q.out_stride[0] + head[j] * q.out_stride[1] + (t - z * p.tokens) * q.out_stride[2];
      } else {
        if (s_page[tok] < 0) continue;
        dst += s_page[tok] * q.out_stride[0] + (s_pos[tok] & (slots - 1)) * q.out_stride[1] + head[j] * q.out_stride[2];
      }
      if (k < q.turned) {
        const int c1 = p.rope.interleaved ? 2 * k * V : k * V;
        const int c2 = p.rope.interleaved ? c1 + V : c1 + half_dim;
        const float2 *cs = turn + tok * half_dim + k * V;
        T flat[2 * V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
          flat[i] = a[j].x[i];
          flat[V + i] = b[j].x[i];
        }
        if (p.rope.interleaved) {
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const float x1 = rot_f32(flat[2 * i]), x2 = rot_f32(flat[2 * i + 1]);
            flat[2 * i] = rot_from<T>(x1 * cs[i].x - x2 * cs[i].y);
            flat[2 * i + 1] = rot_from<T>(x2 * cs[i].x + x1 * cs[i].y);
          }
        } else {
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const float x1 = rot_f32(flat[i]), x2 = rot_f32(flat[V + i]);
            flat[i] = rot_from<T>(x1 * cs[i].x - x2 * cs[i].y);
            flat[V + i] = rot_from<T>(x2 * cs[i].x + x1 * cs[i].y);
          }
        }
#pragma unroll
        for (int i = 0; i < V; ++i) {
          a[j].x[i] = flat[i];
          b[j].x[i] = flat[V + i];
        }
        *reinterpret_cast<Pack<T, V> *>(dst + c1) = a[j];
        *reinterpret_cast<Pack<T, V> *>(dst + c2) = b[j];
      } else {
        *reinterpret_cast<Pack<T, V> *>(dst + (q.turned ? p.rope.rotary_dim : 0) + (k - q.turned) * V) = a[j];
      }
    }
  }
}

}  // namespace txp
