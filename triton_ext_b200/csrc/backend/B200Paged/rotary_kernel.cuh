// Rotary positions, and the append of new tokens to a paged cache.
//
// Pair i of a head is the complex number x1 + i x2; a position p turns it by the angle 2 pi p f_i, where f_i is kept as
// a 64-bit fraction of a turn. p * f_i in 64-bit wrap-around arithmetic IS the angle modulo whole turns, so no range
// reduction loses anything at far positions (a product in fp32 is off by 0.06 rad at position 2^20 already); its upper
// 32 bits go through sincospi. What is left is f_i's own rounding, p 2^-65 of a turn: less than the cut to 32 bits up to
// position 2^32, 2^-25 of a turn at 2^40.
//
// The work is one read and one write of every value: HBM bound when there are many tokens, launch bound when there are
// few. A warp takes one token (a slice of its heads when there are few tokens): its lanes are the vectors of a head, by as
// many heads as fit 32 lanes, and step over the rest, so a lane keeps the cosines and sines of its V pairs in registers for
// all heads. The warp computes each angle once and passes it on through its own piece of shared memory. Warps never wait for
// one another. (A block per few tokens with the angles in shared memory, two barriers apart from its loads,
// took 229 us for the training case, 4 x 4096 tokens of 40 heads
// of 128 bf16 forward and backward; this takes 111 us, 6.0 TB/s. An append of 8150 tokens of 32 + 2 x 8 heads: 35 us, 4.6 TB/s;
// what is missing there is the chain of loads from the token to its page.)
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "paged_host.h"
#include "sm100_ptx.cuh"

namespace txp {

constexpr int kRotaryThreads = 128;
constexpr int kUnroll = 2;  // heads whose vectors a lane has in flight

enum RotaryKind : int32_t { kTurn = 0, kTurnToPage = 1, kCopyToPage = 2 };

struct RotaryPart {
  const void *in;
  void *out;               // kTurn: the tensor; else the pool
  long long in_stride[3];  // batch, head, token
  long long out_stride[3]; // kTurn: batch, head, token; else page, slot, head
  int32_t kind, heads;
  int32_t pass;            // vectors of a head behind the turned columns that have to be copied
  int32_t lanes_shift;     // log2 of the lanes that one head takes (at most 5)
};

struct RotaryParams {
  tx_rope rope;
  RotaryPart part[3];
  const void *positions;   // NULL in an append
  long long position_stride[2];
  const int32_t *table, *kv_lens, *cu_q;
  long long table_stride;
  uint32_t *status;
  uint32_t total;          // tokens of all batch entries
  uint32_t tokens, slices; // slices: warps that share a token's heads
  int32_t parts, turned;   // turned: pairs of vectors of a head
  int32_t positions_64, inverse;
  int32_t batch, table_width, num_pages, page_shift;
};

template <typename T, int V>
struct alignas(sizeof(T) * V) Pack {
  T x[V];
};

// Turns the V pairs in a and b by (c, s): pairs (a[e], b[e]), or neighbours of the sequence a, b when interleaved. 16-bit
// values are taken two to a word: with one value at a time, extracting and packing took more instructions than the rest
// (training case: 196 us, against 121).
template <typename T>
struct Word;
template <>
struct Word<__half> {
  static __device__ __forceinline__ float2 up(uint32_t w) { return __half22float2(*reinterpret_cast<__half2 *>(&w)); }
  static __device__ __forceinline__ uint32_t down(float x, float y) {
    __half2 h = __floats2half2_rn(x, y);
    return *reinterpret_cast<uint32_t *>(&h);
  }
  static __device__ __forceinline__ float one(__half x) { return __half2float(x); }
  static __device__ __forceinline__ __half back(float x) { return __float2half_rn(x); }
};
template <>
struct Word<__nv_bfloat16> {
  static __device__ __forceinline__ float2 up(uint32_t w) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
  static __device__ __forceinline__ uint32_t down(float x, float y) {
    __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    return *reinterpret_cast<uint32_t *>(&h);
  }
  static __device__ __forceinline__ float one(__nv_bfloat16 x) { return __bfloat162float(x); }
  static __device__ __forceinline__ __nv_bfloat16 back(float x) { return __float2bfloat16_rn(x); }
};
template <>
struct Word<float> {
  static __device__ __forceinline__ float one(float x) { return x; }
  static __device__ __forceinline__ float back(float x) { return x; }
};

template <typename T, int V>
__device__ __forceinline__ void turn_pairs(Pack<T, V> &a, Pack<T, V> &b, const float2 (&cs)[V], bool interleaved) {
  if constexpr (sizeof(T) == 2 && V > 1) {
    uint32_t (&x)[V / 2] = *reinterpret_cast<uint32_t (*)[V / 2]>(&a);
    uint32_t (&y)[V / 2] = *reinterpret_cast<uint32_t (*)[V / 2]>(&b);
    if (interleaved) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        uint32_t &w = i < V / 2 ? x[i] : y[i - V / 2];
        const float2 v = Word<T>::up(w);
        w = Word<T>::down(v.x * cs[i].x - v.y * cs[i].y, v.y * cs[i].x + v.x * cs[i].y);
      }
    } else {
#pragma unroll
      for (int i = 0; i < V / 2; ++i) {
        const float2 u = Word<T>::up(x[i]), v = Word<T>::up(y[i]), c0 = cs[2 * i], c1 = cs[2 * i + 1];
        x[i] = Word<T>::down(u.x * c0.x - v.x * c0.y, u.y * c1.x - v.y * c1.y);
        y[i] = Word<T>::down(v.x * c0.x + u.x * c0.y, v.y * c1.x + u.y * c1.y);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      T &first = !interleaved ? a.x[i] : 2 * i < V ? a.x[2 * i] : b.x[2 * i - V];
      T &second = !interleaved ? b.x[i] : 2 * i + 1 < V ? a.x[2 * i + 1] : b.x[2 * i + 1 - V];
      const float x1 = Word<T>::one(first), x2 = Word<T>::one(second);
      first = Word<T>::back(x1 * cs[i].x - x2 * cs[i].y);
      second = Word<T>::back(x2 * cs[i].x + x1 * cs[i].y);
    }
  }
}

// The last entry of cu[0 .. n] that is at most t, by 32 probes a step.
__device__ __forceinline__ int find_sequence(const int32_t *cu, int n, int t, int lane) {
  int lo = 0, left = n + 1;
  while (left > 1) {
    const int step = (left + 31) / 32;
    const int at = lo + lane * step;
    const uint32_t below = __ballot_sync(0xffffffffu, lane * step < left && cu[min(at, n)] <= t);
    const int hit = below ? 31 - __clz(below) : 0;
    lo += hit * step;
    left = min(step, left - hit * step);
  }
  return lo;
}

template <typename T, int V>
__global__ void __launch_bounds__(kRotaryThreads, 8) rotary_kernel(const __grid_constant__ RotaryParams p) {
  // cosine and sine of pair k * V + i at [i][k]: the lanes of a head read neighbouring banks
  __shared__ float2 s_turn[kRotaryThreads / 32][TX_ROPE_MAX_PAIRS];
  float2 *turn = s_turn[threadIdx.x >> 5];
  const int lane = threadIdx.x & 31;
  const uint32_t id = blockIdx.x * (kRotaryThreads / 32) + (threadIdx.x >> 5);
  const uint32_t t = p.slices == 1 ? id : id / p.slices;
  if (t >= p.total) return;
  txd::grid_dep_wait();
  txd::grid_dep_launch();  // an attention behind an append sets itself up meanwhile (a layer of one token over 500: 15.2 to 14.9 us)
  const int slice = static_cast<int>(id - t * p.slices);
  const bool append = p.positions == nullptr;
  // ---- the token's position, and where an append puts it ----
  long long pos, page = -1, z = 0, n = t;
  if (append) {
    if (id == 0 && p.cu_q) {  // one warp looks at all offsets
      bool bad = p.cu_q[0] < 0 || p.cu_q[p.batch] > static_cast<int>(p.total);
      for (int b = lane; b < p.batch; b += 32) bad |= p.cu_q[b + 1] < p.cu_q[b];
      if (bad) atomicOr(p.status, kBadOffsets);
    }
    const int s = p.cu_q ? find_sequence(p.cu_q, p.batch, static_cast<int>(t), lane) : static_cast<int>(t);
    if (s >= p.batch || (p.cu_q && p.cu_q[0] > static_cast<int>(t))) return;  // behind the last sequence
    pos = p.cu_q ? static_cast<long long>(p.kv_lens[s]) - (p.cu_q[s + 1] - static_cast<int>(t)) : p.kv_lens[s] - 1;
    uint32_t bad = 0;
    if (p.cu_q && (p.cu_q[s + 1] <= static_cast<int>(t) || p.cu_q[s + 1] > static_cast<int>(p.total))) {
      bad = kBadOffsets;  // which sequence the token belongs to, or where in it, is not known
    } else if (pos < 0) {
      bad = kBadLength;
    } else if ((pos >> p.page_shift) >= p.table_width) {
      bad = kNoRoomInRow;
    } else {
      page = p.table[s * p.table_stride + (pos >> p.page_shift)];
      if (page < 0 || page >= p.num_pages) bad = kBadPage, page = -1;
    }
    if (bad && lane == 0) atomicOr(p.status, bad);
  } else {
    z = t / p.tokens;
    n = t - static_cast<uint32_t>(z) * p.tokens;
    const long long at = z * p.position_stride[0] + n * p.position_stride[1];
    pos = p.positions_64 ? static_cast<const long long *>(p.positions)[at]
                         : static_cast<long long>(static_cast<const int32_t *>(p.positions)[at]);
  }
  const int slot = static_cast<int>(pos & ((1ll << p.page_shift) - 1));
  const int half_dim = p.rope.rotary_dim / 2;
  // read through a generic address: the lanes' words are neighbours, which the constant port would serve one after another
  // (121 us instead of 114 for the training case)
  const uint64_t *turns_at = p.rope.turns;
  asm volatile("" : "+l"(turns_at));
  for (int i = lane; i < half_dim; i += 32) {
    const unsigned long long angle = static_cast<unsigned long long>(pos) * turns_at[i];
    float c, s;
    sincospif(static_cast<float>(static_cast<int32_t>(angle >> 32)) * 0x1p-31f, &s, &c);
    turn[(i % V) * p.turned + i / V] = make_float2(c * p.rope.magnitude, (p.inverse ? -s : s) * p.rope.magnitude);
  }
  __syncwarp();

  for (int i = 0; i < p.parts; ++i) {
    const RotaryPart &q = p.part[i];
    if (q.kind != kTurn && page < 0) continue;
    const T *src = static_cast<const T *>(q.in) + z * q.in_stride[0] + n * q.in_stride[2];
    T *dst = static_cast<T *>(q.out);
    long long dst_head;
    if (q.kind == kTurn) {
      dst += z * q.out_stride[0] + n * q.out_stride[2];
      dst_head = q.out_stride[1];
    } else {
      dst += page * q.out_stride[0] + slot * q.out_stride[1];
      dst_head = q.out_stride[2];
    }
    const int turned = q.kind == kCopyToPage ? 0 : p.turned, from = q.kind == kCopyToPage ? 0 : p.rope.rotary_dim;
    const int lanes = 1 << q.lanes_shift, hl = lane >> q.lanes_shift, beside = 32 >> q.lanes_shift;
    for (int k0 = 0; k0 < turned + q.pass; k0 += lanes) {
      const int k = k0 + (lane & (lanes - 1));
      const bool turns = k < turned, active = k < turned + q.pass;
      float2 cs[V];
#pragma unroll
      for (int e = 0; e < V; ++e) cs[e] = turns ? turn[e * p.turned + k] : make_float2(1.f, 0.f);
      // ---- the heads ----
      const int c1 = turns ? (p.rope.interleaved ? 2 * k * V : k * V) : from + (k - turned) * V;
      const int c2 = p.rope.interleaved ? c1 + V : c1 + half_dim;
      const int step = static_cast<int>(p.slices) * beside;
      for (int h0 = slice * beside; h0 < q.heads; h0 += step * kUnroll) {
        Pack<T, V> a[kUnroll], b[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
          const int h = h0 + u * step + hl;
          if (active && h < q.heads) {
            const T *x = src + h * q.in_stride[1];
            a[u] = *reinterpret_cast<const Pack<T, V> *>(x + c1);
            if (turns) b[u] = *reinterpret_cast<const Pack<T, V> *>(x + c2);
          }
        }
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
          const int h = h0 + u * step + hl;
          if (!(active && h < q.heads)) continue;
          T *y = dst + h * dst_head;
          if (turns) {
            turn_pairs<T, V>(a[u], b[u], cs, p.rope.interleaved != 0);
            *reinterpret_cast<Pack<T, V> *>(y + c2) = b[u];
          }
          *reinterpret_cast<Pack<T, V> *>(y + c1) = a[u];
        }
      }
    }
  }
}

}  // namespace txp
