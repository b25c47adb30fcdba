// Rotary position embedding, and its form that writes keys and values into a paged cache.
//
// A pair (a, b) of a head's elements at position p is turned by the angle p f of its pair and scaled:
//   a' = m (a cos - b sin), b' = m (b cos + a sin);   backward: the same with -sin (the transpose).
// Pairs are (i, i + rot / 2) or, interleaved, (2 i, 2 i + 1) of the first `rot` elements of a head; the others are copied.
//
// The angle. p f in fp32 is off by 0.03 rad at position 500k (half a step of 2^19), and 64-bit sines for every token cost more than
// the rotation. But only the fraction of a turn matters: t = f / 2 pi is held as a 64-bit fraction, p t is an integer
// product whose overflow drops the whole turns, and what is left is split into quarters of a turn and a rest of at most an eighth,
// whose sine and cosine are good to fp32 (the rest is exact to 2^-32 turns). No table, no largest position; the 64
// angles of a token are found once per block and shared by its heads.
//
// Bound by memory: every element is read and written once.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "host_common.cuh"
#include "paged_args.h"
#include "ptx.cuh"

namespace ua {

constexpr int ROT_THREADS = 256;
constexpr int ROT_MAX_PAIRS = 256;     // rotated elements of a head: 512 at most
constexpr int ROT_MAX_TOKENS = 8;      // tokens of a block

struct RotParams {
  UaRotPart part[3];
  int n_parts;
  long tokens;            // of the whole batch
  int per_batch;          // tokens of a sequence
  const void* pos;
  int pos64;
  long pos_batch, pos_token;
  const int* slots;       // paged parts: page * page size + offset, negative: nothing is written
  int page_shift;
  long n_slots;
  const double* inv_freq; // [pairs]
  int pairs, dim;
  float magnitude;
  int inverse;
  int block_tokens;       // tokens of a block
  int* status;
};

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
template <typename T> __device__ __forceinline__ T from_f(float x);
template <> __device__ __forceinline__ float from_f<float>(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ __half from_f<__half>(float x) { return __float2half_rn(x); }

template <typename T, int V>
struct alignas(sizeof(T) * V) Vec {
  T v[V];
};

// cos and sin of position * (turns / 2^64) turns, times m
__device__ __forceinline__ float2 turn_of(long pos, unsigned long long turns, float m) {
  const unsigned hi = static_cast<unsigned>((static_cast<unsigned long long>(pos) * turns) >> 32);
  const unsigned quarter = (hi + 0x20000000u) >> 30;
  const int rest = static_cast<int>(hi - (quarter << 30));            // [-2^29, 2^29): an eighth of a turn either way
  float s, c;
  sincospif(static_cast<float>(rest) * 4.656612873077393e-10f, &s, &c);   // 2^-31: half turns
  s *= m;
  c *= m;
  switch (quarter & 3) {
    case 0: return make_float2(c, s);
    case 1: return make_float2(-s, c);
    case 2: return make_float2(-c, -s);
    default: return make_float2(s, -c);
  }
}

// V: elements per load and store (one otherwise); a unit is V elements of each half of the pairs (interleaved: V pairs' worth,
// 2 elements at least), or V elements that are copied.
template <typename T, int V, bool INTERLEAVED>
__global__ void __launch_bounds__(ROT_THREADS) rotary_kernel(const __grid_constant__ RotParams p) {
  __shared__ float2 cs[ROT_MAX_TOKENS * ROT_MAX_PAIRS];
  __shared__ long dst_off[ROT_MAX_TOKENS];       // of a token in its pages; negative: none
  grid_wait();
  grid_trigger();
  const long tok0 = static_cast<long>(blockIdx.x) * p.block_tokens;
  const int here = static_cast<int>(min(static_cast<long>(p.block_tokens), p.tokens - tok0));
  auto pos_of = [&](long t) -> long {
    const long i = t / p.per_batch * p.pos_batch + t % p.per_batch * p.pos_token;
    return p.pos64 ? static_cast<const long*>(p.pos)[i] : static_cast<const int*>(p.pos)[i];
  };
  if (p.pairs > 0) {
    for (int i = threadIdx.x; i < here * p.pairs; i += ROT_THREADS) {
      const int t = i / p.pairs, f = i % p.pairs;
      double turns = p.inv_freq[f] * 0.15915494309189535;                  // 1 / 2 pi
      turns -= floor(turns);
      const float2 v = turn_of(pos_of(tok0 + t), __double2ull_rn(turns * 18446744073709551616.0), p.magnitude);
      cs[i] = make_float2(v.x, p.inverse ? -v.y : v.y);
    }
  }
  if (p.slots != nullptr && threadIdx.x < here) {
    const int slot = p.slots[tok0 + threadIdx.x];
    if (slot >= p.n_slots && atomicCAS(p.status, 0, UA_ERR_BAD_ARG) == 0) {
      p.status[1] = 500;
      p.status[2] = static_cast<int>(blockIdx.x);
      p.status[3] = slot;
    }
    dst_off[threadIdx.x] = slot >= p.n_slots ? -1 : slot;
  }
  __syncthreads();
  constexpr int E = INTERLEAVED && V == 1 ? 2 : V;                           // elements of a unit of one half, or of pairs
  const int rot = 2 * p.pairs;
  const int rot_units = INTERLEAVED ? rot / E : p.pairs / E;
  const int units = rot_units + (p.dim - rot + V - 1) / V;
#pragma unroll 1
  for (int ip = 0; ip < p.n_parts; ++ip) {
    const UaRotPart& q = p.part[ip];
    const int per_token = q.heads * (q.rotate ? units : p.dim / V);
    const T* src0 = static_cast<const T*>(q.src);
    T* dst0 = static_cast<T*>(q.dst);
#pragma unroll 2
    for (int i = threadIdx.x; i < here * per_token; i += ROT_THREADS) {
      const int t = i / per_token, in = i % per_token;
      const int per_head = per_token / q.heads;
      const int head = in / per_head;
      int u = in % per_head;
      const long tok = tok0 + t, b = tok / p.per_batch, s = tok % p.per_batch;
      const T* src = src0 + b * q.src_batch + s * q.src_token + head * q.src_head;
      T* dst = dst0 + head * q.dst_head;
      if (q.paged) {
        const long slot = dst_off[t];
        if (slot < 0) continue;
        dst += (slot >> p.page_shift) * q.dst_batch + (slot & ((1 << p.page_shift) - 1)) * q.dst_token;
      } else {
        dst += b * q.dst_batch + s * q.dst_token;
      }
      if (!q.rotate || u >= rot_units) {
        const int e = q.rotate ? rot + (u - rot_units) * V : u * V;
        *reinterpret_cast<Vec<T, V>*>(dst + e) = *reinterpret_cast<const Vec<T, V>*>(src + e);
        continue;
      }
      const float2* w = cs + t * p.pairs;
      if constexpr (INTERLEAVED) {
        float x[E];
        if constexpr (V > 1) {
          const Vec<T, V> v = *reinterpret_cast<const Vec<T, V>*>(src + u * V);
#pragma unroll
          for (int k = 0; k < V; ++k) x[k] = to_f(v.v[k]);
        } else {
          x[0] = to_f(src[u * 2]);
          x[1] = to_f(src[u * 2 + 1]);
        }
        float y[E];
#pragma unroll
        for (int k = 0; k < E; k += 2) {
          const float2 c = w[u * (E / 2) + k / 2];
          y[k] = x[k] * c.x - x[k + 1] * c.y;
          y[k + 1] = x[k + 1] * c.x + x[k] * c.y;
        }
        if constexpr (V > 1) {
          Vec<T, V> o;
#pragma unroll
          for (int k = 0; k < V; ++k) o.v[k] = from_f<T>(y[k]);
          *reinterpret_cast<Vec<T, V>*>(dst + u * V) = o;
        } else {
          dst[u * 2] = from_f<T>(y[0]);
          dst[u * 2 + 1] = from_f<T>(y[1]);
        }
      } else {
        const Vec<T, V> lo = *reinterpret_cast<const Vec<T, V>*>(src + u * V);
        const Vec<T, V> hi = *reinterpret_cast<const Vec<T, V>*>(src + p.pairs + u * V);
        Vec<T, V> a, b2;
#pragma unroll
        for (int k = 0; k < V; ++k) {
          const float2 c = w[u * V + k];
          const float x = to_f(lo.v[k]), y = to_f(hi.v[k]);
          a.v[k] = from_f<T>(x * c.x - y * c.y);
          b2.v[k] = from_f<T>(y * c.x + x * c.y);
        }
        *reinterpret_cast<Vec<T, V>*>(dst + u * V) = a;
        *reinterpret_cast<Vec<T, V>*>(dst + p.pairs + u * V) = b2;
      }
    }
  }
}

template <typename T, bool INTERLEAVED>
static int launch_rotary(const RotParams& p, bool wide, unsigned grid, cudaStream_t stream) {
  constexpr int V = 16 / sizeof(T);
  if (wide) UA_CUDA(launch_kernel(rotary_kernel<T, V, INTERLEAVED>, grid, ROT_THREADS, 0, stream, true, p));
  else UA_CUDA(launch_kernel(rotary_kernel<T, 1, INTERLEAVED>, grid, ROT_THREADS, 0, stream, true, p));
  return 0;
}

}  // namespace ua

using namespace ua;

extern "C" int ua_rotary(const UaRotary* a, float magnitude, int* status, cudaStream_t stream) {
  const int size = a->dtype == 2 ? 4 : 2, V = 16 / size;
  if (a->n_parts < 0 || a->n_parts > 3) UA_FAIL("ua_rotary: %ld tensors (3 at most)", a->n_parts);
  if (a->pairs < 0 || a->pairs > ROT_MAX_PAIRS || 2 * a->pairs > a->dim)
    UA_FAIL("ua_rotary: %ld pairs in heads of %ld elements (%d pairs at most)", a->pairs, a->dim, ROT_MAX_PAIRS);
  if (a->batch <= 0 || a->per_batch <= 0) return 0;
  RotParams p;
  memset(&p, 0, sizeof(p));
  // 16 bytes at a time where every row of every tensor starts on 16 bytes and the parts of a head are whole vectors
  bool wide = a->dim % V == 0 && (a->interleaved ? 2 * a->pairs : a->pairs) % V == 0;
  for (int i = 0; i < a->n_parts; ++i) {
    const UaRotPart& q = p.part[i] = a->part[i];
    const long strides = q.src_batch | q.src_token | q.src_head | q.dst_batch | q.dst_token | q.dst_head;
    wide = wide && strides % V == 0 && ((reinterpret_cast<uintptr_t>(q.src) | reinterpret_cast<uintptr_t>(q.dst)) & 15) == 0;
  }
  p.n_parts = static_cast<int>(a->n_parts);
  p.tokens = a->batch * a->per_batch;
  p.per_batch = static_cast<int>(a->per_batch);
  p.pos = a->pos;
  p.pos64 = static_cast<int>(a->pos64);
  p.pos_batch = a->pos_batch;
  p.pos_token = a->pos_token;
  p.slots = a->slots;
  p.page_shift = static_cast<int>(a->page_shift);
  p.n_slots = a->n_slots;
  p.inv_freq = a->inv_freq;
  p.pairs = static_cast<int>(a->pairs);
  p.dim = static_cast<int>(a->dim);
  p.magnitude = magnitude;
  p.inverse = static_cast<int>(a->inverse);
  p.status = status;
  p.block_tokens = 1;
  const unsigned grid = static_cast<unsigned>((p.tokens + p.block_tokens - 1) / p.block_tokens);
  switch (a->dtype * 2 + (a->interleaved ? 1 : 0)) {
    case 0: return launch_rotary<__nv_bfloat16, false>(p, wide, grid, stream);
    case 1: return launch_rotary<__nv_bfloat16, true>(p, wide, grid, stream);
    case 2: return launch_rotary<__half, false>(p, wide, grid, stream);
    case 3: return launch_rotary<__half, true>(p, wide, grid, stream);
    case 4: return launch_rotary<float, false>(p, wide, grid, stream);
    case 5: return launch_rotary<float, true>(p, wide, grid, stream);
  }
  UA_FAIL("ua_rotary: unknown type %ld", a->dtype);
}
