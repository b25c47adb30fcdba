// Attention of a ragged batch of new tokens over a paged key/value cache.
//
// Query i of request r (n new tokens, c keys in all) stands at position p = c - n + i and sees the keys 0 .. p, with a window those
// from p - left on and the first `sink`:  o = softmax(scale q K^T) V,  lse = log sum exp(scale q k).
//
// The plain kernel: a warp for each query head of a token, four head-dim elements per lane, running maximum and sum.
#include "host_common.cuh"
#include "paged_args.h"
#include "ptx.cuh"

namespace ua {

__device__ __forceinline__ float4 bf16x4(const __nv_bfloat16* p) {
  const uint2 u = *reinterpret_cast<const uint2*>(p);
  return make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xFFFF0000u), __uint_as_float(u.y << 16),
                     __uint_as_float(u.y & 0xFFFF0000u));
}

__global__ void __launch_bounds__(256) attn_paged_plain_kernel(const __grid_constant__ UaPagedAttn a, float scale, int* status) {
  grid_wait();
  grid_trigger();
  const long row = static_cast<long>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  const long tok = row / a.heads, head = row % a.heads;
  if (tok >= a.tokens || tok >= a.cu_new[a.requests]) return;
  int lo = 0, hi = static_cast<int>(a.requests);
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a.cu_new[mid] <= tok) lo = mid;
    else hi = mid;
  }
  const int r = lo, first = a.cu_new[r], n = a.cu_new[r + 1] - first, c = a.context[r];
  const int pos = c - n + static_cast<int>(tok - first);
  const long kvh = head / (a.heads / a.kv_heads);
  const float4 q = bf16x4(static_cast<const __nv_bfloat16*>(a.q) + tok * a.q_token + head * a.q_head + lane * 4);
  float m = -INFINITY, l = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int j = 0; j <= pos; ++j) {
    if (a.left >= 0 && j < pos - a.left && j >= a.sink) j = static_cast<int>(pos - a.left);
    const long col = j >> a.page_shift, off = j & ((1 << a.page_shift) - 1);
    const int page = col < a.columns ? a.table[r * a.table_stride + col] : -1;
    if (page < 0 || page >= a.pages) {
      if (lane == 0 && atomicCAS(status, 0, UA_ERR_BAD_ARG) == 0) {
        status[1] = 520;
        status[2] = r;
        status[3] = page;
      }
      continue;
    }
    const float4 k = bf16x4(static_cast<const __nv_bfloat16*>(a.k) + page * a.k_page + off * a.k_token + kvh * a.k_head + lane * 4);
    float s = q.x * k.x + q.y * k.y + q.z * k.z + q.w * k.w;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, d);
    s *= scale;
    const float mn = fmaxf(m, s), al = mn == -INFINITY ? 1.f : __expf(m - mn), w = mn == -INFINITY ? 0.f : __expf(s - mn);
    m = mn;
    l = l * al + w;
    const float4 v = bf16x4(static_cast<const __nv_bfloat16*>(a.v) + page * a.v_page + off * a.v_token + kvh * a.v_head + lane * 4);
    acc.x = acc.x * al + w * v.x;
    acc.y = acc.y * al + w * v.y;
    acc.z = acc.z * al + w * v.z;
    acc.w = acc.w * al + w * v.w;
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
  uint2 o;
  o.x = pack_bf16x2(acc.x * inv, acc.y * inv);
  o.y = pack_bf16x2(acc.z * inv, acc.w * inv);
  *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(a.o) + tok * a.o_token + head * a.o_head + lane * 4) = o;
  if (lane == 0) a.lse[head * a.lse_head + tok] = l > 0.f ? m + __logf(l) : -INFINITY;
}

}  // namespace ua

using namespace ua;

extern "C" int ua_attn_paged(const UaPagedAttn* a, float softmax_scale, int* status, cudaStream_t stream) {
  if (a->tokens <= 0 || a->requests <= 0) return 0;
  if (a->kv_heads <= 0 || a->heads % a->kv_heads != 0)
    UA_FAIL("ua_attn_paged: %ld query heads do not divide into %ld key/value heads", a->heads, a->kv_heads);
  const uintptr_t bases = reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->k) | reinterpret_cast<uintptr_t>(a->v) |
                          reinterpret_cast<uintptr_t>(a->o);
  const long strides = a->q_token | a->q_head | a->k_page | a->k_token | a->k_head | a->v_page | a->v_token | a->v_head | a->o_token | a->o_head;
  if (bases % 16 != 0 || strides % 8 != 0) UA_FAIL("ua_attn_paged: rows of q, o and the cache must start on 16 bytes");
  const unsigned grid = static_cast<unsigned>((a->tokens * a->heads + 7) / 8);
  UA_CUDA(launch_kernel(attn_paged_plain_kernel, grid, 256, 0, stream, true, *a, softmax_scale, status));
  return 0;
}
