// Packed and paged attention for any head dimension up to 256, any strides and any page
// size: one warp per (query row, head), CUDA cores, fp32 arithmetic.
//
//   O = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),  s_j = scale q . k_j,  m = max_j s_j,
// over the keys the row sees, in one pass with the running maximum and sum. A row that
// sees no key gives zeros; rows that belong to no request are left as they were.
//
// It serves what the tensor-core kernels do not take (head dimensions other than 64 and
// 128, rows that are not 16-byte aligned, page sizes that do not fit a copy box), so it is
// written for coverage: it is bound by the warp reductions, 5 shuffles per key and row.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "attn_params.cuh"

namespace {

using namespace tb;

__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ void store_as(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }
__device__ __forceinline__ void store_as(__half* p, float x) { *p = __float2half_rn(x); }

template <typename T>
__device__ __forceinline__ void attention_rows(const AttnParams& p) {
  begin_after_earlier_grids();
  const int lane = threadIdx.x & 31;
  const int* cu_q = reinterpret_cast<const int*>(p.cu_q);
  const long long units = (long long)p.tq * p.heads;
  const long long step = (long long)gridDim.x * (blockDim.x >> 5);
  for (long long u = (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); u < units; u += step) {
    const int t = (int)(u / p.heads), h = (int)(u % p.heads);
    // The last request that starts at or before row t.
    int lo = 0, hi = p.batch;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (load_index(cu_q + mid) <= t) lo = mid + 1;
      else hi = mid;
    }
    if (lo == 0) continue;
    const int b = lo - 1;
    const AttnRequest r = request_of(p, b);
    if (t < r.q0 || t >= r.q0 + r.lq || is_token_request(p, r)) continue;
    const int n = visible_keys(p, r, t - r.q0);
    const int hk = h / (p.heads / p.kv_heads);
    const T* q = reinterpret_cast<const T*>(p.q) + t * p.q_tok + h * p.q_head;
    float qv[8], acc[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int d = lane + 32 * j;
      qv[j] = d < p.dim ? to_f32(q[d]) : 0.f;
      acc[j] = 0.f;
    }
    float m = -3.402823466e38f, l = 0.f;  // a finite start: a score of -inf then weighs exp(-inf) = 0
    for (int key = 0; key < n; ++key) {
      const T *k = nullptr, *v = nullptr;
      if (p.table) {
        const int id = page_of(p, b, key / p.page);
        if (id >= 0) {
          k = reinterpret_cast<const T*>(p.k) + id * p.k_page + (key % p.page) * p.k_tok + hk * p.k_head;
          v = reinterpret_cast<const T*>(p.v) + id * p.v_page + (key % p.page) * p.v_tok + hk * p.v_head;
        }
      } else {
        k = reinterpret_cast<const T*>(p.k) + (r.k0 + key) * p.k_tok + hk * p.k_head;
        v = reinterpret_cast<const T*>(p.v) + (r.k0 + key) * p.v_tok + hk * p.v_head;
      }
      float part = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int d = lane + 32 * j;
        if (k && d < p.dim) part = fmaf(qv[j], to_f32(k[d]), part);
      }
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) part += __shfl_xor_sync(0xffffffffu, part, off);
      const float s = part * p.scale;
      const float top = fmaxf(m, s);
      const float old = expf(m - top), w = expf(s - top);
      l = l * old + w;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int d = lane + 32 * j;
        acc[j] *= old;
        if (v && d < p.dim) acc[j] = fmaf(w, to_f32(v[d]), acc[j]);
      }
      m = top;
    }
    const float inv = l == 0.f ? 0.f : 1.0f / l;
    T* o = reinterpret_cast<T*>(p.o) + t * p.o_tok + h * p.o_head;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int d = lane + 32 * j;
      if (d < p.dim) store_as(o + d, acc[j] * inv);
    }
  }
}

}  // namespace

extern "C" __global__ void __launch_bounds__(256) attention_rows_bf16(const __grid_constant__ tb::AttnParams p) {
  attention_rows<__nv_bfloat16>(p);
}
extern "C" __global__ void __launch_bounds__(256) attention_rows_f16(const __grid_constant__ tb::AttnParams p) {
  attention_rows<__half>(p);
}
