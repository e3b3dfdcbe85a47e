// Attention of whole prompts: packed sequences of different lengths, grouped
// query heads, causal.
//
//   s_ij = scale q_i . k_j,  j <= i + (len_k - len_q) when causal,
//   out_i = sum_j exp(s_ij - m_i) v_j / sum_j exp(s_ij - m_i),  m_i = max_j s_ij
//
// with row i of a sequence's len_q new tokens and key j of its len_k tokens
// (len_k > len_q: the chunk follows an earlier context). A row without keys
// is zero. The maxima, sums and the output accumulate in fp32.
#include <cuda_bf16.h>

#include <algorithm>

#include "kq_internal.h"
#include "kq_device.cuh"

namespace kq {
namespace {

__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void store_f(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void store_f(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// Sequence that owns packed row i: the last b with cu[b] <= i (empty ones
// before it share that start and come earlier).
__device__ __forceinline__ int find_seq(const int32_t* cu, int B, long long i) {
  int lo = 0, hi = B;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid] <= i) lo = mid;
    else hi = mid;
  }
  return lo;
}

// ---- any shape: one warp per (row, query head) ----------------------------------
// 32 keys per step, one per lane for q . k (q in shared memory as fp32), then
// the lanes own output dimensions for p . v. Bound by its scalar loads and
// FMAs; it serves the head sizes and strides that the tensor-core kernel
// does not take.
constexpr int kSimpleWarps = 4;
constexpr int kMaxD = 256;

template <typename T>
__global__ void __launch_bounds__(kSimpleWarps * 32) fa_prompt_simple_kernel(const FaPromptArgs a) {
  __shared__ float s_q[kSimpleWarps][kMaxD];
  __shared__ float s_p[kSimpleWarps][32];
  const unsigned full = 0xffffffffu;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long item = (long long)blockIdx.x * kSimpleWarps + warp;
  if (item >= (long long)a.Tq * a.Hq) return;
  const long long row = item / a.Hq;
  const int h = (int)(item % a.Hq), kh = h / (a.Hq / a.Hkv);
  const int b = find_seq(a.cu_q, a.B, row);
  T* out = static_cast<T*>(a.out) + (row * a.Hq + h) * a.D;
  const int q0 = a.cu_q[b], lq = a.cu_q[b + 1] - q0, k0 = a.cu_k[b], lk = a.cu_k[b + 1] - k0;
  const int i = (int)(row - q0);
  const int keys = i >= lq || i < 0 ? 0 : a.causal ? max(0, min(lk, i + lk - lq + 1)) : lk;
  const T* q = static_cast<const T*>(a.q) + row * a.q_row + (long long)h * a.q_head;
  const T* kb = static_cast<const T*>(a.k) + (long long)k0 * a.k_row + (long long)kh * a.k_head;
  const T* vb = static_cast<const T*>(a.v) + (long long)k0 * a.v_row + (long long)kh * a.v_head;
  for (int d = lane; d < a.D; d += 32) s_q[warp][d] = to_f(q[d]) * a.scale;
  __syncwarp();
  float m = -INFINITY, l = 0.0f, acc[kMaxD / 32];
#pragma unroll
  for (int t = 0; t < kMaxD / 32; ++t) acc[t] = 0.0f;
  for (int j0 = 0; j0 < keys; j0 += 32) {
    const int j = j0 + lane;
    float s = -INFINITY;
    if (j < keys) {
      const T* k = kb + (long long)j * a.k_row;
      float dot = 0.0f;
      for (int d = 0; d < a.D; ++d) dot = fmaf(s_q[warp][d], to_f(k[d]), dot);
      s = dot;
    }
    const float mn = fmaxf(m, warp_max(s));
    // all keys so far at -inf: no weight yet (and no inf - inf)
    const float base = mn == -INFINITY ? 0.0f : mn;
    const float p = __expf(s - base);
    const float c = __expf(m - base);
    float ps = p;
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) ps += __shfl_xor_sync(full, ps, o);
    l = l * c + ps;
    m = mn;
    s_p[warp][lane] = p;
    __syncwarp();
#pragma unroll
    for (int t = 0; t < kMaxD / 32; ++t) acc[t] *= c;
    const int n = min(32, keys - j0);
    for (int jj = 0; jj < n; ++jj) {
      const float pj = s_p[warp][jj];
      const T* v = vb + (long long)(j0 + jj) * a.v_row;
#pragma unroll
      for (int t = 0; t < kMaxD / 32; ++t) {
        const int d = lane + 32 * t;
        if (d < a.D) acc[t] = fmaf(pj, to_f(v[d]), acc[t]);
      }
    }
    __syncwarp();
  }
  const float inv = l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l);  // NaN stays NaN
#pragma unroll
  for (int t = 0; t < kMaxD / 32; ++t) {
    const int d = lane + 32 * t;
    if (d < a.D) store_f(out + d, acc[t] * inv);
  }
}

}  // namespace

size_t fa_prompt_workspace(const FaPromptArgs&) { return 0; }

kq_status_t launch_fa_prompt(const FaPromptArgs& a, int dtype, cudaStream_t s) {
  const long long items = (long long)a.Tq * a.Hq;
  const unsigned grid = (unsigned)((items + kSimpleWarps - 1) / kSimpleWarps);
  if (dtype == KQ_F16) fa_prompt_simple_kernel<__half><<<grid, kSimpleWarps * 32, 0, s>>>(a);
  else fa_prompt_simple_kernel<__nv_bfloat16><<<grid, kSimpleWarps * 32, 0, s>>>(a);
  return check_launch("fa_prompt");
}

}  // namespace kq
