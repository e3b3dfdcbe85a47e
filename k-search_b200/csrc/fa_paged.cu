// Decode attention over the paged q8_0 cache for a batch whose sequences may
// share a prefix: one query token per sequence,
//
//   out[b, h] = softmax_j(scale q[b, h] . k_j) v_j,  j < seq_lens[b],
//
// token j of sequence b in page block_tables[b, j / page_size]; the first
// prefix_len tokens are the same pages for every sequence and are read
// through row 0 of the table. q8_0 values are d * code; the softmax state and
// the output accumulate in fp32. A sequence of length 0 yields zeros; a page
// id outside the cache hides its tokens.
#include <cuda_bf16.h>

#include <algorithm>

#include "kq_internal.h"
#include "kq_device.cuh"

namespace kq {
namespace {

constexpr int kQ8 = 34;
constexpr int kMaxNB = 8;

__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void store_f(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void store_f(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

// One warp per (sequence, query head), 32 tokens per step: a lane per token
// for q . k, then a lane per dimension for p . v.
constexpr int kWarps = 4;

template <typename T>
__global__ void __launch_bounds__(kWarps * 32) fa_paged_simple_kernel(const FaPagedArgs a) {
  __shared__ float s_q[kWarps][kMaxNB * 32];
  __shared__ float s_p[kWarps][32];
  __shared__ long long s_row[kWarps][32];
  const unsigned full = 0xffffffffu;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long item = (long long)blockIdx.x * kWarps + warp;
  if (item >= (long long)a.B * a.Hq) return;
  const int b = (int)(item / a.Hq), h = (int)(item % a.Hq), kh = h / (a.Hq / a.Hkv);
  const int nb = a.D / 32;
  const long long row_bytes = (long long)a.Hkv * nb * kQ8;
  const int len = (int)min((long long)max(0, min(a.seq_lens[b], a.max_seqlen)), (long long)a.W * a.ps);
  const T* q = static_cast<const T*>(a.q) + ((long long)b * a.Hq + h) * a.D;
  for (int d = lane; d < a.D; d += 32) s_q[warp][d] = to_f(q[d]) * a.scale;
  __syncwarp();
  float m = -INFINITY, l = 0.0f, acc[kMaxNB];
#pragma unroll
  for (int t = 0; t < kMaxNB; ++t) acc[t] = 0.0f;
  for (int j0 = 0; j0 < len; j0 += 32) {
    const int j = j0 + lane;
    float s = -INFINITY;
    long long off = -1;
    if (j < len) {
      const long long page = a.table[(long long)(j < a.prefix_len ? 0 : b) * a.W + j / a.ps];
      if (page >= 0 && page < a.num_pages) {
        off = (page * a.ps + j % a.ps) * row_bytes + (long long)kh * nb * kQ8;
        const uint8_t* k = a.k + off;
        s = 0.0f;
        for (int t = 0; t < nb; ++t) {
          const float d = half_bits_to_float(*reinterpret_cast<const uint16_t*>(k + t * kQ8));
          float dot = 0.0f;
          for (int e = 0; e < 32; ++e) dot = fmaf(s_q[warp][t * 32 + e], (float)(int8_t)k[t * kQ8 + 2 + e], dot);
          s = fmaf(d, dot, s);
        }
      }
    }
    const float mn = fmaxf(m, warp_max(s));
    const float base = mn == -INFINITY ? 0.0f : mn;
    const float p = off < 0 ? 0.0f : __expf(s - base);
    const float c = __expf(m - base);
    float ps = p;
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) ps += __shfl_xor_sync(full, ps, o);
    l = l * c + ps;
    m = mn;
    s_p[warp][lane] = p;
    s_row[warp][lane] = off;
    __syncwarp();
#pragma unroll
    for (int t = 0; t < kMaxNB; ++t) acc[t] *= c;
    const int n = min(32, len - j0);
    for (int jj = 0; jj < n; ++jj) {
      if (s_row[warp][jj] < 0) continue;
      const float pj = s_p[warp][jj];
      const uint8_t* v = a.v + s_row[warp][jj];
#pragma unroll
      for (int t = 0; t < kMaxNB; ++t)
        if (t < nb) {
          const float d = half_bits_to_float(*reinterpret_cast<const uint16_t*>(v + t * kQ8));
          acc[t] = fmaf(pj * d, (float)(int8_t)v[t * kQ8 + 2 + lane], acc[t]);
        }
    }
    __syncwarp();
  }
  T* out = static_cast<T*>(a.out) + ((long long)b * a.Hq + h) * a.D;
  const float inv = l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l);  // NaN stays NaN
#pragma unroll
  for (int t = 0; t < kMaxNB; ++t)
    if (t < nb) store_f(out + t * 32 + lane, acc[t] * inv);
}

}  // namespace

size_t fa_paged_workspace(const FaPagedArgs&) { return 0; }

kq_status_t launch_fa_paged(const FaPagedArgs& a, int dtype, cudaStream_t s) {
  const long long items = (long long)a.B * a.Hq;
  const unsigned grid = (unsigned)((items + kWarps - 1) / kWarps);
  if (dtype == KQ_F16) fa_paged_simple_kernel<__half><<<grid, kWarps * 32, 0, s>>>(a);
  else fa_paged_simple_kernel<__nv_bfloat16><<<grid, kWarps * 32, 0, s>>>(a);
  return check_launch("fa_paged");
}

}  // namespace kq
