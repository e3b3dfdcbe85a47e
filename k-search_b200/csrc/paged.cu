// The paged q8_0 KV cache: block tables and slot maps from request lengths
// (page_plan), rows quantised into their pages (page_write), and rows read
// back in packed order (page_read).
//
// A cache is [num_pages, page_size, Hkv, D/32] q8_0 blocks (34 bytes: fp16 d,
// 32 int8 codes); token slot s = page * page_size + offset is one row of
// Hkv * D/32 blocks. Byte offsets are 64-bit throughout.
#include <cuda_bf16.h>

#include <algorithm>

#include "kq_internal.h"
#include "kq_device.cuh"

namespace kq {
namespace {

constexpr int kQ8 = 34;

// ---- page plan ---------------------------------------------------------------
// c = cached, n = new length of request b (negative counts as 0), W columns:
//   have = min(ceil(c / ps), W), need = min(ceil((c + n) / ps), W),
//   take = need - have, start = exclusive sum of take over requests,
//   table[b, have + i] = free[start + i]  (-1 past the end of the list),
//   slot of new token i of b: pos = c + i, page = table[b, pos / ps],
//   page * ps + pos % ps (-1 without a page).
// One launch: every CTA scans the lengths itself (a batch of kPlan requests
// at a time, in registers and shared memory) instead of waiting for another
// kernel's prefix sums, then takes its grid-stride share of the new pages and
// the new tokens, each found by binary search in the scans. The reads are a
// few KB from L2, so the repeated scan costs less than a second launch.
constexpr int kPlan = 512;

struct PlanArgs {
  const int32_t* cached;
  const int32_t* fresh;
  int B;
  int32_t* table;
  int W;
  const int32_t* free_pages;
  int F;
  int ps;
  long long T;
  long long* slots;
  int32_t* seq_lens;
  int32_t* cu_new;
  int32_t* cu_seqlens;
  int32_t* counts;
};

// Inclusive block scan of three values at once (kPlan threads).
__device__ __forceinline__ void scan3(int (&v)[3], int (*warp_sums)[3], int lane, int warp) {
  const unsigned full = 0xffffffffu;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      const int t = __shfl_up_sync(full, v[i], o);
      if (lane >= o) v[i] += t;
    }
  }
  if (lane == 31) {
#pragma unroll
    for (int i = 0; i < 3; ++i) warp_sums[warp][i] = v[i];
  }
  __syncthreads();
  if (warp == 0) {
    int s[3];
#pragma unroll
    for (int i = 0; i < 3; ++i) s[i] = lane < kPlan / 32 ? warp_sums[lane][i] : 0;
#pragma unroll
    for (int o = 1; o < kPlan / 32; o <<= 1) {
#pragma unroll
      for (int i = 0; i < 3; ++i) {
        const int t = __shfl_up_sync(full, s[i], o);
        if (lane >= o) s[i] += t;
      }
    }
    if (lane < kPlan / 32) {
#pragma unroll
      for (int i = 0; i < 3; ++i) warp_sums[lane][i] = s[i];
    }
  }
  __syncthreads();
  if (warp > 0) {
#pragma unroll
    for (int i = 0; i < 3; ++i) v[i] += warp_sums[warp - 1][i];
  }
}

// First r in [0, n) with ends[r] > x (ends non-decreasing, ends[n - 1] > x).
__device__ __forceinline__ int find_row(const int* ends, int n, int x) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (ends[mid] > x) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}

__global__ void __launch_bounds__(kPlan) page_plan_kernel(const PlanArgs a) {
  __shared__ int s_new_end[kPlan], s_take_end[kPlan];  // inclusive sums within the batch
  __shared__ int s_cached[kPlan], s_have[kPlan], s_take[kPlan], s_new[kPlan];
  __shared__ int s_warp[kPlan / 32][3];
  __shared__ unsigned long long s_placed;  // new tokens that got a slot (CTA 0)
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const bool lead = blockIdx.x == 0;
  int base_new = 0, base_take = 0, base_len = 0;  // sums over the earlier batches
  if (tid == 0) s_placed = 0;
  if (lead && tid == 0) {
    a.cu_new[0] = 0;
    a.cu_seqlens[0] = 0;
  }
  for (int b0 = 0; b0 < a.B; b0 += kPlan) {
    const int b = b0 + tid, rows = min(kPlan, a.B - b0);
    int c = 0, n = 0;
    if (b < a.B) {
      c = max(0, a.cached[b]);
      n = max(0, a.fresh[b]);
    }
    const int have = (int)min((long long)a.W, ((long long)c + a.ps - 1) / a.ps);
    const int need = (int)min((long long)a.W, ((long long)c + n + a.ps - 1) / a.ps);
    const int take = need - have;
    int sums[3] = {n, take, c + n};
    scan3(sums, s_warp, lane, warp);
    s_cached[tid] = c;
    s_new[tid] = n;
    s_have[tid] = have;
    s_take[tid] = take;
    s_new_end[tid] = sums[0];
    s_take_end[tid] = sums[1];
    if (lead && b < a.B) {
      a.seq_lens[b] = c + n;
      a.cu_new[b + 1] = base_new + sums[0];
      a.cu_seqlens[b + 1] = base_len + sums[2];
      // positions with a slot: up to the table's end, the free list's end and
      // the slot map's end; past a partly filled page that has no entry
      const int start = base_take + sums[1] - take;
      const int got = max(0, min(take, a.F - start));
      long long lo = c, hi = min((long long)c + n, ((long long)have + got) * a.ps);
      if (c % a.ps != 0 && c / a.ps < a.W && a.table[(long long)b * a.W + c / a.ps] < 0)
        lo = min(hi, (long long)have * a.ps);
      hi = min(hi, (long long)c + a.T - (base_new + sums[0] - n));
      if (hi > lo) atomicAdd(&s_placed, (unsigned long long)(hi - lo));  // integers: any order gives the same sum
    }
    __syncthreads();
    const int batch_new = s_new_end[kPlan - 1], batch_take = s_take_end[kPlan - 1];
    const int step = gridDim.x * kPlan;
    for (int i = blockIdx.x * kPlan + tid; i < batch_take; i += step) {
      const int r = find_row(s_take_end, rows, i);
      const int at = i - (s_take_end[r] - s_take[r]);
      const int idx = base_take + i;
      a.table[(long long)(b0 + r) * a.W + s_have[r] + at] = idx < a.F ? a.free_pages[idx] : -1;
    }
    const long long end = min((long long)batch_new, a.T - base_new);
    for (long long i = (long long)blockIdx.x * kPlan + tid; i < end; i += step) {
      const int r = find_row(s_new_end, rows, (int)i);
      const int pos = s_cached[r] + (int)i - (s_new_end[r] - s_new[r]);
      const int col = pos / a.ps;
      int page = -1;
      if (col < s_have[r]) {
        page = a.table[(long long)(b0 + r) * a.W + col];  // an earlier page, partly filled
      } else if (col < a.W) {
        const int idx = base_take + s_take_end[r] - s_take[r] + col - s_have[r];
        if (idx < a.F) page = a.free_pages[idx];
      }
      a.slots[base_new + i] = page < 0 ? -1ll : (long long)page * a.ps + pos % a.ps;
    }
    base_new += batch_new;
    base_take += batch_take;
    base_len += s_warp[kPlan / 32 - 1][2];
    __syncthreads();
  }
  for (long long i = base_new + (long long)blockIdx.x * kPlan + tid; i < a.T; i += (long long)gridDim.x * kPlan)
    a.slots[i] = -1;
  if (lead && tid == 0) {
    a.counts[0] = base_take;
    a.counts[1] = (int)(base_new - (long long)s_placed);
  }
}

// ---- page write ----------------------------------------------------------------
template <typename T>
__device__ __forceinline__ float2 to_float2(uint32_t v);
template <>
__device__ __forceinline__ float2 to_float2<__half>(uint32_t v) {
  return __half22float2(*reinterpret_cast<const __half2*>(&v));
}
template <>
__device__ __forceinline__ float2 to_float2<__nv_bfloat16>(uint32_t v) {
  return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}

struct WriteArgs {
  const void* x[2];        // k, v
  long long row_stride[2], head_stride[2];  // elements
  uint8_t* cache[2];
  const long long* slots;
  long long blocks;        // T * Hkv * NB
  long long num_slots;
  int H, NB;
};

// The q8_0 quantiser of quantize_rows (amax / 127, IEEE division, round half
// to even) on 16-bit rows: 8 lanes per block, 4 values each, so a warp reads
// 256 contiguous bytes per step. blockIdx.y picks K or V.
template <typename T>
__global__ void __launch_bounds__(256) page_write_kernel(const WriteArgs a) {
  const unsigned full = 0xffffffffu;
  const int lane = threadIdx.x & 31, sub = lane & 7;
  const int which = blockIdx.y;
  const long long per_row = (long long)a.H * a.NB;
  const long long nwarps = (long long)gridDim.x * (blockDim.x >> 5);
  const T* x = static_cast<const T*>(a.x[which]);
  for (long long b0 = ((long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5)) * 4; b0 < a.blocks;
       b0 += nwarps * 4) {
    const long long blk = min(b0 + (lane >> 3), a.blocks - 1);  // a repeated last block keeps all lanes in the shuffles
    const long long t = blk / per_row;
    const int rem = (int)(blk % per_row), h = rem / a.NB, j = rem % a.NB;
    const T* src = x + t * a.row_stride[which] + (long long)h * a.head_stride[which] + j * 32 + sub * 4;
    float v[4];
    const uint16_t* s16 = reinterpret_cast<const uint16_t*>(src);
    uint2 raw;
    if ((reinterpret_cast<uintptr_t>(src) & 7) == 0) {
      raw = *reinterpret_cast<const uint2*>(src);
    } else {
      raw.x = s16[0] | ((uint32_t)s16[1] << 16);
      raw.y = s16[2] | ((uint32_t)s16[3] << 16);
    }
    const float2 f0 = to_float2<T>(raw.x), f1 = to_float2<T>(raw.y);
    v[0] = f0.x, v[1] = f0.y, v[2] = f1.x, v[3] = f1.y;
    float amax = fmaxf(fmaxf(fabsf(v[0]), fabsf(v[1])), fmaxf(fabsf(v[2]), fabsf(v[3])));
#pragma unroll
    for (int o = 1; o <= 4; o <<= 1) amax = fmaxf(amax, __shfl_xor_sync(full, amax, o));
    const float d = amax > 0.0f ? __fdiv_rn(amax, 127.0f) : 1.0f;
    uint32_t code = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int q = max(-128, min(127, __float2int_rn(__fdiv_rn(v[i], d))));
      code |= (uint32_t)(q & 0xff) << (8 * i);
    }
    const long long slot = a.slots[t];
    if (slot < 0 || slot >= a.num_slots || b0 + (lane >> 3) >= a.blocks) continue;
    uint16_t* dst = reinterpret_cast<uint16_t*>(a.cache[which] + (slot * per_row + rem) * kQ8);
    dst[1 + 2 * sub] = (uint16_t)code;
    dst[2 + 2 * sub] = (uint16_t)(code >> 16);
    if (sub == 0) dst[0] = (uint16_t)float_to_half_bits(d);
  }
}

// ---- page read -----------------------------------------------------------------
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

struct ReadArgs {
  const uint8_t* cache[2];
  void* out[2];
  const int32_t* table;
  const int32_t* cu;
  int B, W, ps, H, NB;
  long long num_pages, rows;
};

// One warp per packed row (all heads of one token): lane l takes chunks of 8
// codes l, l + 32, ... of the row, 16 bytes out per chunk. blockIdx.y picks K
// or V. A row whose page id is outside the cache, and a row that no sequence
// owns, is zero.
template <typename T>
__global__ void __launch_bounds__(256) page_read_kernel(const ReadArgs a) {
  const int lane = threadIdx.x & 31, which = blockIdx.y;
  const long long nwarps = (long long)gridDim.x * (blockDim.x >> 5);
  const int per_row = a.H * a.NB;
  for (long long r = (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); r < a.rows; r += nwarps) {
    int lo = 0, hi = a.B;  // last b with cu[b] <= r
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (a.cu[mid] <= r) lo = mid;
      else hi = mid;
    }
    long long page = -1;
    const long long pos = r - a.cu[lo];
    if (pos >= 0 && r < a.cu[lo + 1] && pos / a.ps < a.W) page = a.table[(long long)lo * a.W + pos / a.ps];
    const bool valid = page >= 0 && page < a.num_pages;
    const uint8_t* src = a.cache[which] + (valid ? (page * a.ps + pos % a.ps) * per_row * kQ8 : 0);
    uint4* dst = reinterpret_cast<uint4*>(static_cast<T*>(a.out[which]) + r * per_row * 32);
    for (int c = lane; c < per_row * 4; c += 32) {
      uint4 o = make_uint4(0, 0, 0, 0);
      if (valid) {
        const uint16_t* blk = reinterpret_cast<const uint16_t*>(src + (c >> 2) * kQ8);
        const float d = half_bits_to_float(blk[0]);
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t two = blk[1 + (c & 3) * 4 + i];
          w[i] = pack2<T>(d * (float)(int8_t)(two & 0xff), d * (float)(int8_t)(two >> 8));
        }
        o = make_uint4(w[0], w[1], w[2], w[3]);
      }
      dst[c] = o;
    }
  }
}

int grid_for(long long items, int per_cta, int per_sm) {
  const long long want = (items + per_cta - 1) / per_cta;
  return (int)std::max(1ll, std::min(want, (long long)sm_count() * per_sm));
}

}  // namespace

kq_status_t launch_page_plan(const int32_t* cached, const int32_t* fresh, int B, int32_t* table, int W,
                             const int32_t* free_pages, int F, int ps, int64_t T, int64_t* slots, int32_t* seq_lens,
                             int32_t* cu_new, int32_t* cu_seqlens, int32_t* counts, cudaStream_t s) {
  PlanArgs a{cached, fresh, B, table, W, free_pages, F, ps, T, reinterpret_cast<long long*>(slots), seq_lens, cu_new,
             cu_seqlens, counts};
  page_plan_kernel<<<grid_for(T, kPlan * 4, 1), kPlan, 0, s>>>(a);
  return check_launch("page_plan");
}

kq_status_t launch_page_write_q8_0(int dtype, const void* k, const void* v, const int64_t* strides,
                                   const int64_t* slots, int64_t T, int H, int D, void* k_cache, void* v_cache,
                                   int64_t num_slots, cudaStream_t s) {
  WriteArgs a;
  a.x[0] = k, a.x[1] = v;
  a.row_stride[0] = strides[0], a.head_stride[0] = strides[1];
  a.row_stride[1] = strides[2], a.head_stride[1] = strides[3];
  a.cache[0] = static_cast<uint8_t*>(k_cache), a.cache[1] = static_cast<uint8_t*>(v_cache);
  a.slots = reinterpret_cast<const long long*>(slots);
  a.H = H, a.NB = D / 32;
  a.blocks = (long long)T * H * a.NB;
  a.num_slots = num_slots;
  const dim3 grid(grid_for(a.blocks, 32, 8), 2);
  if (dtype == KQ_F16) page_write_kernel<__half><<<grid, 256, 0, s>>>(a);
  else page_write_kernel<__nv_bfloat16><<<grid, 256, 0, s>>>(a);
  return check_launch("page_write");
}

kq_status_t launch_page_read_q8_0(int dtype, const void* k_cache, const void* v_cache, int64_t num_pages, int ps,
                                  int H, int D, const int32_t* table, int W, const int32_t* cu, int B, int64_t rows,
                                  void* k, void* v, cudaStream_t s) {
  ReadArgs a;
  a.cache[0] = static_cast<const uint8_t*>(k_cache), a.cache[1] = static_cast<const uint8_t*>(v_cache);
  a.out[0] = k, a.out[1] = v;
  a.table = table, a.cu = cu;
  a.B = B, a.W = W, a.ps = ps, a.H = H, a.NB = D / 32;
  a.num_pages = num_pages, a.rows = rows;
  const dim3 grid(grid_for(rows, 8, 8), 2);
  if (dtype == KQ_F16) page_read_kernel<__half><<<grid, 256, 0, s>>>(a);
  else page_read_kernel<__nv_bfloat16><<<grid, 256, 0, s>>>(a);
  return check_launch("page_read");
}

}  // namespace kq
