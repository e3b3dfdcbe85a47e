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
// few KB from L2, so the repeated scan costs less than a second launch. Bound
// by latency: 3.5 us for 8 requests of one token, 4.8 us for 256 prompts of
// 65536 tokens together (16.5 with CTAs of 128 threads).
constexpr int kPlan = 512;
constexpr int kFreeAtOnce = 8;  // entries of the free list that a thread looks at side by side

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
  int32_t* seq_lens;  // null: written by plan_lens_kernel
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
    const int have = min((unsigned)a.W, ((unsigned)c + a.ps - 1) / (unsigned)a.ps);
    const int need = min((unsigned)a.W, ((unsigned)c + n + a.ps - 1) / (unsigned)a.ps);
    const int take = need - have;
    int sums[3] = {n, take, c + n};
    scan3(sums, s_warp, lane, warp);
    s_cached[tid] = c;
    s_new[tid] = n;
    s_have[tid] = have;
    s_take[tid] = take;
    s_new_end[tid] = sums[0];
    s_take_end[tid] = sums[1];
    long long placed = 0;
    if (lead && b < a.B) {
      if (a.seq_lens) a.seq_lens[b] = c + n;
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
      placed = max(0ll, hi - lo);
    }
    if (lead) {
      // one addition per warp (integers: any order gives the same sum)
#pragma unroll
      for (int o = 16; o >= 1; o >>= 1) placed += __shfl_xor_sync(0xffffffffu, placed, o);
      if (lane == 0 && placed > 0) atomicAdd(&s_placed, (unsigned long long)placed);
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
    // new pages whose entry of the free list is negative (a list of fixed size,
    // padded): their tokens got no slot either
    if (lead) {
      for (int i0 = tid; i0 < batch_take; i0 += kFreeAtOnce * kPlan) {
        int page[kFreeAtOnce];
#pragma unroll
        for (int k = 0; k < kFreeAtOnce; ++k) {
          const int i = i0 + k * kPlan;
          page[k] = i < batch_take && base_take + i < a.F ? a.free_pages[base_take + i] : 0;
        }
#pragma unroll
        for (int k = 0; k < kFreeAtOnce; ++k) {
          if (page[k] >= 0) continue;
          const int i = i0 + k * kPlan, r = find_row(s_take_end, rows, i);
          const long long first = ((long long)s_have[r] + i - (s_take_end[r] - s_take[r])) * a.ps;
          const long long stop = s_cached[r] + min((long long)s_new[r], a.T - (base_new + s_new_end[r] - s_new[r]));
          const long long lost = min(first + a.ps, stop) - first;
          if (lost > 0) atomicAdd(&s_placed, (unsigned long long)-lost);
        }
      }
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

// Lengths updated in place by a plan of several CTAs, each of which reads all of
// them: only once that launch has ended.
__global__ void __launch_bounds__(256) plan_lens_kernel(const int32_t* cached, const int32_t* fresh, int B, int32_t* seq_lens) {
  for (int b = blockIdx.x * 256 + threadIdx.x; b < B; b += gridDim.x * 256)
    seq_lens[b] = max(0, cached[b]) + max(0, fresh[b]);
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
  long long T, num_slots;
  int H, NB, segs;         // segments of kSegBlocks blocks per row
};

// round_half_even(x / d) as IEEE division gives it, without the division:
// x * (1 / d) is within 2^-21 of x / d relatively, under 1e-4 for |x / d| <=
// 128, so the two round to different integers only that close to a half; only
// there (one value in 5000) the division runs. Adding 1.5 * 2^23 rounds to an
// integer, whose low byte is the code.
__device__ __forceinline__ uint32_t code_of(float x, float d, float inv) {
  const float q = x * inv, t = q + 12582912.0f;
  if (!(fabsf(q - (t - 12582912.0f)) < 0.4999f)) return (uint32_t)max(-128, min(127, __float2int_rn(__fdiv_rn(x, d)))) & 0xffu;
  return __float_as_uint(t) & 0xffu;
}

// The q8_0 quantiser of quantize_rows (amax / 127, IEEE division, round half
// to even) on 16-bit rows: a warp takes a segment of up to 32 blocks of one row
// of K or V, 8 lanes per block and 4 values each, all loads in flight at once.
// The bytes go through shared memory, laid out as far from a 16-byte boundary
// as their place in the cache is, so that they leave in whole 16-byte pieces:
// blocks of 34 bytes stored code by code leave half-written sectors behind,
// which made 4096 rows of 8 x 128 (26 MB in and out, 3.9 us of traffic) take 24
// us instead of 16; 13.8 with one division per block and no conversions. While
// it runs it issues 2.7 of 4 instructions a clock, with 40% of the warps that fit:
// 64 to 80 registers leave three or four CTAs per SM, 1.7 waves of one segment per
// warp, so that no segment's loads run under another one's quantiser. Segments of
// 16 blocks gain 1 us on single rows and lose 10 there.
constexpr int kSegBlocks = 32;
static_assert(kSegBlocks == 32, "a lane divides out the scale of one block of the segment");
constexpr int kSegRoom = (kSegBlocks * kQ8 + 16 + 15) / 16 * 16;

template <typename T>
__global__ void __launch_bounds__(256) page_write_kernel(const WriteArgs a) {
  __shared__ __align__(16) uint8_t s_seg[8][kSegRoom];
  const unsigned full = 0xffffffffu;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane & 7;
  const int per_row = a.H * a.NB;
  const long long units = a.T * 2 * a.segs;
  for (long long u = (long long)blockIdx.x * 8 + warp; u < units; u += (long long)gridDim.x * 8) {
    const long long t = u / (2 * a.segs);
    const int which = (int)(u / a.segs & 1), b0 = (int)(u % a.segs) * kSegBlocks, blocks = min(kSegBlocks, per_row - b0);
    const long long slot = a.slots[t];
    const T* x = static_cast<const T*>(which ? a.x[1] : a.x[0]) + t * (which ? a.row_stride[1] : a.row_stride[0]);
    const long long head_stride = which ? a.head_stride[1] : a.head_stride[0];
    uint2 raw[kSegBlocks / 4];
#pragma unroll
    for (int i = 0; i < kSegBlocks / 4; ++i) {
      const int blk = b0 + min(4 * i + (lane >> 3), blocks - 1);  // a repeated last block keeps all lanes in the shuffles
      const int h = blk / a.NB, j = blk - h * a.NB;
      const T* src = x + h * head_stride + j * 32 + sub * 4;
      if ((reinterpret_cast<uintptr_t>(src) & 7) == 0) {
        raw[i] = *reinterpret_cast<const uint2*>(src);
      } else {
        const uint16_t* s16 = reinterpret_cast<const uint16_t*>(src);
        raw[i] = make_uint2(s16[0] | ((uint32_t)s16[1] << 16), s16[2] | ((uint32_t)s16[3] << 16));
      }
    }
    const bool keep = slot >= 0 && slot < a.num_slots;
    uint8_t* dst = (which ? a.cache[1] : a.cache[0]) + (keep ? (slot * per_row + b0) * kQ8 : 0);
    const int off = (int)(reinterpret_cast<uintptr_t>(dst) & 15);
    __syncwarp();
    // every block's maximum in its 8 lanes; lane `sub` of them then takes block
    // 4 sub + lane / 8, so that each scale is divided out once, not by 8 lanes
    float mine = 0.0f;
#pragma unroll
    for (int i = 0; i < kSegBlocks / 4; ++i) {
      const float2 f0 = to_float2<T>(raw[i].x), f1 = to_float2<T>(raw[i].y);
      float amax = fmaxf(fmaxf(fabsf(f0.x), fabsf(f0.y)), fmaxf(fabsf(f1.x), fabsf(f1.y)));
#pragma unroll
      for (int o = 1; o <= 4; o <<= 1) amax = fmaxf(amax, __shfl_xor_sync(full, amax, o));
      if (sub == i) mine = amax;
    }
    const float my_d = mine > 0.0f ? __fdiv_rn(mine, 127.0f) : 1.0f, my_inv = 1.0f / my_d;
#pragma unroll
    for (int i = 0; i < kSegBlocks / 4; ++i) {
      const float2 f0 = to_float2<T>(raw[i].x), f1 = to_float2<T>(raw[i].y);
      const float v[4] = {f0.x, f0.y, f1.x, f1.y};
      const float d = __shfl_sync(full, my_d, (lane & 24) | i), inv = __shfl_sync(full, my_inv, (lane & 24) | i);
      uint32_t code = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) code |= code_of(v[k], d, inv) << (8 * k);
      const int blk = 4 * i + (lane >> 3);
      if (blk < blocks) {
        uint16_t* o = reinterpret_cast<uint16_t*>(s_seg[warp] + off + blk * kQ8);
        o[1 + 2 * sub] = (uint16_t)code;
        o[2 + 2 * sub] = (uint16_t)(code >> 16);
        if (sub == 0) o[0] = (uint16_t)float_to_half_bits(d);
      }
    }
    __syncwarp();
    if (keep) {
      const int end = off + blocks * kQ8;
      for (int p = lane * 16; p < end; p += 512) {
        if (p >= off && p + 16 <= end) {
          *reinterpret_cast<uint4*>(dst - off + p) = *reinterpret_cast<const uint4*>(s_seg[warp] + p);
        } else {  // the segment's ragged ends
          for (int k = max(p, off); k < min(p + 16, end); k += 2)
            *reinterpret_cast<uint16_t*>(dst - off + k) = *reinterpret_cast<const uint16_t*>(s_seg[warp] + k);
        }
      }
    }
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
  int B, W, ps, H, NB, segs;
  long long num_pages, rows;
};

// A unit is a segment of up to 32 blocks of one packed row of K or V; a warp
// takes kReadUnits of them. Lanes look the units' cache slots up side by side,
// the loads of all units (whole 16-byte pieces, from the boundary below) are in
// flight at once, then each unit is laid out in shared memory and lane l
// converts its codes 8 l, 8 l + 256, ..., 16 bytes out at a time. A row whose
// page id is outside the cache, and a row that no sequence owns, is zero.
// 34 bytes in and 64 out per block, 4.8 TB/s, next to the issue slots (2.8 of 4
// instructions a clock) and half of the conversion pipe. More units per warp put
// more loads in flight but leave fewer warps: 22445 rows of 8 x 128 after 4096
// written take 50.7 us with 1, 46.0 with 2, 51.4 with 4 (both calls; 43.5 since the
// write is faster).
constexpr int kReadUnits = 2;
constexpr int kUnitPieces = (kSegRoom / 16 + 31) / 32;  // of a unit, per lane

template <typename T>
__global__ void __launch_bounds__(256, 4) page_read_kernel(const ReadArgs a) {
  __shared__ __align__(16) uint8_t s_seg[8][kSegRoom];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int per_row = a.H * a.NB;
  const long long row_bytes = (long long)per_row * kQ8, cache_bytes = a.num_pages * a.ps * row_bytes;
  uint8_t* seg = s_seg[warp];
  const long long units = a.rows * 2 * a.segs;
  for (long long u0 = ((long long)blockIdx.x * 8 + warp) * kReadUnits; u0 < units; u0 += (long long)gridDim.x * 8 * kReadUnits) {
    // lane i: the place of unit i's first byte in its cache, -1 without one
    long long at = -1;
    if (lane < kReadUnits && u0 + lane < units) {
      const long long r = (u0 + lane) / (2 * a.segs);
      int lo = 0, hi = a.B;  // last b with cu[b] <= r
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.cu[mid] <= r) lo = mid;
        else hi = mid;
      }
      const long long pos = r - a.cu[lo];
      if (pos >= 0 && r < a.cu[lo + 1] && pos / a.ps < a.W) {
        const long long page = a.table[(long long)lo * a.W + pos / a.ps];
        if (page >= 0 && page < a.num_pages)
          at = (page * a.ps + pos % a.ps) * row_bytes + (u0 + lane) % a.segs * (kSegBlocks * kQ8);
      }
    }
    uint4 v[kReadUnits][kUnitPieces];
    long long from[kReadUnits];
#pragma unroll
    for (int i = 0; i < kReadUnits; ++i) {
      from[i] = __shfl_sync(0xffffffffu, at, i);
      const uint8_t* cache = ((u0 + i) / a.segs & 1) ? a.cache[1] : a.cache[0];
      const int b0 = (int)((u0 + i) % a.segs) * kSegBlocks, blocks = min(kSegBlocks, per_row - b0);
      const long long first = from[i] & ~15ll, end = min(from[i] + blocks * kQ8, cache_bytes);
#pragma unroll
      for (int k = 0; k < kUnitPieces; ++k) {
        const long long p = first + 16 * (lane + 32 * k);
        v[i][k] = make_uint4(0, 0, 0, 0);
        if (from[i] < 0 || p >= end) continue;
        if (p + 16 <= cache_bytes) {
          v[i][k] = *reinterpret_cast<const uint4*>(cache + p);
        } else {  // the cache's last bytes
          const int left = (int)(cache_bytes - p);
          const uint16_t* h = reinterpret_cast<const uint16_t*>(cache + p);
          auto half = [&](int x) { return 2 * x < left ? (uint32_t)h[x] : 0u; };
          v[i][k] = make_uint4(half(0) | half(1) << 16, half(2) | half(3) << 16, half(4) | half(5) << 16, half(6));
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kReadUnits; ++i) {
      if (u0 + i >= units) break;
      const long long r = (u0 + i) / (2 * a.segs);
      const int which = (int)((u0 + i) / a.segs & 1), b0 = (int)((u0 + i) % a.segs) * kSegBlocks;
      const int blocks = min(kSegBlocks, per_row - b0), off = from[i] < 0 ? 0 : (int)(from[i] & 15);
      uint4* dst = reinterpret_cast<uint4*>(static_cast<T*>(which ? a.out[1] : a.out[0]) + (r * per_row + b0) * 32);
      __syncwarp();
#pragma unroll
      for (int k = 0; k < kUnitPieces; ++k)
        if (16 * (lane + 32 * k) < kSegRoom) *reinterpret_cast<uint4*>(seg + 16 * (lane + 32 * k)) = v[i][k];
      __syncwarp();
      for (int c = lane; c < blocks * 4; c += 32) {
        const int blk = off + (c >> 2) * kQ8, x = blk + 2 + (c & 3) * 8;  // even
        const float d = half_bits_to_float(*reinterpret_cast<const uint16_t*>(seg + blk));
        const uint32_t* w = reinterpret_cast<const uint32_t*>(seg + (x & ~3));
        const uint32_t sh = (uint32_t)(x & 2) * 8, top = sh ? w[2] : 0u;
        const uint32_t w0 = __funnelshift_r(w[0], w[1], sh), w1 = __funnelshift_r(w[1], top, sh);
        auto value = [&](uint32_t word, int k) { return d * (float)(int8_t)(word >> (8 * k)); };
        uint4 o = make_uint4(pack2<T>(value(w0, 0), value(w0, 1)), pack2<T>(value(w0, 2), value(w0, 3)),
                             pack2<T>(value(w1, 0), value(w1, 1)), pack2<T>(value(w1, 2), value(w1, 3)));
        dst[c] = from[i] < 0 ? make_uint4(0, 0, 0, 0) : o;
      }
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
  const int grid = grid_for(T, kPlan, 1);
  // in place, a single CTA reads a request's lengths before the same thread writes its sum
  const bool later = grid > 1 && (seq_lens == cached || seq_lens == fresh);
  PlanArgs a{cached, fresh, B, table, W, free_pages, F, ps, T, reinterpret_cast<long long*>(slots),
             later ? nullptr : seq_lens, cu_new, cu_seqlens, counts};
  page_plan_kernel<<<grid, kPlan, 0, s>>>(a);
  if (kq_status_t st = check_launch("page_plan")) return st;
  if (!later || B == 0) return KQ_OK;
  plan_lens_kernel<<<grid_for(B, 256, 1), 256, 0, s>>>(cached, fresh, B, seq_lens);
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
  a.T = T;
  a.segs = (H * a.NB + kSegBlocks - 1) / kSegBlocks;
  a.num_slots = num_slots;
  const int grid = grid_for(T * 2 * a.segs, 8, 8);
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
  a.segs = (H * a.NB + kSegBlocks - 1) / kSegBlocks;
  const int grid = grid_for(rows * 2 * a.segs, 8 * kReadUnits, 8);
  if (dtype == KQ_F16) page_read_kernel<__half><<<grid, 256, 0, s>>>(a);
  else page_read_kernel<__nv_bfloat16><<<grid, 256, 0, s>>>(a);
  return check_launch("page_read");
}

}  // namespace kq
