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
#include <cmath>
#include <type_traits>

#include "kq_internal.h"
#include "kq_device.cuh"
#include "kq_tc.cuh"

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

// ---- tensor cores: D <= 128, rows TMA can address -------------------------------
// One CTA takes up to two query tiles of one KV head. A tile is 128 rows: TQ =
// 128 / G tokens x the G query heads that share the KV head (row = token * G +
// g), so K and V are read once per group and short prompts fill the tile.
// Keys come in blocks of 128. Per block and tile:
//   S = Q K^T   tcgen05, Q and K in shared memory, S fp32 in TMEM
//   P = 2^(S sl - m + kBias)   one thread per row (TMEM lane), P to TMEM over S
//   O += P V    tcgen05, P from TMEM, V in shared memory, O fp32 in TMEM
// The two tiles alternate: while the softmax warps of one work, the tensor
// core runs the other's two products. The running maximum m only moves when a
// row's maximum grows by more than 2^kLazy (then O is rescaled in TMEM): p
// stays below 2^(kBias + kLazy), inside fp16, and the factor cancels in O / l.
// P is rounded to the inputs' type, as the product with V needs both operands
// in it; l sums the unrounded p in fp32.
//
// Warps: 0-3 softmax of tile 0, 4-7 of tile 1 (warp w reaches TMEM lanes
// 32 (w % 4) ..), 8 MMA issue and TMEM, 9 TMA.
constexpr int kTile = 128;            // rows of a query tile, keys of a block
constexpr int kTcThreads = 320;
constexpr int kMmaWarp = 8, kLoadWarp = 9;
constexpr float kBias = 7.0f, kLazy = 8.0f;

template <int DP>
struct TcTraits {
  static constexpr int PANELS = DP / 64;           // 128-byte swizzled panels of 64 dims
  static constexpr int PANEL = kTile * 128;        // bytes
  static constexpr int OPERAND = PANELS * PANEL;   // a Q tile, K block or V block
  static constexpr int STAGES = DP == 128 ? 5 : 10;  // K and V blocks in flight (alternating)
  static constexpr int OFF_Q = 0;
  static constexpr int OFF_KV = 2 * OPERAND;
  static constexpr int OFF_BAR = OFF_KV + STAGES * OPERAND;
  static constexpr int SMEM = OFF_BAR + 256 + 1024;
  static_assert(SMEM <= 232448, "shared memory budget");
};
constexpr uint32_t kColS = 0, kColO = 256;         // TMEM: S0 S1 | O0 O1 (O tiles DP columns apart)

struct TcArgs {
  const int32_t *cu_q, *cu_k;
  int B, Tq, Hq, Hkv, G, TQ, D, causal, tiles, slots;
  float sl;             // scale * log2(e), not negative
  uint32_t flip;        // sign bit where scale < 0: scores are negated first
  void* out;
  int* err;
};

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

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
          smem_u32(dst)),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
      : "memory");
}
// Instruction descriptor, kind::f16: fp32 D, A and B of type T, M = 128; bit 16: B is MN-major.
template <typename T>
__host__ __device__ constexpr uint32_t idesc(int n, bool b_mn) {
  const uint32_t f = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
  return (1u << 4) | (f << 7) | (f << 10) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((128u >> 4) << 24);
}

// Tokens and keys of a CTA's work.
struct Work {
  int q0, lq, k0, lk, tok;  // sequence's first row, rows, first key, keys; first token of the CTA
};
// Slot -> (sequence, tile): sequence b owns slots cu_q[b] / TT + b .., at
// least ceil(len / TT) of them, so no prefix sum over tiles is needed; slots
// past a sequence's end are empty (at most one or two per sequence).
__device__ __forceinline__ bool find_work(const TcArgs& a, int slot, Work& w) {
  const int tt = a.TQ * a.tiles;
  int lo = 0, hi = a.B;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a.cu_q[mid] / tt + mid <= slot) lo = mid;
    else hi = mid;
  }
  w.q0 = a.cu_q[lo];
  w.lq = min(a.cu_q[lo + 1], a.Tq) - w.q0;
  w.k0 = a.cu_k[lo];
  w.lk = max(0, a.cu_k[lo + 1] - w.k0);
  w.tok = (slot - (w.q0 / tt + lo)) * tt;
  return w.tok < w.lq;
}
// Keys that token i of the sequence sees.
__device__ __forceinline__ int keys_of(const TcArgs& a, const Work& w, int i) {
  return a.causal ? max(0, min(w.lk, i + w.lk - w.lq + 1)) : w.lk;
}
// Key blocks of tile t (0 when it has no token or sees no key).
__device__ __forceinline__ int blocks_of(const TcArgs& a, const Work& w, int t) {
  const int first = w.tok + t * a.TQ;
  if (t >= a.tiles || first >= w.lq) return 0;
  return (keys_of(a, w, min(w.lq, first + a.TQ) - 1) + kTile - 1) / kTile;
}

template <typename T, int DP>
__global__ void __launch_bounds__(kTcThreads, 1)
    fa_prompt_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                        const __grid_constant__ CUtensorMap map_v, const __grid_constant__ TcArgs a) {
  using R = TcTraits<DP>;
  constexpr int STAGES = R::STAGES;
  const int head = blockIdx.x % a.Hkv;
  Work w;
  // later tiles of a causal sequence see more keys: they start first
  if (!find_work(a, a.slots - 1 - blockIdx.x / a.Hkv, w)) return;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint64_t* q_full = reinterpret_cast<uint64_t*>(smem + R::OFF_BAR);
  uint64_t* kv_full = q_full + 2;
  uint64_t* kv_empty = kv_full + STAGES;
  uint64_t* s_full = kv_empty + STAGES;   // S of a tile is there (and its earlier P V is done)
  uint64_t* p_full = s_full + 2;          // P of a tile is there, its S is read
  uint64_t* o_full = p_full + 2;          // the tile's last P V is done
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(o_full + 2);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
      mbar_init(&o_full[i], 1);
    }
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(&kv_full[i], 1);
      mbar_init(&kv_empty[i], 1);
    }
    fence_mbar_init();
  }
  // rows of a query tile that no token fills stay zero
  for (int i = threadIdx.x; i < 2 * R::PANELS * (kTile - a.TQ * a.G) * 8; i += kTcThreads) {
    const int rows = kTile - a.TQ * a.G, c = i % 8, r = i / 8 % rows, panel = i / 8 / rows;
    *reinterpret_cast<uint4*>(smem + R::OFF_Q + panel * R::PANEL + (a.TQ * a.G + r) * 128 + c * 16) = make_uint4(0, 0, 0, 0);
  }
  fence_proxy_async_smem();
  if (warp == kMmaWarp) tc::tmem_alloc(tmem_slot, 512);
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int n0 = blocks_of(a, w, 0), n1 = blocks_of(a, w, 1), n = max(n0, n1);
  bool dead = false;

  if (warp == kLoadWarp) {
    if (lane == 0) {
      tc::prefetch_tmap(&map_q);
      tc::prefetch_tmap(&map_k);
      tc::prefetch_tmap(&map_v);
      for (int t = 0; t < 2; ++t) {
        if ((t ? n1 : n0) == 0) continue;
        mbar_arrive_expect_tx(&q_full[t], R::PANELS * a.TQ * a.G * 128);
        for (int p = 0; p < R::PANELS; ++p)
          tma_load_3d(smem + R::OFF_Q + t * R::OPERAND + p * R::PANEL, &map_q, p * 64, head * a.G,
                      w.q0 + w.tok + t * a.TQ, &q_full[t]);
      }
      for (int i = 0; i < 2 * n; ++i) {  // K0 V0 K1 V1 ..
        const int st = i % STAGES;
        if (i >= STAGES) mbar_wait_idle_or_poison(&kv_empty[st], ((i / STAGES) - 1) & 1, a.err, DEV_TIMEOUT_EMPTY, dead);
        mbar_arrive_expect_tx(&kv_full[st], R::OPERAND);
        for (int p = 0; p < R::PANELS; ++p)
          tma_load_3d(smem + R::OFF_KV + st * R::OPERAND + p * R::PANEL, (i & 1) ? &map_v : &map_k, p * 64, head,
                      w.k0 + (i >> 1) * kTile, &kv_full[st]);
      }
    }
    __syncwarp();
  } else if (warp == kMmaWarp) {
    constexpr uint32_t idesc_s = idesc<T>(kTile, false), idesc_o = idesc<T>(DP, true);
    const uint32_t q_base = smem_u32(smem + R::OFF_Q), kv_base = smem_u32(smem + R::OFF_KV);
    const uint32_t go = tc::elect_one();
    // S_t = Q_t K_j^T
    auto score = [&](int t, int j) {
      const int st = 2 * j % STAGES;
      mbar_wait_or_poison(&kv_full[st], (2 * j / STAGES) & 1, a.err, DEV_TIMEOUT_FULL, dead);
      tc::tc_fence_after();
      const uint64_t qd = tc::sw128_desc(q_base + t * R::OPERAND), kd = tc::sw128_desc(kv_base + st * R::OPERAND);
#pragma unroll
      for (int k = 0; k < DP / 16; ++k) {
        const uint64_t off = (uint64_t)((k >> 2) * (R::PANEL >> 4) + (k & 3) * 2);
        tc::mma_ss_go(tmem + kColS + t * kTile, qd + off, kd + off, idesc_s, k > 0, go);
      }
      tc::mma_commit_go(&s_full[t], go);
    };
    for (int t = 0; t < 2; ++t)
      if ((t ? n1 : n0) > 0) {
        mbar_wait_or_poison(&q_full[t], 0, a.err, DEV_TIMEOUT_FULL, dead);
        score(t, 0);
      }
    if (n > 0) tc::mma_commit_go(&kv_empty[0], go);
    for (int j = 0; j < n; ++j) {
      const int sv = (2 * j + 1) % STAGES;
#pragma unroll 1
      for (int t = 0; t < 2; ++t) {
        const int nt = t ? n1 : n0;
        if (j >= nt) continue;
        mbar_wait_or_poison(&kv_full[sv], ((2 * j + 1) / STAGES) & 1, a.err, DEV_TIMEOUT_FULL, dead);
        mbar_wait_or_poison(&p_full[t], j & 1, a.err, DEV_TIMEOUT_FULL, dead);
        tc::tc_fence_after();
        const uint64_t vd = tc::sw128_desc_mn(kv_base + sv * R::OPERAND, R::PANEL);  // dims across, tokens down
#pragma unroll
        for (int k = 0; k < kTile / 16; ++k)
          tc::mma_ts_go(tmem + kColO + t * DP, tmem + kColS + t * kTile + 8 * k, vd + (uint64_t)(k * (2048 >> 4)), idesc_o,
                        (j > 0 || k > 0) ? 1u : 0u, go);
        if (j + 1 == nt) tc::mma_commit_go(&o_full[t], go);
        if (j + 1 < nt) score(t, j + 1);
      }
      tc::mma_commit_go(&kv_empty[sv], go);
      if (j + 1 < n) tc::mma_commit_go(&kv_empty[(2 * j + 2) % STAGES], go);
    }
    __syncwarp();
  } else {
    const int t = warp >> 2, row = threadIdx.x & 127, nt = t ? n1 : n0;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_addr = tmem + lanes + kColS + t * kTile, o_addr = tmem + lanes + kColO + t * DP;
    const int first = w.tok + t * a.TQ;                     // the tile's first token
    const int tok = first + row / a.G, g = row % a.G;
    const bool mine = row < a.TQ * a.G && t < a.tiles && tok < w.lq;
    const int keys = mine ? keys_of(a, w, tok) : 0;
    const int all_see = keys_of(a, w, first);               // keys that every row of the tile sees
    float m = -INFINITY, l = 0.0f;
    for (int j = 0; j < nt; ++j) {
      mbar_wait_or_poison(&s_full[t], j & 1, a.err, DEV_TIMEOUT_FULL, dead);
      __syncwarp();
      tc::tc_fence_after();
      uint32_t s[kTile];
#pragma unroll
      for (int c = 0; c < kTile / 32; ++c) tc::tmem_ld32(s_addr + 32 * c, reinterpret_cast<uint32_t(&)[32]>(s[32 * c]));
      tc::tmem_ld_wait();
      if (a.flip) {
#pragma unroll
        for (int i = 0; i < kTile; ++i) s[i] ^= a.flip;
      }
      if ((j + 1) * kTile > all_see) {
        const int lim = keys - j * kTile;
#pragma unroll
        for (int i = 0; i < kTile; ++i)
          if (i >= lim) s[i] = 0xff800000u;
        const int valid = w.lk - j * kTile;
        if (valid < kTile) {
          // rows of V behind the sequence's end belong to others: what they
          // hold must not meet P (0 x inf); both tiles write the same zeros
          const int sv = (2 * j + 1) % STAGES;
          mbar_wait_or_poison(&kv_full[sv], ((2 * j + 1) / STAGES) & 1, a.err, DEV_TIMEOUT_FULL, dead);
          for (int i = row; i < (kTile - valid) * 8 * R::PANELS; i += kTile) {
            const int c = i % 8, p = i / 8 % R::PANELS, r = valid + i / (8 * R::PANELS);
            *reinterpret_cast<uint4*>(smem + R::OFF_KV + sv * R::OPERAND + p * R::PANEL + r * 128 + c * 16) =
                make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();
        }
      }
      float mx[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) mx[i] = __uint_as_float(s[i]);
#pragma unroll
      for (int i = 4; i < kTile; ++i) mx[i & 3] = fmaxf(mx[i & 3], __uint_as_float(s[i]));
      const float mn = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * a.sl;
      float f = 1.0f;
      if (mn > m + kLazy) {  // also the row's first keys (m = -inf)
        f = ex2(m - mn);
        m = mn;
        l *= f;
      }
      if (j > 0 && __any_sync(0xffffffffu, f != 1.0f)) {
#pragma unroll 1
        for (int c = 0; c < DP / 32; ++c) {
          uint32_t o[32];
          tc::tmem_ld32(o_addr + 32 * c, o);
          tc::tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
          tc::tmem_st32(o_addr + 32 * c, o);
        }
      }
      const float off = m == -INFINITY ? 0.0f : kBias - m;
      float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      uint32_t p[kTile / 2];
#pragma unroll
      for (int i = 0; i < kTile / 2; ++i) {
        const float p0 = ex2(fmaf(__uint_as_float(s[2 * i]), a.sl, off));
        const float p1 = ex2(fmaf(__uint_as_float(s[2 * i + 1]), a.sl, off));
        sum[(2 * i) & 3] += p0;
        sum[(2 * i + 1) & 3] += p1;
        p[i] = pack2<T>(p0, p1);
      }
      l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
      __syncwarp();
      tc::tmem_st32(s_addr, p);
      tc::tmem_st32(s_addr + 32, p + 32);
      tc::tmem_st_wait();
      tc::tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[t]);
    }
    // O / l
    if (nt > 0) {
      mbar_wait_or_poison(&o_full[t], 0, a.err, DEV_TIMEOUT_FULL, dead);
      __syncwarp();
      tc::tc_fence_after();
    }
    T* out = static_cast<T*>(a.out) + ((long long)(w.q0 + tok) * a.Hq + head * a.G + g) * a.D;
    const bool none = nt == 0 || l == 0.0f;
    const float inv = 1.0f / l;
#pragma unroll 1
    for (int c = 0; c < DP / 32; ++c) {
      uint32_t o[32];
      __syncwarp();
      if (nt > 0) {
        tc::tmem_ld32(o_addr + 32 * c, o);
        tc::tmem_ld_wait();
      }
      if (mine) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint4 v = make_uint4(0, 0, 0, 0);
          if (!none) {
            v.x = pack2<T>(__uint_as_float(o[8 * i]) * inv, __uint_as_float(o[8 * i + 1]) * inv);
            v.y = pack2<T>(__uint_as_float(o[8 * i + 2]) * inv, __uint_as_float(o[8 * i + 3]) * inv);
            v.z = pack2<T>(__uint_as_float(o[8 * i + 4]) * inv, __uint_as_float(o[8 * i + 5]) * inv);
            v.w = pack2<T>(__uint_as_float(o[8 * i + 6]) * inv, __uint_as_float(o[8 * i + 7]) * inv);
          }
          if (32 * c + 8 * i < a.D) *reinterpret_cast<uint4*>(out + 32 * c + 8 * i) = v;
        }
      }
    }
  }
  tc::tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) tc::tmem_dealloc(tmem, 512);
}

// [T, H, D] rows as a 3-D map of 64-dim x `heads` x `tokens` boxes, 128-byte swizzled
bool encode_rows(CUtensorMap* map, int dtype, const void* base, int D, int H, int64_t T, int64_t head, int64_t row,
                 int heads, int tokens) {
  cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)H, (cuuint64_t)T};
  cuuint64_t strides[2] = {(cuuint64_t)(H > 1 ? head * 2 : D * 2), (cuuint64_t)(T > 1 ? row * 2 : D * 2)};
  cuuint32_t box[3] = {64, (cuuint32_t)heads, (cuuint32_t)tokens}, estr[3] = {1, 1, 1};
  return tc::encode_tiled(map, dtype == KQ_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3,
                          const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// TMA wants 16-byte aligned bases and strides (a stride of 0 or below is a
// broadcast or reversed view).
bool tma_rows(const void* p, int H, int64_t T, int64_t head, int64_t row) {
  auto ok = [](int64_t n, int64_t s) { return n <= 1 || (s > 0 && s % 8 == 0 && s < (int64_t)1 << 38); };
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ok(H, head) && ok(T, row);
}

bool tc_supported(const FaPromptArgs& a) {
  return a.D <= 128 && a.Hq / a.Hkv <= kTile && a.Tk > 0 && tma_rows(a.q, a.Hq, a.Tq, a.q_head, a.q_row) &&
         tma_rows(a.k, a.Hkv, a.Tk, a.k_head, a.k_row) && tma_rows(a.v, a.Hkv, a.Tk, a.v_head, a.v_row);
}

template <typename T, int DP>
kq_status_t launch_tc(const FaPromptArgs& a, int dtype, cudaStream_t s) {
  TcArgs p{};
  p.cu_q = a.cu_q, p.cu_k = a.cu_k;
  p.B = a.B, p.Tq = a.Tq, p.Hq = a.Hq, p.Hkv = a.Hkv, p.D = a.D, p.causal = a.causal;
  p.G = a.Hq / a.Hkv;
  p.TQ = kTile / p.G;
  // two tiles per CTA where that still gives every SM work
  p.tiles = (long long)(a.Tq / (2 * p.TQ)) * a.Hkv >= sm_count() ? 2 : 1;
  p.slots = a.Tq / (p.TQ * p.tiles) + a.B;
  const float sl = a.scale * 1.44269504088896340736f;
  p.flip = sl < 0.0f ? 0x80000000u : 0u;
  p.sl = fmaxf(fabsf(sl), 1e-30f);  // a scale of 0 keeps -inf for hidden keys
  p.out = a.out;
  p.err = device_error_word();
  CUtensorMap mq, mk, mv;
  if (!encode_rows(&mq, dtype, a.q, a.D, a.Hq, a.Tq, a.q_head, a.q_row, p.G, p.TQ) ||
      !encode_rows(&mk, dtype, a.k, a.D, a.Hkv, a.Tk, a.k_head, a.k_row, 1, kTile) ||
      !encode_rows(&mv, dtype, a.v, a.D, a.Hkv, a.Tk, a.v_head, a.v_row, 1, kTile))
    return fail(KQ_ERR_CUDA, "fa_prompt: tensor map encoding failed");
  auto kernel = fa_prompt_tc_kernel<T, DP>;
  if (kq_status_t st = ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), TcTraits<DP>::SMEM, "fa_prompt")) return st;
  kernel<<<(unsigned)(p.slots * a.Hkv), kTcThreads, TcTraits<DP>::SMEM, s>>>(mq, mk, mv, p);
  return check_launch("fa_prompt_tc");
}

}  // namespace

size_t fa_prompt_workspace(const FaPromptArgs&) { return 0; }

kq_status_t launch_fa_prompt(const FaPromptArgs& a, int dtype, cudaStream_t s) {
  if (tc_supported(a)) {
    if (a.D <= 64)
      return dtype == KQ_F16 ? launch_tc<__half, 64>(a, dtype, s) : launch_tc<__nv_bfloat16, 64>(a, dtype, s);
    return dtype == KQ_F16 ? launch_tc<__half, 128>(a, dtype, s) : launch_tc<__nv_bfloat16, 128>(a, dtype, s);
  }
  const long long items = (long long)a.Tq * a.Hq;
  const unsigned grid = (unsigned)((items + kSimpleWarps - 1) / kSimpleWarps);
  if (dtype == KQ_F16) fa_prompt_simple_kernel<__half><<<grid, kSimpleWarps * 32, 0, s>>>(a);
  else fa_prompt_simple_kernel<__nv_bfloat16><<<grid, kSimpleWarps * 32, 0, s>>>(a);
  return check_launch("fa_prompt");
}

}  // namespace kq
