// Attention of whole prompts: packed sequences of different lengths, grouped
// query heads, causal.
//
//   s_ij = scale q_i . k_j,  j <= i + (len_k - len_q) when causal,
//   out_i = sum_j exp(s_ij - m_i) v_j / sum_j exp(s_ij - m_i),  m_i = max_j s_ij
//
// with row i of a sequence's len_q new tokens and key j of its len_k tokens
// (len_k > len_q: the chunk follows an earlier context). A row without keys
// is zero. The maxima, sums and the output accumulate in fp32.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "kq_internal.h"
#include "kq_attn.cuh"
#include "kq_device.cuh"
#include "kq_tc.cuh"

namespace kq {
namespace {

using namespace attn;

// An entry of the prefix sums, cut to the rows that there are: nothing outside
// them is read or written whatever the sums say.
__device__ __forceinline__ int cut(int x, int rows) { return max(0, min(x, rows)); }

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

// ---- one row by one warp ----------------------------------------------------------
// The softmax state (natural units) of keys j0 .. j1 - 1 for the scaled query s_q
// in shared memory; s_p holds 32 values. 32 keys per step, one per lane for q . k,
// then the lanes own output dimensions (lane + 32 t) for p . v. SHORT: little code
// instead of unrolled loops.
template <bool SHORT, int ND, typename T>
__device__ __forceinline__ void attend_keys(const T* kb, const T* vb, long long k_row, long long v_row, int D, int j0, int j1,
                                            const float* s_q, float* s_p, float& m, float& l, float (&acc)[ND]) {
  const unsigned full = 0xffffffffu;
  const int lane = threadIdx.x & 31;
  m = -INFINITY, l = 0.0f;
#pragma unroll
  for (int t = 0; t < ND; ++t) acc[t] = 0.0f;
  for (; j0 < j1; j0 += 32) {
    const int j = j0 + lane;
    float s = -INFINITY;
    if (j < j1) {
      const T* k = kb + (long long)j * k_row;
      float dot = 0.0f;
      if constexpr (SHORT) {
#pragma unroll 1
        for (int d = 0; d < D; ++d) dot = fmaf(s_q[d], to_f(k[d]), dot);
      } else {
        for (int d = 0; d < D; ++d) dot = fmaf(s_q[d], to_f(k[d]), dot);
      }
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
    s_p[lane] = p;
    __syncwarp();
#pragma unroll
    for (int t = 0; t < ND; ++t) acc[t] *= c;
    const int n = min(32, j1 - j0);
    auto add = [&](int jj) {
      const float pj = s_p[jj];
      const T* v = vb + (long long)(j0 + jj) * v_row;
#pragma unroll
      for (int t = 0; t < ND; ++t) {
        const int d = lane + 32 * t;
        if (d < D) acc[t] = fmaf(pj, to_f(v[d]), acc[t]);
      }
    };
    if constexpr (SHORT) {
#pragma unroll 1
      for (int jj = 0; jj < n; ++jj) add(jj);
    } else {
      for (int jj = 0; jj < n; ++jj) add(jj);
    }
    __syncwarp();
  }
}

// ---- any shape ------------------------------------------------------------------
// One warp per (row, query head). Bound by its scalar loads and FMAs; it serves
// the head sizes and strides that the tensor-core kernel does not take.
constexpr int kSimpleWarps = 4;
constexpr int kMaxD = 256;

template <typename T>
__global__ void __launch_bounds__(kSimpleWarps * 32) fa_prompt_simple_kernel(const FaPromptArgs a) {
  __shared__ float s_q[kSimpleWarps][kMaxD];
  __shared__ float s_p[kSimpleWarps][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long item = (long long)blockIdx.x * kSimpleWarps + warp;
  if (item >= (long long)a.Tq * a.Hq) return;
  const long long row = item / a.Hq;
  const int h = (int)(item % a.Hq), kh = h / (a.Hq / a.Hkv);
  const int b = find_seq(a.cu_q, a.B, row);
  T* out = static_cast<T*>(a.out) + (row * a.Hq + h) * a.D;
  const int q0 = cut(a.cu_q[b], a.Tq), lq = cut(a.cu_q[b + 1], a.Tq) - q0;
  const int k0 = cut(a.cu_k[b], a.Tk), lk = max(0, cut(a.cu_k[b + 1], a.Tk) - k0);
  const int i = (int)(row - q0);
  const int keys = i >= lq || i < 0 ? 0 : a.causal ? max(0, min(lk, i + lk - lq + 1)) : lk;
  const T* q = static_cast<const T*>(a.q) + row * a.q_row + (long long)h * a.q_head;
  const T* kb = static_cast<const T*>(a.k) + (long long)k0 * a.k_row + (long long)kh * a.k_head;
  const T* vb = static_cast<const T*>(a.v) + (long long)k0 * a.v_row + (long long)kh * a.v_head;
  for (int d = lane; d < a.D; d += 32) s_q[warp][d] = to_f(q[d]) * a.scale;
  __syncwarp();
  float m, l, acc[kMaxD / 32];
  attend_keys<false>(kb, vb, a.k_row, a.v_row, a.D, 0, keys, s_q[warp], s_p[warp], m, l, acc);
  const float inv = l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l);  // NaN stays NaN
#pragma unroll
  for (int t = 0; t < kMaxD / 32; ++t) {
    const int d = lane + 32 * t;
    if (d < a.D) store_f(out + d, acc[t] * inv);
  }
}

// ---- tensor cores: D <= 128, rows TMA can address -------------------------------
// A CTA takes TILES query tiles of one KV head. A tile is 128 rows: TQ = 128 / G
// tokens x the G query heads that share the KV head (row = token * G + g), so K
// and V are read once per group and short prompts fill the tile. Keys come in
// blocks of BLK. Per block and tile:
//   S = Q K^T   tcgen05, Q and K in shared memory, S fp32 in TMEM
//   P = 2^(S sl - m + kBias)   one thread per row (TMEM lane), P to TMEM over S
//   O += P V    tcgen05, P from TMEM, V in shared memory, O fp32 in TMEM
// The running maximum m only moves when a row's maximum grows by more than
// 2^kLazy (then O is rescaled in TMEM): p stays below 2^(kBias + kLazy), inside
// fp16, and the factor cancels in O / l. P is rounded to the inputs' type, as
// the product with V needs both operands in it; l sums the unrounded p in fp32.
// That is one more rounding of the output's own size, averaged over the keys
// (relative errors 2.6e-4 in fp16 and 2.3e-3 in bf16 at most, 2.0e-4 and 1.7e-3
// with P in fp32); a second product with P's remainder would double P V.
//
// TILES = 2, BLK = 128: one CTA per SM, K and V read once for 256 rows. The
// tiles alternate: the softmax warps of one work while the tensor core runs
// the other's products; P is handed over in halves of 64 keys, so that the
// product with V starts under the second half's exponentials. Per block of two
// tiles the tensor core needs 2048 clocks, shared memory about as many (each
// product reads both operands of S there; 64-key blocks would read Q twice as
// often), the special-function unit another 2048 at 16 exponentials a clock. A
// block takes about 3300: the chain S -> maximum -> P -> next S of each tile is
// what bounds it. Without exponentials, maxima and sums it would be 2700; some
// exponentials as a polynomial on the FMA pipe changed nothing (474 us with 16
// of 64, 474 without, 479 with 24; 8192 tokens, 32 heads over 8).
// TILES = 1, BLK = 64: two CTAs per SM, each hiding the other's start and end,
// with two S buffers; for short sequences.
// CTAs are persistent: the TMA warp looks up the next job and starts its loads
// while the softmax warps still work on the last one, and the MMA warp runs
// its first products under their epilogue. A short job is otherwise mostly
// set-up: TMEM, look-ups, first loads, last stores.
// Warps: 4 softmax warps per tile (warp w reaches TMEM lanes 32 (w % 4) ..),
// one that issues MMAs, one for jobs and TMA (and two idle ones that complete
// the warpgroup whose registers go to the softmax warps where TILES = 2).
// A key that the causal mask hides enters P V with weight 0, which an infinity or
// NaN in its V row turns into NaN. So the rows' sums are looked at on their way
// out, and a row with one that is not finite is done again in fp32 from its own
// keys, if such a V row is among those that its tile went through and it does not
// see (24 packed prompts 67.2 -> 68.6 us; a look at the V rows instead, by the load
// warp or in shared memory, cost 5 us and more).
// Every arrival has a waiter before the CTA ends: with two CTAs on an SM their
// products share one queue, and an arrival that came after the CTA's end would
// land in the next one's shared memory.
constexpr int kTile = 128;            // rows of a query tile
constexpr float kBias = 7.0f, kLazy = 8.0f;

template <int DP, int TILES>
struct TcTraits {
  static constexpr int THREADS = TILES == 2 ? 384 : 192;
  static constexpr int BLK = TILES == 2 ? 128 : 64;  // keys of a block
  static constexpr int NBUF = 128 / BLK;             // S buffers of a tile
  static constexpr int HALVES = BLK / 64;            // parts in which P is handed over
  static constexpr int PANELS = DP / 64;            // 128-byte swizzled panels of 64 dims
  static constexpr int QPANEL = kTile * 128, PANEL = BLK * 128;
  static constexpr int QTILE = PANELS * QPANEL, OPERAND = PANELS * PANEL;
  static constexpr int STAGES = 4 * (128 / DP);  // K and V blocks in flight
  static constexpr int OUT = 2048;                   // staging of an output warp: 32 rows x 64 bytes
  static constexpr int OFF_KV = TILES * QTILE;
  static constexpr int OFF_OUT = OFF_KV + STAGES * OPERAND;
  static constexpr int OFF_BAR = OFF_OUT + TILES * 4 * OUT;
  static constexpr int SMEM = OFF_BAR + 768 + 1024;
  static constexpr int COLS = TILES * 256;          // TMEM columns: 128 of S per tile, then O
  static_assert(2 * (SMEM + 1024) <= 233472 || TILES == 2, "two CTAs per SM");
  static_assert(SMEM <= 232448, "shared memory budget");
};

struct TcArgs {
  const int32_t *cu_q, *cu_k;
  int B, Tq, Tk, Hq, Hkv, G, TQ, D, causal, slots, splits;
  float sl;             // scale * log2(e), not negative
  uint32_t flip;        // sign bit where scale < 0: scores are negated first
  void* out;
  float* part;          // splits > 1: [split][Tq * Hq][D] unnormalised outputs
  float2* ml;           //             [split][Tq * Hq] maximum (log2 units), sum
  int* err;
  int redo;             // rows may be done again: causal, and their queries are not overwritten
  const void *q, *k, *v;
  int64_t q_row, q_head, k_row, k_head, v_row, v_head;
  float scale;
};

__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
          smem_u32(dst)),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
      : "memory");
}

// Cluster launch control: takes one CTA that has not started yet out of the
// grid; the answer (16 bytes) arrives at `bar`. After an answer without a CTA
// no further request is made.
__device__ __forceinline__ void cancel_next_cta(void* answer, uint64_t* bar) {
  asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(
                   smem_u32(answer)),
               "r"(smem_u32(bar))
               : "memory");
}
// Its index, -1 where there was none.
__device__ __forceinline__ int cancelled_cta(const void* answer) {
  int x;
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b128 r;\n\t"
      "ld.shared.b128 r, [%1];\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, r;\n\t"
      "mov.b32 %0, -1;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %0, r;\n\t}"
      : "=r"(x)
      : "r"(smem_u32(answer))
      : "memory");
  return x;
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
// The whole warp searches: 32 candidates per step.
__device__ __forceinline__ bool find_work(const TcArgs& a, int tt, int slot, Work& w) {
  const int lane = threadIdx.x & 31;
  int lo = 0, n = a.B;
  while (n > 1) {
    const int step = (n + 31) / 32, mid = lo + lane * step;
    const bool before = mid < lo + n && cut(a.cu_q[mid], a.Tq) / tt + mid <= slot;
    const int last = 31 - __clz(__ballot_sync(0xffffffffu, before) | 1u);
    n = min(step, n - last * step);
    lo += last * step;
  }
  w.q0 = cut(a.cu_q[lo], a.Tq);
  w.lq = cut(a.cu_q[lo + 1], a.Tq) - w.q0;
  w.k0 = cut(a.cu_k[lo], a.Tk);
  w.lk = max(0, cut(a.cu_k[lo + 1], a.Tk) - w.k0);
  w.tok = (slot - (w.q0 / tt + lo)) * tt;
  return w.tok >= 0 && w.tok < w.lq;  // slots in front of the first sequence are empty too
}
// Keys that token i of the sequence sees.
__device__ __forceinline__ int keys_of(const TcArgs& a, const Work& w, int i) {
  return a.causal ? max(0, min(w.lk, i + w.lk - w.lq + 1)) : w.lk;
}
// Blocks of blk keys of tile t (0 when it has no token or sees no key).
__device__ __forceinline__ int blocks_of(const TcArgs& a, const Work& w, int t, int blk) {
  const int first = w.tok + t * a.TQ;
  if (first >= w.lq) return 0;
  return (keys_of(a, w, min(w.lq, first + a.TQ) - 1) + blk - 1) / blk;
}

// A job as the TMA warp hands it to the others; n < 0 ends the CTA.
struct Job {
  Work w;
  int head, split, j0, n;  // KV head, key split, its first block and blocks
  int cnt[2];              // blocks of each tile
};
constexpr int kJobs = 3;   // jobs in the ring

// Rows (bit: row of the warp's 32 of a tile) whose sums are not finite. A row that
// shares its tile's blocks with hidden V rows that are not finite is computed
// from its own keys. Everything is derived anew, so that nothing of it is kept in
// registers before. scratch: 640 bytes of the warp.
template <typename T, int ND, int BLK>
__device__ __forceinline__ void redo_rows(const TcArgs& a, const Job* j, uint8_t* scratch, uint32_t bits) {
  int tid = threadIdx.x;
  asm volatile("" : "+r"(tid), "+l"(j), "+l"(scratch));
  const int lane = tid & 31, t = tid >> 7, first = j->w.tok + t * a.TQ;
  const int begin = j->j0 * BLK, end = min(j->w.lk, (j->j0 + j->cnt[t]) * BLK);  // the tile's keys
  const T* kb = static_cast<const T*>(a.k) + (long long)j->w.k0 * a.k_row + (long long)j->head * a.k_head;
  const T* vb = static_cast<const T*>(a.v) + (long long)j->w.k0 * a.v_row + (long long)j->head * a.v_head;
  float* s_q = reinterpret_cast<float*>(scratch);
#pragma unroll 1
  for (; bits; bits &= bits - 1) {
    const int row = (tid & 96) + __ffs(bits) - 1, g = row % a.G;
    const int tok = first + row / a.G, keys = min(end, keys_of(a, j->w, tok)), lo = max(begin, keys);
    bool odd = false;
#pragma unroll 1
    for (int r = lo; r < end; ++r)
      for (int d = lane; d < a.D; d += 32) odd |= to_f(vb[r * a.v_row + d]) * 0.0f != 0.0f;
    if (!__any_sync(0xffffffffu, odd)) continue;
    const T* q = static_cast<const T*>(a.q) + (long long)(j->w.q0 + tok) * a.q_row + (long long)(j->head * a.G + g) * a.q_head;
    __syncwarp();
    for (int d = lane; d < a.D; d += 32) s_q[d] = to_f(q[d]) * a.scale;
    __syncwarp();
    float m, l, acc[ND];
    attend_keys<true>(kb, vb, a.k_row, a.v_row, a.D, begin, keys, s_q, s_q + ND * 32, m, l, acc);
    const long long at = (long long)(j->w.q0 + tok) * a.Hq + j->head * a.G + g, rows = (long long)a.Tq * a.Hq;
    const float inv = l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l);  // NaN stays NaN
#pragma unroll
    for (int x = 0; x < ND; ++x) {
      const int d = lane + 32 * x;
      if (d >= a.D) continue;
      if (a.splits > 1) a.part[(j->split * rows + at) * a.D + d] = acc[x];
      else store_f(static_cast<T*>(a.out) + at * a.D + d, acc[x] * inv);
    }
    // the other splits' sums carry 2^kBias: as if this m were higher
    if (a.splits > 1 && lane == 0) a.ml[j->split * rows + at] = make_float2(m * 1.44269504088896340736f + kBias, l);
  }
}

template <typename T, int DP, int TILES>
__global__ void __launch_bounds__(TILES == 2 ? 384 : 192, TILES == 2 ? 1 : 2)
    fa_prompt_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                        const __grid_constant__ CUtensorMap map_v, const __grid_constant__ TcArgs a) {
  using R = TcTraits<DP, TILES>;
  constexpr int STAGES = R::STAGES, BLK = R::BLK, NBUF = R::NBUF, HALVES = R::HALVES;
  constexpr int kMmaWarp = TILES * 4, kLoadWarp = kMmaWarp + 1;
  constexpr uint32_t kColO = TILES * 128;  // S of tile t, buffer x at 128 t + BLK x; O of tile t at kColO + DP t
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint64_t* job_full = reinterpret_cast<uint64_t*>(smem + R::OFF_BAR);
  uint64_t* job_empty = job_full + kJobs;
  uint64_t* q_full = job_empty + kJobs;      // [tile]: queries are there
  uint64_t* q_empty = q_full + TILES;        // ... and no product reads them any more
  uint64_t* kv_full = q_empty + TILES;
  uint64_t* kv_empty = kv_full + STAGES;
  uint64_t* s_full = kv_empty + STAGES;      // [tile][buffer]: S is there
  uint64_t* p_full = s_full + NBUF * TILES;  // [tile][half]: 64 keys of P are there
  uint64_t* pv_done = p_full + HALVES * TILES;  // [tile]: the product of a block with V is done (one S buffer: a job's last)
  uint64_t* o_empty = pv_done + TILES;       // [tile]: O is read, the next job may overwrite it
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(o_empty + TILES);
  Job* jobs = reinterpret_cast<Job*>(tmem_slot + 2);
  uint8_t* next = smem + R::OFF_BAR + 704;   // answer to a cancel request (16 bytes), and its barrier
  uint64_t* next_full = reinterpret_cast<uint64_t*>(next + 16);
  static_assert((2 * kJobs + 2 * STAGES + (4 + NBUF + HALVES) * TILES) * 8 + 8 + kJobs * sizeof(Job) <= 704, "barrier area");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kJobs; ++i) {
      mbar_init(&job_full[i], 1);
      mbar_init(&job_empty[i], TILES * 4 + 1);
    }
    for (int i = 0; i < TILES; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&q_empty[i], 1);
      for (int x = 0; x < NBUF; ++x) mbar_init(&s_full[NBUF * i + x], 1);
      for (int x = 0; x < HALVES; ++x) mbar_init(&p_full[HALVES * i + x], 4);
      mbar_init(&pv_done[i], 1);
      mbar_init(&o_empty[i], 4);
    }
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(&kv_full[i], 1);
      mbar_init(&kv_empty[i], 1);
    }
    mbar_init(next_full, 1);
    fence_mbar_init();
  }
  // rows of a query tile that no token fills stay zero
  for (int i = threadIdx.x; i < TILES * R::PANELS * (kTile - a.TQ * a.G) * 8; i += R::THREADS) {
    const int rows = kTile - a.TQ * a.G, c = i % 8, r = i / 8 % rows, panel = i / 8 / rows;
    *reinterpret_cast<uint4*>(smem + panel * R::QPANEL + (a.TQ * a.G + r) * 128 + c * 16) = make_uint4(0, 0, 0, 0);
  }
  fence_proxy_async_smem();
  if (warp == kMmaWarp) tc::tmem_alloc(tmem_slot, R::COLS);
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  bool dead = false;
  // The K and V blocks of a job are loaded in the order they are used: K0 K1 V0
  // K2 V1 .. V(n - 1); item numbers run on from job to job.
  auto item_k = [](int i) { return i == 0 ? 0 : 2 * i - 1; };
  auto item_v = [](int i, int n) { return i + 1 == n ? 2 * i + 1 : 2 * i + 2; };
  // Job c, for the warps that work on it; they read it in place until they are
  // done with it.
  auto take_job = [&](int c) -> const Job& {
    mbar_wait_or_poison(&job_full[c % kJobs], (c / kJobs) & 1, a.err, DEV_TIMEOUT_FULL, dead);
    return jobs[c % kJobs];
  };
  auto finish_job = [&](int c) {
    __syncwarp();
    if (lane == 0) mbar_arrive(&job_empty[c % kJobs]);
  };

  // 384 x 168 registers at launch: 256 x 216 + 128 x 72
  if constexpr (TILES == 2) {
    if (warp >= kMmaWarp) asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
  }
  if (warp == kLoadWarp) {
    if (lane == 0) {
      tc::prefetch_tmap(&map_q);
      tc::prefetch_tmap(&map_k);
      tc::prefetch_tmap(&map_v);
    }
    int c = 0, items = 0, queries[TILES];  // jobs, K / V blocks and query tiles so far
#pragma unroll
    for (int t = 0; t < TILES; ++t) queries[t] = 0;
    auto push = [&](const Job& j) {
      if (c >= kJobs) mbar_wait_idle_or_poison(&job_empty[c % kJobs], ((c / kJobs) - 1) & 1, a.err, DEV_TIMEOUT_EMPTY, dead);
      __syncwarp();
      if (lane == 0) {
        jobs[c % kJobs] = j;
        mbar_arrive(&job_full[c % kJobs]);
      }
      ++c;
    };
    // The CTA's first job is its own index; further ones are those of CTAs that
    // have not started yet, which it cancels one by one (later tiles of a
    // causal sequence see more keys and have the lower indexes). A job is taken
    // once the loads of the last one are out: late enough for an even end.
    for (int id = blockIdx.x, round = 0; id >= 0 && !dead; ++round) {
      Job j;
      j.head = id % a.Hkv;
      j.split = id / a.Hkv % a.splits;
      const bool real = find_work(a, a.TQ * TILES, a.slots - 1 - id / a.Hkv / a.splits, j.w);
      if (real) {
        int n = 0;
#pragma unroll
        for (int t = 0; t < TILES; ++t) j.cnt[t] = blocks_of(a, j.w, t, BLK), n = max(n, j.cnt[t]);
        j.j0 = (int)((long long)n * j.split / a.splits);
        const int j1 = (int)((long long)n * (j.split + 1) / a.splits);
#pragma unroll
        for (int t = 0; t < TILES; ++t) j.cnt[t] = max(0, min(j.cnt[t], j1) - j.j0);
        j.n = n = j1 - j.j0;
        push(j);
        if (lane == 0) {
#pragma unroll
          for (int t = 0; t < TILES; ++t) {
            if (j.cnt[t] == 0) continue;
            if (queries[t] > 0) mbar_wait_idle_or_poison(&q_empty[t], (queries[t] - 1) & 1, a.err, DEV_TIMEOUT_EMPTY, dead);
            ++queries[t];
            mbar_arrive_expect_tx(&q_full[t], R::PANELS * a.TQ * a.G * 128);
            for (int p = 0; p < R::PANELS; ++p)
              tma_load_3d(smem + t * R::QTILE + p * R::QPANEL, &map_q, p * 64, j.head * a.G, j.w.q0 + j.w.tok + t * a.TQ,
                          &q_full[t]);
          }
          for (int x = 0; x < 2 * n; ++x, ++items) {
            const bool is_v = x > 0 && ((x & 1) == 0 || x + 1 == 2 * n);
            const int i = x == 0 ? 0 : is_v ? (x + 1 == 2 * n ? n - 1 : (x - 2) >> 1) : (x + 1) >> 1;
            const int st = items % STAGES;
            if (items >= STAGES)
              mbar_wait_idle_or_poison(&kv_empty[st], ((items / STAGES) - 1) & 1, a.err, DEV_TIMEOUT_EMPTY, dead);
            mbar_arrive_expect_tx(&kv_full[st], R::OPERAND);
            for (int p = 0; p < R::PANELS; ++p)
              tma_load_3d(smem + R::OFF_KV + st * R::OPERAND + p * R::PANEL, is_v ? &map_v : &map_k, p * 64, j.head,
                          j.w.k0 + (j.j0 + i) * BLK, &kv_full[st]);
          }
        }
      }
      if (lane == 0) {
        mbar_arrive_expect_tx(next_full, 16);
        cancel_next_cta(next, next_full);
        mbar_wait_idle_or_poison(next_full, round & 1, a.err, DEV_TIMEOUT_FULL, dead);
        id = dead ? -1 : cancelled_cta(next);
        fence_proxy_async_smem();  // read before it is written again
      }
      id = __shfl_sync(0xffffffffu, id, 0);
      dead = __shfl_sync(0xffffffffu, (int)dead, 0) != 0;
    }
    Job last{};
    last.n = -1;
    push(last);
    if (lane == 0) {
      // the releases that no load waited for
      for (int x = max(0, items - STAGES); x < items; ++x)
        mbar_wait_idle_or_poison(&kv_empty[x % STAGES], (x / STAGES) & 1, a.err, DEV_TIMEOUT_EMPTY, dead);
#pragma unroll
      for (int t = 0; t < TILES; ++t)
        if (queries[t] > 0) mbar_wait_idle_or_poison(&q_empty[t], (queries[t] - 1) & 1, a.err, DEV_TIMEOUT_EMPTY, dead);
    }
    __syncwarp();
  } else if (warp == kMmaWarp) {
    constexpr uint32_t idesc_s = idesc<T>(BLK, false), idesc_o = idesc<T>(DP, true);
    const uint32_t q_base = smem_u32(smem), kv_base = q_base + R::OFF_KV;
    const uint32_t go = tc::elect_one();
    int items = 0, done[TILES], queries[TILES];  // K / V blocks of earlier jobs; blocks and jobs of each tile so far
#pragma unroll
    for (int t = 0; t < TILES; ++t) done[t] = queries[t] = 0;
    for (int c = 0;; ++c) {
      const Job& j = take_job(c);
      if (dead || j.n < 0) break;
      const int n = j.n;
      // S_t = Q_t K_i^T into the tile's next buffer
      auto score = [&](int t, int i) {
        const int x = items + item_k(i), st = x % STAGES, u = done[t] + i;
        mbar_wait_or_poison(&kv_full[st], (x / STAGES) & 1, a.err, DEV_TIMEOUT_FULL, dead);
        if (i == 0) mbar_wait_or_poison(&q_full[t], queries[t] & 1, a.err, DEV_TIMEOUT_FULL, dead);
        tc::tc_fence_after();
        const uint64_t kd = tc::sw128_desc(kv_base + st * R::OPERAND), qd = tc::sw128_desc(q_base + t * R::QTILE);
#pragma unroll
        for (int k = 0; k < DP / 16; ++k)
          tc::mma_ss_go(tmem + t * 128 + (u % NBUF) * BLK, qd + (uint64_t)((k >> 2) * (R::QPANEL >> 4) + (k & 3) * 2),
                        kd + (uint64_t)((k >> 2) * (R::PANEL >> 4) + (k & 3) * 2), idesc_s, k > 0, go);
        tc::mma_commit_go(&s_full[NBUF * t + u % NBUF], go);
        if (i + 1 == j.cnt[t]) tc::mma_commit_go(&q_empty[t], go);
      };
      auto release = [&](int x) { tc::mma_commit_go(&kv_empty[(items + x) % STAGES], go); };
      if (n > 0) {
#pragma unroll
        for (int t = 0; t < TILES; ++t)
          if (j.cnt[t] > 0) score(t, 0);
        release(0);
      }
      for (int i = 0; i < n; ++i) {
        if (NBUF == 2 && i + 1 < n) {
          // the other buffer held P of block i - 1, whose product was issued before
#pragma unroll
          for (int t = 0; t < TILES; ++t)
            if (i + 1 < j.cnt[t]) score(t, i + 1);
          release(item_k(i + 1));
        }
        const int x = items + item_v(i, n), st = x % STAGES;
        mbar_wait_or_poison(&kv_full[st], (x / STAGES) & 1, a.err, DEV_TIMEOUT_FULL, dead);
        const uint64_t vd = tc::sw128_desc_mn(kv_base + st * R::OPERAND, R::PANEL);  // dims across, tokens down
#pragma unroll
        for (int t = 0; t < TILES; ++t) {
          if (i >= j.cnt[t]) continue;
          const int u = done[t] + i;
          if (i == 0 && queries[t] > 0)  // the tile's last O is read
            mbar_wait_or_poison(&o_empty[t], (queries[t] - 1) & 1, a.err, DEV_TIMEOUT_EMPTY, dead);
#pragma unroll
          for (int h = 0; h < HALVES; ++h) {
            mbar_wait_or_poison(&p_full[HALVES * t + h], u & 1, a.err, DEV_TIMEOUT_FULL, dead);
            tc::tc_fence_after();
#pragma unroll
            for (int k = 4 * h; k < 4 * h + 4; ++k)
              tc::mma_ts_go(tmem + kColO + t * DP, tmem + t * 128 + (u % NBUF) * BLK + 8 * k, vd + (uint64_t)(k * (2048 >> 4)),
                            idesc_o, (i > 0 || k > 0) ? 1u : 0u, go);
          }
          if (NBUF == 2 || i + 1 == j.cnt[t]) tc::mma_commit_go(&pv_done[t], go);
          // one buffer: the next scores take the place of the P just consumed (the products run in order)
          if (NBUF == 1 && i + 1 < j.cnt[t]) score(t, i + 1);
        }
        release(item_v(i, n));
        if (NBUF == 1 && i + 1 < n) release(item_k(i + 1));
      }
      items += 2 * n;
#pragma unroll
      for (int t = 0; t < TILES; ++t) done[t] += j.cnt[t], queries[t] += j.cnt[t] > 0;
      finish_job(c);
    }
    __syncwarp();
  } else if (warp < kMmaWarp) {
    if constexpr (TILES == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    const int t = warp >> 2, row = threadIdx.x & 127, rt = row / a.G, g = row % a.G;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_addr = tmem + lanes + t * 128, o_addr = tmem + lanes + kColO + t * DP;
    uint8_t* stage = smem + R::OFF_OUT + warp * R::OUT;
    int items = 0, done = 0, ended = 0;  // K / V blocks of earlier jobs, this tile's blocks and jobs so far
    for (int c = 0;; ++c) {
      const Job& j = take_job(c);
      if (dead || j.n < 0) break;
      const Work& w = j.w;
      const int nt = j.cnt[t];
      const int first = w.tok + t * a.TQ;                     // the tile's first token
      const int tok = first + rt;
      const bool mine = row < a.TQ * a.G && tok < w.lq;
      const int keys = mine ? keys_of(a, w, tok) : 0;
      const int all_see = keys_of(a, w, first);               // keys that every row of the tile sees
      float m = -INFINITY;
      F2 l2 = f2(0.0f, 0.0f);
      for (int i = 0; i < nt; ++i) {
        const int key0 = (j.j0 + i) * BLK, u = done + i;
        const uint32_t sp = s_addr + (u % NBUF) * BLK;
        mbar_wait_or_poison(&s_full[NBUF * t + u % NBUF], (u / NBUF) & 1, a.err, DEV_TIMEOUT_FULL, dead);
        __syncwarp();
        tc::tc_fence_after();
        uint32_t s[BLK];
#pragma unroll
        for (int x = 0; x < BLK; x += 32) tc::tmem_ld32(sp + x, *reinterpret_cast<uint32_t(*)[32]>(s + x));
        tc::tmem_ld_wait();
        if (a.flip) {
#pragma unroll
          for (int x = 0; x < BLK; ++x) s[x] ^= a.flip;
        }
        if (key0 + BLK > all_see) {
          const int lim = keys - key0;
#pragma unroll
          for (int x = 0; x < BLK; ++x)
            if (x >= lim) s[x] = 0xff800000u;
          const int valid = w.lk - key0;
          if (valid < BLK) {
            // rows of V behind the sequence's end belong to others: what they
            // hold must not meet P (0 x inf); both tiles write the same zeros
            const int v = items + item_v(i, j.n), st = v % STAGES;
            mbar_wait_or_poison(&kv_full[st], (v / STAGES) & 1, a.err, DEV_TIMEOUT_FULL, dead);
            for (int x = row; x < (BLK - valid) * 8 * R::PANELS; x += kTile) {
              const int y = x % 8, p = x / 8 % R::PANELS, r = valid + x / (8 * R::PANELS);
              *reinterpret_cast<uint4*>(smem + R::OFF_KV + st * R::OPERAND + p * R::PANEL + r * 128 + y * 16) =
                  make_uint4(0, 0, 0, 0);
            }
            fence_proxy_async_smem();
          }
        }
        const float mn = row_max(s) * a.sl;
        float f = 1.0f;
        if (mn > m + kLazy) {  // also the row's first keys (m = -inf)
          f = ex2(m - mn);
          m = mn;
          l2 = mul2(l2, f2(f, f));
        }
        // Before O is touched the product of the block before must be done. With
        // one buffer it is, as S came after it, and pv_done arrives at a job's end
        // only; with two, its arrival (normally long there) is taken before this
        // block's P goes out. Either way no wait falls two arrivals behind, where
        // the parity would let it through early.
        if (NBUF == 2 && i > 0) mbar_wait_or_poison(&pv_done[t], (u - 1) & 1, a.err, DEV_TIMEOUT_FULL, dead);
        if (i > 0 && __any_sync(0xffffffffu, f != 1.0f)) {
          __syncwarp();
          tc::tc_fence_after();
          rescale_row(o_addr, DP, f);
        }
        const float off = m == -INFINITY ? 0.0f : kBias - m;
        const F2 sl2 = f2(a.sl, a.sl), off2 = f2(off, off);
        F2 sum = f2(0.0f, 0.0f);
#pragma unroll
        for (int h = 0; h < HALVES; ++h) {
          uint32_t p[32];
#pragma unroll
          for (int x = 0; x < 32; ++x) {
            const F2 e = fma2(f2(__uint_as_float(s[64 * h + 2 * x]), __uint_as_float(s[64 * h + 2 * x + 1])), sl2, off2);
            float e0, e1;
            unpack(e, e0, e1);
            e0 = ex2(e0), e1 = ex2(e1);
            sum = add2(sum, f2(e0, e1));
            p[x] = pack2<T>(e0, e1);
          }
          __syncwarp();
          tc::tmem_st32(sp + 32 * h, p);
          tc::tmem_st_wait();
          tc::tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_full[HALVES * t + h]);
        }
        l2 = add2(l2, sum);
      }
      done += nt;
      items += 2 * j.n;
      float l, l1;
      unpack(l2, l, l1);
      l += l1;
      if (nt > 0) {
        mbar_wait_or_poison(&pv_done[t], (NBUF == 2 ? done - 1 : ended) & 1, a.err, DEV_TIMEOUT_FULL, dead);
        ++ended;
        __syncwarp();
        tc::tc_fence_after();
      }
      const bool none = m == -INFINITY && l == l;             // no key seen (a NaN score is one)
      // rows leave through shared memory, 64 bytes of each at a time
      const int at = mine ? (w.q0 + tok) * a.Hq + j.head * a.G + g : -1;
      const float inv = 1.0f / l;
      const bool partial = a.splits > 1;
      const int cols = partial ? 16 : 32, item = partial ? 4 : 2;  // columns of 64 bytes, bytes of an element
      uint8_t* base = partial ? reinterpret_cast<uint8_t*>(a.part + (long long)j.split * a.Tq * a.Hq * a.D)
                              : static_cast<uint8_t*>(a.out);
      if (partial && mine)
        a.ml[(long long)j.split * a.Tq * a.Hq + at] = make_float2(none ? -INFINITY : m, none ? 0.0f : l);
      uint8_t* dst[4];                                        // of the pieces this lane stores, rows lane / 4 + 8 x
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int r = __shfl_sync(0xffffffffu, at, 8 * x + (lane >> 2));
        dst[x] = r >= 0 ? base + (long long)r * a.D * item + (lane & 3) * 16 : nullptr;
      }
      F2 odd[2] = {f2(0.0f, 0.0f), f2(0.0f, 0.0f)};           // NaN after a sum that is not finite
#pragma unroll 1
      for (int x0 = 0; x0 < a.D; x0 += 32) {
        uint32_t o[32];
        __syncwarp();
        if (nt > 0) {
          tc::tmem_ld32(o_addr + x0, o);
          tc::tmem_ld_wait();
          if (x0 + 32 >= a.D) {
            tc::tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&o_empty[t]);
          }
        }
        if (none) {
#pragma unroll
          for (int x = 0; x < 32; ++x) o[x] = 0;
        }
#pragma unroll
        for (int x = 0; x < 16; ++x)
          odd[x & 1] = fma2(f2(__uint_as_float(o[2 * x]), __uint_as_float(o[2 * x + 1])), f2(0.0f, 0.0f), odd[x & 1]);
        if (!partial) {
#pragma unroll
          for (int x = 0; x < 16; ++x)
            o[x] = none ? 0u : pack2<T>(__uint_as_float(o[2 * x]) * inv, __uint_as_float(o[2 * x + 1]) * inv);
        }
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          if (half == 1 && !partial) break;
          __syncwarp();
#pragma unroll
          for (int x = 0; x < 4; ++x)
            *stage_row(stage, lane, x) =
                make_uint4(o[16 * half + 4 * x], o[16 * half + 4 * x + 1], o[16 * half + 4 * x + 2], o[16 * half + 4 * x + 3]);
          __syncwarp();
          uint4 v[4];
#pragma unroll
          for (int x = 0; x < 4; ++x) v[x] = *stage_piece(stage, lane, x);
          const int col = x0 + cols * half;
          const bool inside = (col * item + (lane & 3) * 16) < a.D * item;
#pragma unroll
          for (int x = 0; x < 4; ++x)
            if (dst[x] && inside) *reinterpret_cast<uint4*>(dst[x] + col * item) = v[x];
        }
      }
      float odd0, odd1;
      unpack(add2(odd[0], odd[1]), odd0, odd1);
      const uint32_t again = __ballot_sync(0xffffffffu, mine && nt > 0 && odd0 + odd1 != 0.0f);
      if (a.redo && again) redo_rows<T, DP / 32, BLK>(a, &j, stage, again);
      finish_job(c);
    }
  }
  tc::tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) tc::tmem_dealloc(tmem, R::COLS);
}

// Merges the splits of a row: one warp per (row, query head), 4 dims per lane.
// A split that saw none of the row's keys has l = 0 and no output.
template <typename T>
__global__ void __launch_bounds__(256) fa_prompt_combine_kernel(const TcArgs a) {
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const long long rows = (long long)a.Tq * a.Hq, row = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (row >= rows) return;
  const float2 s = lane < a.splits ? a.ml[lane * rows + row] : make_float2(-INFINITY, 0.0f);
  const float M = warp_max(s.x), base = M == -INFINITY ? 0.0f : M;
  const float wgt = s.y == 0.0f ? 0.0f : ex2(s.x - base);
  float L = wgt * s.y;
#pragma unroll
  for (int x = 16; x >= 1; x >>= 1) L += __shfl_xor_sync(0xffffffffu, L, x);
  float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
  for (int i = 0; i < a.splits; ++i) {
    const float wi = __shfl_sync(0xffffffffu, wgt, i), li = __shfl_sync(0xffffffffu, s.y, i);
    if (li == 0.0f || 4 * lane >= a.D) continue;
    const float4 v = *reinterpret_cast<const float4*>(a.part + (i * rows + row) * a.D + 4 * lane);
    o.x = fmaf(wi, v.x, o.x), o.y = fmaf(wi, v.y, o.y), o.z = fmaf(wi, v.z, o.z), o.w = fmaf(wi, v.w, o.w);
  }
  const float inv = L == 0.0f ? 0.0f : 1.0f / L;
  if (4 * lane < a.D)
    *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + row * a.D + 4 * lane) =
        make_uint2(pack2<T>(o.x * inv, o.y * inv), pack2<T>(o.z * inv, o.w * inv));
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
  return a.D <= 128 && a.Hq / a.Hkv <= kTile && a.Tk > 0 && (int64_t)a.Tq * a.Hq <= INT32_MAX && tma_rows(a.q, a.Hq, a.Tq, a.q_head, a.q_row) &&
         tma_rows(a.k, a.Hkv, a.Tk, a.k_head, a.k_row) && tma_rows(a.v, a.Hkv, a.Tk, a.v_head, a.v_row);
}

// How a call is cut up.
struct Plan {
  int tiles, slots, splits;  // query tiles per CTA, CTAs per KV head, key splits
};
constexpr int kMaxSplits = 32;
Plan plan_of(const FaPromptArgs& a) {
  const int TQ = kTile / (a.Hq / a.Hkv);
  const long long keys = a.Tk / std::max(a.B, 1);  // per sequence, on average
  Plan p;
  // two tiles per CTA where sequences are long (us for 8192 tokens of equal
  // sequences, 32 heads over 8 of 128, one tile and two: 256 each 52 and 56, 768
  // 75 and 80, 1024 95 and 96, 2048 158 and 152, 8192 521 and 480; heads of 64: 512
  // 58 and 64, 1024 82 and 85, 2048 135 and 130; 16 ungrouped heads: 45 and 49, 60
  // and 62, 86 and 84; 8 heads over one: 27 and 31, 38 and 41, 58 and 58)
  p.tiles = keys >= 1024 ? 2 : 1;
  p.slots = a.Tq / (TQ * p.tiles) + a.B;
  // few CTAs against many keys: split the keys so that the SMs are full once,
  // with at least 512 keys each (256 rows against 24000 keys: 110 us in 4 parts,
  // which leave 20 SMs idle; 109 in 9, 121 in 13)
  const long long ctas = ((a.Tq + (long long)TQ * p.tiles - 1) / (TQ * p.tiles)) * a.Hkv;
  const long long room = (long long)sm_count() * (p.tiles == 2 ? 1 : 2);
  p.splits = (int)std::max(1ll, std::min({room / std::max(ctas, 1ll), keys / 512, (long long)kMaxSplits}));
  return p;
}

template <typename T, int DP, int TILES>
kq_status_t launch_tc(const FaPromptArgs& a, int dtype, const Plan& plan, cudaStream_t s) {
  using R = TcTraits<DP, TILES>;
  TcArgs p{};
  p.cu_q = a.cu_q, p.cu_k = a.cu_k;
  p.B = a.B, p.Tq = a.Tq, p.Tk = a.Tk, p.Hq = a.Hq, p.Hkv = a.Hkv, p.D = a.D, p.causal = a.causal;
  p.G = a.Hq / a.Hkv;
  p.TQ = kTile / p.G;
  p.slots = plan.slots;
  p.splits = plan.splits;
  const float sl = a.scale * 1.44269504088896340736f;
  p.flip = sl < 0.0f ? 0x80000000u : 0u;
  p.sl = fmaxf(fabsf(sl), 1e-30f);  // a scale of 0 keeps -inf for hidden keys
  p.out = a.out;
  p.part = static_cast<float*>(a.ws);
  p.ml = reinterpret_cast<float2*>(p.part + (size_t)plan.splits * a.Tq * a.Hq * a.D);
  p.err = device_error_word();
  p.q = a.q, p.k = a.k, p.v = a.v;
  p.q_row = a.q_row, p.q_head = a.q_head, p.k_row = a.k_row, p.k_head = a.k_head, p.v_row = a.v_row, p.v_head = a.v_head;
  p.scale = a.scale;
  const char *q0 = static_cast<const char*>(a.q), *o0 = static_cast<const char*>(a.out);
  const int64_t q_bytes = 2 * ((a.Tq - 1) * (a.Tq > 1 ? a.q_row : 0) + (a.Hq - 1) * (a.Hq > 1 ? a.q_head : 0) + a.D);
  p.redo = a.causal && (q0 + q_bytes <= o0 || o0 + 2 * (int64_t)a.Tq * a.Hq * a.D <= q0);
  CUtensorMap mq, mk, mv;
  if (!encode_rows(&mq, dtype, a.q, a.D, a.Hq, a.Tq, a.q_head, a.q_row, p.G, p.TQ) ||
      !encode_rows(&mk, dtype, a.k, a.D, a.Hkv, a.Tk, a.k_head, a.k_row, 1, R::BLK) ||
      !encode_rows(&mv, dtype, a.v, a.D, a.Hkv, a.Tk, a.v_head, a.v_row, 1, R::BLK))
    return fail(KQ_ERR_CUDA, "fa_prompt: tensor map encoding failed");
  auto kernel = fa_prompt_tc_kernel<T, DP, TILES>;
  if (kq_status_t st = ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), R::SMEM, "fa_prompt")) return st;
  kernel<<<(unsigned)(plan.slots * a.Hkv * plan.splits), R::THREADS, R::SMEM, s>>>(mq, mk, mv, p);
  if (kq_status_t st = check_launch("fa_prompt_tc")) return st;
  if (p.splits == 1) return KQ_OK;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(((long long)a.Tq * a.Hq + 7) / 8));
  cfg.blockDim = dim3(256);
  cfg.stream = s;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return check_cuda(cudaLaunchKernelEx(&cfg, fa_prompt_combine_kernel<T>, p), "fa_prompt_combine");
}
template <typename T>
kq_status_t launch_tc_any(const FaPromptArgs& a, int dtype, cudaStream_t s) {
  const Plan p = plan_of(a);
  if (a.D <= 64) return p.tiles == 2 ? launch_tc<T, 64, 2>(a, dtype, p, s) : launch_tc<T, 64, 1>(a, dtype, p, s);
  return p.tiles == 2 ? launch_tc<T, 128, 2>(a, dtype, p, s) : launch_tc<T, 128, 1>(a, dtype, p, s);
}

}  // namespace

size_t fa_prompt_workspace(const FaPromptArgs& a) {
  if (a.D > 128 || a.Hq / a.Hkv > kTile || a.Tq == 0) return 0;
  const int splits = plan_of(a).splits;
  return splits == 1 ? 0 : (size_t)splits * a.Tq * a.Hq * (a.D * sizeof(float) + sizeof(float2));
}

kq_status_t launch_fa_prompt(const FaPromptArgs& a, int dtype, cudaStream_t s) {
  if (tc_supported(a))
    return dtype == KQ_F16 ? launch_tc_any<__half>(a, dtype, s) : launch_tc_any<__nv_bfloat16>(a, dtype, s);
  const long long items = (long long)a.Tq * a.Hq;
  const unsigned grid = (unsigned)((items + kSimpleWarps - 1) / kSimpleWarps);
  if (dtype == KQ_F16) fa_prompt_simple_kernel<__half><<<grid, kSimpleWarps * 32, 0, s>>>(a);
  else fa_prompt_simple_kernel<__nv_bfloat16><<<grid, kSimpleWarps * 32, 0, s>>>(a);
  return check_launch("fa_prompt");
}

}  // namespace kq
