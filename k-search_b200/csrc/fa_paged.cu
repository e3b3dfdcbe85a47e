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
#include <algorithm>
#include <cmath>

#include "kq_internal.h"
#include "kq_attn.cuh"
#include "kq_device.cuh"
#include "kq_tc.cuh"

namespace kq {
namespace {

using namespace attn;

constexpr int kQ8 = 34;
constexpr int kMaxNB = 8;

// ---- work split ------------------------------------------------------------------
// Tokens start .. n_b - 1 of every sequence (n_b its length, cut to max_seqlen
// and the table) are cut into units of 16 at multiples of 16 (so that 8 rows
// of a unit are neighbours in one page); a KV head's units of all sequences
// in a row are divided evenly among C workers, whatever the lengths are.
// Worker c takes U / C units in order, the first U % C one more; the part inside
// sequence b is one segment with its own softmax state, stored at index c + b
// (unique: c and b only grow along the row).
constexpr int kUnit = 16;

struct Split {
  const int32_t* seq_lens;
  int B, start, limit;  // limit: min(max_seqlen, W * ps)
  int workers;          // upper bound of C
  __device__ __forceinline__ int len(int b) const { return max(0, min(seq_lens[b], limit)); }
  __device__ __forceinline__ int first() const { return start & ~(kUnit - 1); }
  __device__ __forceinline__ int units(int b) const {
    const int n = len(b);
    return n > start ? (n - first() + kUnit - 1) / kUnit : 0;
  }
  // C for U units: at least kMinUnits each (one sequence of up to 800 tokens: 8.9
  // us with 2, 11.0 with 3, 12.2 with 4; 1 changes nothing)
  __device__ __forceinline__ int active(int U) const { return max(1, min(workers, U / kMinUnits)); }
  static constexpr int kMinUnits = 2;
};
struct Shares {
  int base, rem;
  __device__ __forceinline__ Shares(int U, int C) : base(U / C), rem(U % C) {}
  __device__ __forceinline__ int begin(int c) const { return c * base + min(c, rem); }
  // the worker that has unit u (base > 0 where there is more than one worker)
  __device__ __forceinline__ int worker(int u) const {
    const int head = rem * (base + 1);
    return u < head ? u / (base + 1) : rem + (u - head) / max(base, 1);
  }
};

// Prefix sums of the units of B sequences, T contiguous runs of them (one per
// thread): scan[i] = units before run i, scan[T] = all.
template <int T>
struct SplitScan {
  int scan[T + 1];
  int warp_sums[T / 32];
};
template <int T>
__device__ __forceinline__ int run_len(const Split& sp) {
  return (sp.B + T - 1) / T;
}
template <int T>
__device__ __forceinline__ void scan_units(const Split& sp, SplitScan<T>& ss) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, per = run_len<T>(sp);
  int v = 0;
  for (int b = tid * per; b < min(sp.B, (tid + 1) * per); ++b) v += sp.units(b);
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int t = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += t;
  }
  if (lane == 31) ss.warp_sums[warp] = v;
  __syncthreads();
  for (int i = 0; i < warp; ++i) v += ss.warp_sums[i];
  ss.scan[tid + 1] = v;
  if (tid == 0) ss.scan[0] = 0;
  __syncthreads();
}
// Units before sequence b.
template <int T>
__device__ __forceinline__ int units_before(const Split& sp, const SplitScan<T>& ss, int b) {
  const int per = run_len<T>(sp), run = b / per;
  int u = ss.scan[run];
  for (int i = run * per; i < b; ++i) u += sp.units(i);
  return u;
}

// ---- streaming kernel --------------------------------------------------------------
// A warp streams one worker's tokens of one KV head (for up to 16 of its query
// heads): 16-token K and V rows arrive by 16-byte asynchronous copies, from the
// 16-byte boundary below each row, in its own ring of stages, so no two warps
// wait for each other; neighbouring warps hold neighbouring heads of the same
// tokens. Products on mma.m16n8k16 with 16 tokens (scores) or 16 dimensions
// (output) as rows and 8 query heads as columns, twice where a group has more:
//   S^T[t, h] = sum_j d_k(t, j) (codes_j . q_j): exact fp16 codes per 32-dim
//     block j, rescaled in fp32, then transposed between the lanes;
//   O^T[:, h] += sum_t codes (p d_v(t, j)): the value block's scale folded into
//     p in fp32, rounded to fp16 once (the codes are exact). Like the output's
//     own rounding that is 2^-11 of each weight, and the weights' errors average
//     out. p carries 2^e with e from the segment's largest d_v so far, so that p d_v
//     stays below 2^15 for every fp16 d_v and the light weights of small values
//     stay in fp16's normal range (down to 2^-29 of the largest possible p d_v).
// With the heads as rows half of every product was empty: 16 conversations of
// 16000 tokens (8 KV heads of 128) took 101 us instead of 89. The head dimension
// is permuted inside a block so that every operand word is one 32-bit load (a
// word of 4 codes) per lane.
// Those conversations are 310 MB: 85.6 us, 3.6 TB/s (84 with a constant 2^e). The
// copies alone take 55; about 600 instructions per 16 tokens and head go beside
// them (codes to fp16, scales, addresses), at 2.2 instructions a clock and SM with
// 12 warps. 14 and 16 warps took 81 and 84 us there, but 1 and 2 us more where
// sequences are short.
constexpr int kStreamWarps = 12;  // 12 warps with 3 stages, or 8 with 6 where there is little to stream
constexpr int kFewWarps = 8;
constexpr float kMaxExp = 40.0f;   // e of a segment without a value scale so far (2^-24 alone needs 38)

template <int NB>
struct Row {
  static constexpr int BYTES = NB * kQ8;
  static constexpr int UNITS16 = BYTES & 15;  // heads and tokens move the row start by multiples of this mod 16
  static constexpr int STEP = UNITS16 == 0 ? 16 : (UNITS16 & 2) ? 2 : (UNITS16 & 4) ? 4 : 8;
  static constexpr int NEED = (BYTES + 16 - STEP + 15) / 16 * 16;
  static constexpr int PITCH = (NEED / 16) % 2 ? NEED : NEED + 16;  // odd multiple of 16: 8 rows hit distinct banks
  static constexpr int CHUNKS = NEED / 16;    // 16-byte pieces of a row
  static constexpr int COPIES = (8 * CHUNKS + 31) / 32;  // per lane, for 8 rows
  static constexpr bool ALWAYS = 16 * (CHUNKS - 1) < BYTES;  // every piece holds bytes of the row wherever it starts
  static constexpr int STAGE = 2 * kUnit * PITCH;
};
// A warp's ring: fewer stages where the rows are long.
template <int NB, int WARPS>
struct Ring {
  static constexpr int MOST = WARPS == kStreamWarps ? 3 : 6;
  static constexpr int STAGES = std::min(MOST, 221184 / (WARPS * Row<NB>::STAGE));
  static constexpr int SMEM = WARPS * STAGES * Row<NB>::STAGE;
};

// 16 bytes to shared memory, asynchronously (groups of them are waited for).
__device__ __forceinline__ void copy16(uint32_t dst, const uint8_t* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
// This lane's pieces of 8 cache rows of one head: rows start at multiples of
// `row_bytes` from a 16-byte aligned place, plus head_off. The pieces run
// along the rows, so a warp's copy instruction covers whole row segments.
template <int NB>
struct Pieces {
  using R = Row<NB>;
  int src[R::COPIES];  // from the first row's start; -1: none
  int dst[R::COPIES];
  __device__ __forceinline__ Pieces(int lane, long long row_bytes, int head_off) {
#pragma unroll
    for (int i = 0; i < R::COPIES; ++i) {
      const int x = lane + 32 * i, r = x / R::CHUNKS, c = x % R::CHUNKS;
      const int at = (int)(r * row_bytes) + head_off, off = at & 15;
      src[i] = r < 8 && (R::ALWAYS || 16 * c < off + R::BYTES) ? at - off + 16 * c : -1;
      dst[i] = r * R::PITCH + 16 * c;
    }
  }
  __device__ __forceinline__ void copy(uint32_t to, const uint8_t* from) const {
#pragma unroll
    for (int i = 0; i < R::COPIES; ++i)
      if (src[i] >= 0) copy16(to + dst[i], from + (uint32_t)src[i]);
  }
};

struct StreamArgs {
  const void* q;
  int q_bf16;
  const uint8_t *k, *v;
  long long num_pages;
  int ps, W, Hq, Hkv, G, QG;  // QG groups of up to 16 query heads per KV head
  const int32_t* table;
  int prefix_len;  // tokens below it (a multiple of 8) lie in row 0's pages
  Split split;
  int warps;    // per CTA
  float sl;     // scale * log2(e)
  float* part;  // [segment][Hq][NB * 32] accumulators
  float2* ml;   // [segment][Hq] maximum (log2 units), sum
};

// d = a b + (c0, c1, c2, c3)
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, float c0, float c1,
                                         float c2, float c3) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}
// The 8 x 8 matrix with elements (g, 2 c) and (g, 2 c + 1) in lane 4 g + c,
// transposed: halves of the 32-bit values in two 16-bit transpositions.
__device__ __forceinline__ uint32_t movm(uint32_t a) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
__device__ __forceinline__ void transpose8(float x0, float x1, float& y0, float& y1) {
  const uint32_t a = __float_as_uint(x0), b = __float_as_uint(x1);
  const uint32_t lo = movm(__byte_perm(a, b, 0x5410)), hi = movm(__byte_perm(a, b, 0x7632));
  y0 = __uint_as_float(__byte_perm(lo, hi, 0x5410));
  y1 = __uint_as_float(__byte_perm(lo, hi, 0x7632));
}
__device__ __forceinline__ uint32_t hsub2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
// 4 codes (one word) -> two fp16 pairs: 0x64uu is 1024 + uu, uu = code + 128.
__device__ __forceinline__ void codes_h2(uint32_t w, uint32_t& lo, uint32_t& hi) {
  const uint32_t u = w ^ 0x80808080u;
  lo = hsub2(__byte_perm(u, 0x64646464u, 0x4140), 0x64806480u);
  hi = hsub2(__byte_perm(u, 0x64646464u, 0x4342), 0x64806480u);
}
// The 32-bit word `off` bytes (even) behind `at` in shared memory. Rows of an
// even number of blocks start at multiples of 4, so a constant `off` decides
// between one load and two; the others decide per lane.
template <int NB>
__device__ __forceinline__ uint32_t word_at(const uint8_t* at, int off) {
  if constexpr (NB % 2 == 0) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(at + (off & ~3));
    return (off & 2) ? __funnelshift_r(w[0], w[1], 16) : w[0];
  } else {
    const uintptr_t x = reinterpret_cast<uintptr_t>(at) + off;
    const uint32_t* w = reinterpret_cast<const uint32_t*>(x & ~(uintptr_t)3);
    return (x & 2) ? __funnelshift_r(w[0], w[1], 16) : w[0];
  }
}

// A position in a worker's row of units.
struct Cursor {
  int b, tok, n;  // sequence, first token of the tile, the sequence's end
  int col, off;   // its page (a column of the table) and place in it
};

template <int NB, bool WIDE, int WARPS>
__global__ void __launch_bounds__(WARPS * 32, 1) fa_paged_stream_kernel(const StreamArgs a) {
  using R = Row<NB>;
  constexpr int kSt = Ring<NB, WARPS>::STAGES, kThreads = WARPS * 32;
  constexpr int RH = WIDE ? 2 : 1;  // row halves in use: query heads lane / 4 (+ 8)
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ __align__(16) float s_scale[WARPS][2][NB][kUnit];  // K and V scales of the tile at hand
  auto& ss = *reinterpret_cast<SplitScan<kThreads>*>(smem);        // before the rings are in use
  // broadcasts of what is the same in a warp anyway: the row of units and the
  // copies' bases then run on uniform registers (16 x 16000 tokens 89 -> 84 us)
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  pdl_launch_dependents();
  scan_units(a.split, ss);
  const int U = ss.scan[kThreads], C = a.split.active(U);
  const int per_worker = a.Hkv * a.QG;
  // few workers: over all CTAs, as many warps in each
  const int used = (C * per_worker + gridDim.x - 1) / gridDim.x;
  const int gw = warp < used ? blockIdx.x * used + warp : C * per_worker;
  const int wk = gw / per_worker, hw = gw % per_worker, h = hw / a.QG, qg = hw % a.QG;
  // a programmatic dependent of the prefix kernel, whose results it does not
  // read: it only may not end before it (the combine waits for this grid)
  int u = 0, ue = 0;
  Cursor f{};  // the worker's first tile
  if (wk < C) {
    const Shares shares(U, C);
    u = shares.begin(wk), ue = shares.begin(wk + 1);
    if (u < ue) {
      int lo = 0, hi = kThreads;
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (ss.scan[mid] <= u) lo = mid;
        else hi = mid;
      }
      f.b = lo * run_len<kThreads>(a.split);
      int before = ss.scan[lo], here;
      while (before + (here = a.split.units(f.b)) <= u) {
        before += here;
        ++f.b;
      }
      f.n = a.split.len(f.b);
      f.tok = a.split.first() + (u - before) * kUnit;
      f.col = f.tok / a.ps, f.off = f.tok % a.ps;
    }
  }
  __syncthreads();  // the scan is read: the rings may be written
  if (u >= ue) return pdl_wait();

  uint8_t* ring = smem + warp * kSt * R::STAGE;
  const long long row_bytes = (long long)a.Hkv * R::BYTES;
  const int head_off = h * R::BYTES, row15 = (int)(row_bytes & 15);

  // The tile being consumed, in the same row of units.
  int cb = f.b, ctok = f.tok, cn = f.n;
  // Places in a stage: rows start at the 16-byte boundary below them, and 8
  // rows of a unit follow each other in a page, so the start within the first
  // 16 bytes depends on the row index mod 8 only.
  auto row_at = [&](int i) { return i * R::PITCH + (((i & 7) * row15 + head_off) & 15); };
  const int at_k = row_at(g) + 4 * c;                                  // K row g (g + 8: 8 rows on)
  const int at_v0 = kUnit * R::PITCH + row_at(2 * c) + 4 * g;          // V rows 2 c, 2 c + 1 (and + 8)
  const int at_v1 = kUnit * R::PITCH + row_at(2 * c + 1) + 4 * g;
  const int at_s = (lane >> 4) * kUnit * R::PITCH + row_at(lane & 15);  // this lane's row, for its scales
  auto advance = [&](Cursor& x) {  // to the next tile of the row (there is one)
    x.tok += kUnit;
    x.off += kUnit;
    while (x.off >= a.ps) x.off -= a.ps, ++x.col;
    if (x.tok >= x.n) {
      do {
        ++x.b;
        x.n = a.split.len(x.b);
      } while (x.n <= a.split.start);
      x.tok = a.split.first();
      x.col = x.tok / a.ps, x.off = x.tok % a.ps;
    }
  };
  // pages of the two groups of 8 tokens of tile x (-1: no such token)
  auto pages_of = [&](const Cursor& x) {
    int2 p = make_int2(-1, -1);
    const int32_t* t = a.table + (long long)x.b * a.W;
    p.x = (x.tok < a.prefix_len ? a.table : t)[x.col];
    if (x.tok + 8 < x.n) p.y = (x.tok + 8 < a.prefix_len ? a.table : t)[x.col + (x.off + 8 >= a.ps)];
    return p;
  };
  const Pieces<NB> pieces(lane, row_bytes, head_off);
  const uint32_t ring32 = smem_u32(ring);
  // issues the copies of tile x, whose pages are p; returns the rows present
  auto issue = [&](const Cursor& x, int2 p, int st) -> uint32_t {
    uint32_t mask = 0;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int page = __shfl_sync(0xffffffffu, half ? p.y : p.x, 0), tok = x.tok + 8 * half;
      if (page >= 0 && page < a.num_pages) {
        const int off = x.off + 8 * half;
        const long long at = ((long long)page * a.ps + (off >= a.ps ? off - a.ps : off)) * row_bytes;
        const uint32_t to = ring32 + st * R::STAGE + half * 8 * R::PITCH;
        pieces.copy(to, a.k + at);
        pieces.copy(to + kUnit * R::PITCH, a.v + at);
        const int lo = max(0, a.split.start - tok), hi = min(8, x.n - tok);  // tokens of the group in use
        if (hi > lo) mask |= ((1u << hi) - (1u << min(lo, 8))) << (8 * half);
      }
    }
    return mask;
  };

  int left = ue - u;         // tiles not yet consumed
  int ahead = left;          // tiles not yet issued
  int2 page = pages_of(f);
  uint32_t masks[kSt];   // rows present in the tiles in flight, oldest first
#pragma unroll
  for (int i = 0; i < kSt; ++i) masks[i] = 0;
#pragma unroll
  for (int i = 0; i < kSt - 1; ++i) {
    if (ahead > 0) {
      masks[i] = issue(f, page, i);
      if (--ahead > 0) {
        advance(f);
        page = pages_of(f);
      }
    }
    copy_commit();
  }

  int st = 0;
  while (left > 0) {
    // ---- a segment: the worker's tiles of sequence cur.b
    const int b = cb;
    uint32_t qa[2 * NB][2 * RH];
    float sl[RH];
#pragma unroll
    for (int r = 0; r < RH; ++r) {
      const int hl = qg * 16 + g + 8 * r;  // query head within the KV head's group
      const bool real = hl < a.G;
      const uint2* q = reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(a.q) +
                                                      ((long long)b * a.Hq + h * a.G + (real ? hl : 0)) * (NB * 32));
      sl[r] = a.sl;
      uint2 w[2 * NB];
#pragma unroll
      for (int i = 0; i < 2 * NB; ++i) w[i] = real ? q[4 * i + c] : make_uint2(0, 0);
      if (a.q_bf16) {
        // bf16 -> fp16 after an exact power of two per row that puts the
        // largest element near 2^14; the factor returns with the scores
        float top = 0.0f;
#pragma unroll
        for (int i = 0; i < 2 * NB; ++i) {
          top = fmaxf(top, fmaxf(fabsf(__uint_as_float(w[i].x << 16)), fabsf(__uint_as_float(w[i].x & 0xffff0000u))));
          top = fmaxf(top, fmaxf(fabsf(__uint_as_float(w[i].y << 16)), fabsf(__uint_as_float(w[i].y & 0xffff0000u))));
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const int e = min(max((int)(__float_as_uint(top) >> 23) - 127 - 14, -100), 100);
        const float down = __uint_as_float((uint32_t)(127 - e) << 23);
        sl[r] *= __uint_as_float((uint32_t)(127 + e) << 23);
#pragma unroll
        for (int i = 0; i < 2 * NB; ++i) {
          w[i].x = pack2<__half>(__uint_as_float(w[i].x << 16) * down, __uint_as_float(w[i].x & 0xffff0000u) * down);
          w[i].y = pack2<__half>(__uint_as_float(w[i].y << 16) * down, __uint_as_float(w[i].y & 0xffff0000u) * down);
        }
      }
#pragma unroll
      for (int i = 0; i < 2 * NB; ++i) {
        qa[i][r] = w[i].x;
        qa[i][RH + r] = w[i].y;
      }
    }
    float acc[NB * 2][RH][4];  // O^T: dims 32 (i / 2) + 4 g + 2 (i % 2) + {0, 1} of heads 8 r + 2 c + {0, 1}
#pragma unroll
    for (int i = 0; i < NB * 2; ++i)
#pragma unroll
      for (int r = 0; r < RH; ++r)
#pragma unroll
        for (int x = 0; x < 4; ++x) acc[i][r][x] = 0.0f;
    float m[RH], l[RH], e = kMaxExp;  // p is 2^(s - m + e)
#pragma unroll
    for (int r = 0; r < RH; ++r) m[r] = -INFINITY, l[r] = 0.0f;

    int tiles = min(left, (cn - ctok + kUnit - 1) / kUnit);
    left -= tiles;
    if (left > 0) {
      do {
        cn = a.split.len(++cb);
      } while (cn <= a.split.start);
      ctok = a.split.first();
    }
    for (; tiles > 0; --tiles) {
      // keep the ring full: the stage read in the previous step is free
      uint32_t fresh = 0;
      if (ahead > 0) {
        int s2 = st + kSt - 1;
        s2 = s2 >= kSt ? s2 - kSt : s2;
        fresh = issue(f, page, s2);
        if (--ahead > 0) {
          advance(f);
          page = pages_of(f);
        }
      }
      copy_commit();
      const uint32_t mask = masks[0];
#pragma unroll
      for (int i = 0; i + 1 < kSt; ++i) masks[i] = masks[i + 1];
      masks[kSt - 2] = fresh;
      copy_wait<kSt - 1>();
      __syncwarp();
      const uint8_t* stage = ring + st * R::STAGE;
      uint32_t top = 0;  // bits of the tile's largest |d_v|
      {
        // a row per lane: its scales in fp32. An absent row may hold anything:
        // its weight is 0, not 0 x scale
        const uint8_t* row = stage + at_s;
        const bool there = mask >> (lane & 15) & 1;
#pragma unroll
        for (int j = 0; j < NB; ++j) {
          const float d = there ? __half2float(*reinterpret_cast<const __half*>(row + j * kQ8)) : 0.0f;
          s_scale[warp][lane >> 4][j][lane & 15] = d;
          top = max(top, __float_as_uint(d) & 0x7fffffffu);
        }
        top = __reduce_max_sync(0xffffffffu, lane < 16 ? 0u : top);
      }
      // 2^e d_v < 2^15; an infinity or NaN among the scales keeps e for the others
      const float en = fminf(e, fmaxf(-1.0f, 141.0f - (float)(top >> 23)));
      __syncwarp();
      auto scales = [&](int kv, int j, int i) { return *reinterpret_cast<const float2*>(&s_scale[warp][kv][j][i]); };

      // S^T: tokens g and g + 8 of heads 8 r + 2 c + {0, 1}
      float st4[RH][4];
#pragma unroll
      for (int r = 0; r < RH; ++r)
#pragma unroll
        for (int x = 0; x < 4; ++x) st4[r][x] = 0.0f;
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        float d[RH][4];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          uint32_t k4[4];
          codes_h2(word_at<NB>(stage + at_k, j * kQ8 + 2 + 16 * half), k4[0], k4[2]);
          codes_h2(word_at<NB>(stage + at_k + 8 * R::PITCH, j * kQ8 + 2 + 16 * half), k4[1], k4[3]);
#pragma unroll
          for (int r = 0; r < RH; ++r) {
            const uint32_t* q = qa[2 * j + half];
            if (half == 0) mma16816(d[r], k4, q[r], q[RH + r], 0.0f, 0.0f, 0.0f, 0.0f);
            else mma16816(d[r], k4, q[r], q[RH + r], d[r][0], d[r][1], d[r][2], d[r][3]);
          }
        }
        const float dk0 = s_scale[warp][0][j][g], dk1 = s_scale[warp][0][j][g + 8];
#pragma unroll
        for (int r = 0; r < RH; ++r)
#pragma unroll
          for (int x = 0; x < 4; ++x) st4[r][x] = fmaf(d[r][x], x < 2 ? dk0 : dk1, st4[r][x]);
      }
      // transposed: head g (+ 8) of tokens 8 t + 2 c + {0, 1}, as P is needed
      float s[2][2 * RH];
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int r = 0; r < RH; ++r) transpose8(st4[r][2 * t], st4[r][2 * t + 1], s[t][2 * r], s[t][2 * r + 1]);
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int r = 0; r < 2 * RH; ++r) s[t][r] *= sl[r >> 1];
      if (mask != 0xffffu) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int r = 0; r < 2 * RH; ++r)
            if (!(mask >> (8 * t + 2 * c + (r & 1)) & 1u)) s[t][r] = -INFINITY;
      }
      float p[2][2 * RH], f_[RH];
      bool moved = en != e;
#pragma unroll
      for (int r = 0; r < RH; ++r) {
        float mx = m[r];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int x = 0; x < 2; ++x) mx = fmaxf(mx, s[t][2 * r + x]);
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const float base = mx == -INFINITY ? 0.0f : mx - en;
        f_[r] = ex2((m[r] - e) - base);
        moved |= mx != m[r];
        m[r] = mx;
        float sum = 0.0f;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            p[t][2 * r + x] = ex2(s[t][2 * r + x] - base);
            sum += p[t][2 * r + x];
          }
        l[r] = fmaf(l[r], f_[r], sum);
      }
      e = en;
      if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
        for (int r = 0; r < RH; ++r) {
          const float f0 = __shfl_sync(0xffffffffu, f_[r], 8 * c), f1 = __shfl_sync(0xffffffffu, f_[r], 8 * c + 4);
#pragma unroll
          for (int i = 0; i < NB * 2; ++i) acc[i][r][0] *= f0, acc[i][r][1] *= f1, acc[i][r][2] *= f0, acc[i][r][3] *= f1;
        }
      }
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          w[i] = word_at<NB>(stage + ((i & 1) ? at_v1 : at_v0) + (i >> 1) * 8 * R::PITCH, j * kQ8 + 2) ^ 0x80808080u;
        const float2 d0 = scales(1, j, 2 * c), d1 = scales(1, j, 8 + 2 * c);
        uint32_t pa[2 * RH];
#pragma unroll
        for (int r = 0; r < RH; ++r) {
          pa[r] = pack2<__half>(p[0][2 * r] * d0.x, p[0][2 * r + 1] * d0.y);
          pa[RH + r] = pack2<__half>(p[1][2 * r] * d1.x, p[1][2 * r + 1] * d1.y);
        }
        // byte i of the two tokens of a pair, for the 4 dims of the word
        const uint32_t x01 = __byte_perm(w[0], w[1], 0x5140), x23 = __byte_perm(w[0], w[1], 0x7362);
        const uint32_t y01 = __byte_perm(w[2], w[3], 0x5140), y23 = __byte_perm(w[2], w[3], 0x7362);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t x = i ? x23 : x01, y = i ? y23 : y01;
          const uint32_t v4[4] = {hsub2(__byte_perm(x, 0x64646464u, 0x4140), 0x64806480u),
                                  hsub2(__byte_perm(x, 0x64646464u, 0x4342), 0x64806480u),
                                  hsub2(__byte_perm(y, 0x64646464u, 0x4140), 0x64806480u),
                                  hsub2(__byte_perm(y, 0x64646464u, 0x4342), 0x64806480u)};
#pragma unroll
          for (int r = 0; r < RH; ++r) {
            float(&o)[4] = acc[2 * j + i][r];
            mma16816(o, v4, pa[r], pa[RH + r], o[0], o[1], o[2], o[3]);
          }
        }
      }
      __syncwarp();  // the stage may be refilled
      if (++st == kSt) st = 0;
    }
    // ---- the segment's state
    const long long seg = wk + b;
#pragma unroll
    for (int r = 0; r < RH; ++r) {
      float sum = l[r];
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      const int hl = qg * 16 + g + 8 * r;
      if (hl < a.G) {
        const long long row = seg * a.Hq + h * a.G + hl;
        if (c == 0) a.ml[row] = make_float2(m[r] - e, sum);  // the sums carry 2^e: as if m were lower
      }
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int ho = qg * 16 + 8 * r + 2 * c + x;
        if (ho < a.G) {
          float4* o = reinterpret_cast<float4*>(a.part + (seg * a.Hq + h * a.G + ho) * (NB * 32)) + g;
#pragma unroll
          for (int j = 0; j < NB; ++j)
            o[8 * j] = make_float4(acc[2 * j][r][x], acc[2 * j][r][2 + x], acc[2 * j + 1][r][x], acc[2 * j + 1][r][2 + x]);
        }
      }
    }
  }
  pdl_wait();
}

// ---- one row in fp32 on scalar instructions ----------------------------------------------
// 32 tokens per step: a lane per token for q . k, then a lane per dimension for
// p . v. For the pages and rows that the other kernels do not take.
struct Tokens {
  const uint8_t *k, *v;
  const int32_t *shared, *own;  // pages of tokens below prefix_len, and of the others
  long long num_pages, row_bytes, head_off;
  int ps, prefix_len;
};
// The softmax state (natural units) of tokens j0 .. j1 - 1 for the scaled query
// s_q; s_p and s_row hold 32 values each. A warp together. U: how far the loops
// are unrolled, 1 where the code should be short.
template <int U, int NB>
__device__ __forceinline__ void attend_tokens(const Tokens& a, int nb, int j0, int j1, const float* s_q, float* s_p,
                                              long long* s_row, float& m, float& l, float (&acc)[NB]) {
  const unsigned full = 0xffffffffu;
  const int lane = threadIdx.x & 31;
  m = -INFINITY, l = 0.0f;
#pragma unroll
  for (int t = 0; t < NB; ++t) acc[t] = 0.0f;
  for (; j0 < j1; j0 += 32) {
    const int j = j0 + lane;
    float s = -INFINITY;
    long long off = -1;
    if (j < j1) {
      const long long page = (j < a.prefix_len ? a.shared : a.own)[j / a.ps];
      if (page >= 0 && page < a.num_pages) {
        off = (page * a.ps + j % a.ps) * a.row_bytes + a.head_off;
        const uint8_t* k = a.k + off;
        s = 0.0f;
#pragma unroll 1
        for (int t = 0; t < nb; ++t) {
          const float d = half_bits_to_float(*reinterpret_cast<const uint16_t*>(k + t * kQ8));
          float dot = 0.0f;
#pragma unroll U
          for (int e = 0; e < 32; ++e) dot = fmaf(s_q[t * 32 + e], (float)(int8_t)k[t * kQ8 + 2 + e], dot);
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
    s_p[lane] = p;
    s_row[lane] = off;
    __syncwarp();
#pragma unroll
    for (int t = 0; t < NB; ++t) acc[t] *= c;
    const int n = min(32, j1 - j0);
#pragma unroll (U > 4 ? 4 : U)
    for (int jj = 0; jj < n; ++jj) {
      if (s_row[jj] < 0) continue;
      const float pj = s_p[jj];
      const uint8_t* v = a.v + s_row[jj];
#pragma unroll
      for (int t = 0; t < NB; ++t)
        if (t < nb) {
          const float d = half_bits_to_float(*reinterpret_cast<const uint16_t*>(v + t * kQ8));
          acc[t] = fmaf(pj * d, (float)(int8_t)v[t * kQ8 + 2 + lane], acc[t]);
        }
    }
    __syncwarp();
  }
}

// ---- shared prefix: one pass of the tensor cores over it for the whole batch -----------
// The B * G query heads of a KV head are the rows of 128-row tiles; a CTA
// takes two tiles and a range of 64-token blocks of the prefix, so each block
// is read and dequantised once for 256 rows. Per block and tile:
//   S = Q K^T (tcgen05, Q from TMEM), P = 2^(S sl - m + kBias) (a thread per
//   row), O += P V (tcgen05, P from TMEM)
// as in the prompt kernel (lazy maximum, two tiles alternating).
// Operands are fp16. K = d * code has up to 19 significant bits: it enters as
// an fp16 high part plus the exact remainder (two products into the same
// accumulator), so that the scores carry fp32's error only: an error of K grows
// with the score and is exponentiated (scores of 100 from a rounded K put the
// output 1 % off). V does the same for fp16 outputs (LO), where P then is the only
// rounded factor; for bf16 outputs, whose own rounding is 8 times coarser, the
// high part alone is used (with both, 256 samples behind 4096 tokens take 62.8 us instead of 61.5).
// bf16 queries become fp16 after an exact power of two per row.
// d of 512 and more (values past fp16's largest number) overflows the high part,
// and a token that a row does not see enters P V with weight 0, which an infinite
// or NaN scale turns into NaN. Where a CTA meets such a scale, its rows are done
// again in fp32, each from its own tokens, by the warps that dequantise (which
// have nothing else to do by then). Watching the scales and that code cost every
// call 0.3 (bf16) to 1 us (fp16); a look at the sums and the code in the combine
// cost 1 to 2.
//
// 8192 tokens for 64 x 32 heads over 8 (128 CTAs of 8 blocks) take 23 us, 4 of
// them the set-up to the first scores, 3 the last stores; a block takes 3900
// clocks (2700 without any low part): the chain S -> P -> P V and next S of a
// tile, of which the products are 1130 (850 without V's low part, 560 without
// either). Steps of 32 keys with the scores one step ahead took as long.
//
// Warps: 0-3 / 4-7 softmax of tile 0 / 1, 8 MMA issue and TMEM, 9-16 copy and
// dequantise 8 tokens of each block (a block of 32 values per thread), each
// from its own ring of rows; 17-19 idle (they complete the last warpgroup).
// Registers: 640 x 96 at launch, 256 x 144 + 384 x 64 after the split.
constexpr int kBlk = 64;
constexpr int kTile = 128;
constexpr int kPrefixThreads = 640;
constexpr int kMmaWarp = 8, kDeqWarp = 9, kDeqWarps = 8;
constexpr float kBias = 7.0f, kLazy = 8.0f;
constexpr float kMinScale = 1e-30f;    // of a row, its power of two included: 0 would turn a hidden key's -inf into NaN
constexpr int kRaw = 3, kOps = 2;      // blocks of raw rows and of operands in flight (K and V each)
constexpr int kMasks = 16;             // blocks whose row masks are kept (more than are in flight)

template <int NB, bool LO>  // LO: V's low part too
struct PrefixTraits {
  static constexpr int DP = NB <= 2 ? 64 : 128;
  static constexpr int PANELS = DP / 64;
  static constexpr int PANEL = kBlk * 128;
  static constexpr int PART = PANELS * PANEL;       // the high (or low) parts of a block
  static constexpr int OP_K = 2 * PART, OP = OP_K + PART * (LO ? 2 : 1);  // K of a block; K and V
  static constexpr int RAW = 2 * kBlk * Row<NB>::PITCH;  // raw rows of a block, K and V
  static constexpr int OFF_RAW = kOps * OP;
  static constexpr int OFF_STAGE = OFF_RAW + kRaw * RAW;  // 4 KB per softmax warp
  static constexpr int OFF_BAR = OFF_STAGE + 8 * 4096;
  static constexpr int OFF_BIG = OFF_BAR + 508;
  static constexpr int SMEM = OFF_BAR + 512 + 1024;
  static_assert(SMEM <= 232448, "shared memory budget");
  static_assert(OFF_RAW % 1024 == 0 && OFF_BAR % 16 == 0, "alignment");
};
constexpr uint32_t kColS = 0, kColQ = 128, kColO = 256;  // TMEM: S0 S1 (64 each) | Q0 Q1 (64 each) | O0 O1

struct PrefixArgs {
  const void* q;
  int q_bf16;
  const uint8_t *k, *v;
  long long num_pages;
  int ps, B, Hq, Hkv, G, prefix_len, limit, chunks;
  const int32_t *table, *seq_lens;  // the table's row 0
  float scale, sl;
  uint32_t flip;
  float* part;  // [chunk][B * Hq][NB * 32]
  float2* ml;
  int* err;
};

__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ uint32_t hfma2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
// fp16 operands, fp32 D, M = 128; bit 16: B is MN-major (V: dims across, tokens down).
__host__ __device__ constexpr uint32_t idesc_h(int n, bool b_mn) {
  return (1u << 4) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((128u >> 4) << 24);
}
// What a CTA of the prefix kernel works on.
struct PrefixJob {
  int chunk, h, row0, j0, n;  // chunk, KV head, first of its rows, its first block and blocks
  __device__ __forceinline__ PrefixJob(const PrefixArgs& a, int cta) {
    const int hp = cta / a.chunks, blocks = (a.prefix_len + kBlk - 1) / kBlk;
    chunk = cta % a.chunks, h = hp % a.Hkv, row0 = hp / a.Hkv * 2 * kTile;
    j0 = (int)((long long)blocks * chunk / a.chunks), n = (int)((long long)blocks * (chunk + 1) / a.chunks) - j0;
  }
};
// Where the CTA met a scale past the operands' range: each dequantising warp does
// 32 of its rows once more in fp32. Everything is derived anew, so that nothing of
// it is kept in registers before.
template <int NB, bool LO>
__device__ __forceinline__ void redo_rows(const PrefixArgs& a, uint8_t* smem) {
  using R = PrefixTraits<NB, LO>;
  int cta = blockIdx.x, tid = threadIdx.x;
  asm volatile("" : "+r"(cta), "+r"(tid), "+l"(smem));
  smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem) + 1023) & ~(uintptr_t)1023);
  if (!*reinterpret_cast<const uint32_t*>(smem + R::OFF_BIG)) return;
  const int lane = tid & 31, dw = (tid >> 5) - kDeqWarp;
  float* scratch = reinterpret_cast<float*>(smem + R::OFF_RAW + dw * kRaw * 16 * Row<NB>::PITCH);
  const PrefixJob job(a, cta);
#pragma unroll 1
  for (int row = job.row0 + dw * 32, end = min(row + 32, a.B * a.G); row < end; ++row) {
    const int b = row / a.G, qrow = b * a.Hq + job.h * a.G + row % a.G;
    const int keys = max(0, min(min(a.seq_lens[b], a.limit), a.prefix_len));
    const Tokens tokens{a.k, a.v, a.table, a.table, a.num_pages, (long long)a.Hkv * Row<NB>::BYTES, job.h * Row<NB>::BYTES,
                        a.ps, a.prefix_len};
    __syncwarp();
    for (int x = lane; x < NB * 32; x += 32) {
      const uint16_t v = static_cast<const uint16_t*>(a.q)[(long long)qrow * (NB * 32) + x];
      scratch[x] = (a.q_bf16 ? __uint_as_float((uint32_t)v << 16) : half_bits_to_float(v)) * a.scale;
    }
    __syncwarp();
    float m, l, acc[NB];
    attend_tokens<1>(tokens, NB, job.j0 * kBlk, min(keys, (job.j0 + job.n) * kBlk), scratch, scratch + NB * 32 + 64,
                  reinterpret_cast<long long*>(scratch + NB * 32), m, l, acc);
    const long long at = (long long)job.chunk * a.B * a.Hq + qrow;
#pragma unroll
    for (int x = 0; x < NB; ++x) a.part[at * (NB * 32) + 32 * x + lane] = acc[x];
    if (lane == 0) a.ml[at] = make_float2(m * 1.44269504088896340736f, l);
  }
}

template <int NB, bool LO>
__global__ void __launch_bounds__(kPrefixThreads, 1) fa_paged_prefix_kernel(const PrefixArgs a) {
  using R = PrefixTraits<NB, LO>;
  constexpr int DP = R::DP;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint64_t* op_full = reinterpret_cast<uint64_t*>(smem + R::OFF_BAR);  // K at 2 (j % kOps), V behind it
  uint64_t* op_empty = op_full + 2 * kOps;
  uint64_t* s_full = op_empty + 2 * kOps;  // S of a tile is there (and its earlier P V is done)
  uint64_t* p_full = s_full + 2;       // P of a tile is there, its S is read
  uint64_t* o_full = p_full + 2;       // the tile's last P V is done
  uint64_t* q_full = o_full + 2;       // the tiles' queries are in TMEM
  uint64_t* drained = q_full + 1;      // all of the MMA warp's products and arrivals are done
  uint64_t* row_mask = drained + 1;    // rows present in block j, at j % kMasks
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(row_mask + kMasks);
  uint32_t* big = reinterpret_cast<uint32_t*>(smem + R::OFF_BIG);  // a scale past the operands' range was met
  static_assert((4 * kOps + 8 + kMasks) * 8 + 4 <= 508, "barrier area");
  static_assert(kDeqWarps == 8 && kRaw * 16 * Row<NB>::PITCH >= NB * 128 + 128 + 256, "a warp's ring holds a row's scratch");
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_launch_dependents();

  const PrefixJob job(a, blockIdx.x);
  const int chunk = job.chunk, h = job.h, row0 = job.row0, j0 = job.j0, n = job.n;
  const int rows = a.B * a.G;
  const bool two = row0 + kTile < rows;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2 * kOps; ++i) {
      mbar_init(&op_full[i], kDeqWarps);
      mbar_init(&op_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
      mbar_init(&o_full[i], 1);
    }
    mbar_init(q_full, two ? 8 : 4);
    mbar_init(drained, 1);
    *big = 0;
    fence_mbar_init();
  }
  // The set-up's barrier, which every role meets with its first loads out.
  auto set_up = [&]() {
    tc::tc_fence_before();
    named_bar_sync(0, kPrefixThreads);
    tc::tc_fence_after();
  };
  bool dead = false;

  if (warp >= 2 * 4) asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
  if (warp >= kDeqWarp + kDeqWarps) {
    set_up();
  } else if (warp >= kDeqWarp) {
    // ---- one block of 32 values per thread: token 8 w + lane % 8, block lane / 8.
    // 8 tokens of a block lie in one page (pages hold a multiple of 8): page
    // `col` of the table, from row `off0` on.
    const long long row_bytes = (long long)a.Hkv * Row<NB>::BYTES;
    const int head_off = h * Row<NB>::BYTES, row15 = (int)(row_bytes & 15);
    const int dw = warp - kDeqWarp;
    uint8_t* ring = smem + R::OFF_RAW + dw * kRaw * 16 * Row<NB>::PITCH;  // per block: 8 K rows, 8 V rows
    const Pieces<NB> pieces(lane, row_bytes, head_off);
    const int last_col = (a.prefix_len - 1) / a.ps;
    int col = (j0 * kBlk + dw * 8) / a.ps, off0 = (j0 * kBlk + dw * 8) % a.ps;
    int page = a.table[min(col, last_col)];
    set_up();
    // copies of block j, one group; the next page id is loaded, not looked at
    auto issue = [&](int j) -> uint32_t {
      const int left = a.prefix_len - ((j0 + j) * kBlk + dw * 8);
      uint32_t present = 0;
      if (page >= 0 && page < a.num_pages && j < n && left > 0) {
        present = left >= 8 ? 0xffu : (1u << left) - 1u;
        const long long at = ((long long)page * a.ps + off0) * row_bytes;
        const uint32_t to = smem_u32(ring) + (j % kRaw) * 16 * Row<NB>::PITCH;
        pieces.copy(to, a.k + at);
        pieces.copy(to + 8 * Row<NB>::PITCH, a.v + at);
      }
      copy_commit();
      for (off0 += kBlk; off0 >= a.ps; off0 -= a.ps) ++col;
      page = a.table[min(col, last_col)];
      return present;
    };
    uint32_t rows_at[kRaw];  // rows of the blocks in flight, oldest first
#pragma unroll
    for (int i = 0; i < kRaw; ++i) rows_at[i] = 0;
#pragma unroll
    for (int i = 0; i < kRaw - 1; ++i) rows_at[i] = issue(i);
    const int tok = dw * 8 + (lane & 7), blk = lane >> 3;
    const int off = (((lane & 7) * row15 + head_off) & 15) + blk * kQ8;
    const uint32_t sh = (uint32_t)(off & 2) * 8;
    const bool used = blk * 32 < DP, real = blk < NB;
    uint8_t* dst = smem + (blk >> 1) * R::PANEL;
    // The 9 words that cover this thread's block of 34 bytes; 0 for an absent
    // row, since whatever its slot holds must not meet P = 0.
    auto words = [&](const uint8_t* row, bool present, uint32_t (&w)[9]) {
      const uint32_t* src = reinterpret_cast<const uint32_t*>(row + (off & ~3));
#pragma unroll
      for (int x = 0; x < 8; ++x) w[x] = present ? src[x] : 0u;
      w[8] = !present ? 0u : sh ? src[8] : *reinterpret_cast<const uint16_t*>(src + 8);
    };
    auto convert = [&](const uint32_t (&w)[9], uint8_t* op, bool low) {
      const uint32_t d = (w[0] >> sh) & 0xffffu, d2 = d | d << 16;
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          uint32_t c[2];
          codes_h2(__funnelshift_rc(w[2 * x + y], w[2 * x + y + 1], sh + 16), c[0], c[1]);
#pragma unroll
          for (int z = 0; z < 2; ++z) {
            hi[2 * y + z] = hmul2(c[z], d2);
            if (low) lo[2 * y + z] = hfma2(c[z], d2, hi[2 * y + z] ^ 0x80008000u);
          }
        }
        uint8_t* o = op + tc::sw128_off(tok, (blk & 1) * 4 + x);
        *reinterpret_cast<uint4*>(o) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        if (low) *reinterpret_cast<uint4*>(o + R::PART) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
      }
    };
    uint32_t top = 0;  // bit 14 or 30: |d| of 512 or more (both high exponent bits), infinite or NaN
    for (int j = 0; j < n; ++j) {
      const int os = j % kOps;
      rows_at[kRaw - 1] = issue(j + kRaw - 1);
      if (lane == 0) reinterpret_cast<uint8_t*>(&row_mask[j % kMasks])[dw] = (uint8_t)rows_at[0];
      copy_wait<kRaw - 1>();
      __syncwarp();
      const bool present = real && (rows_at[0] >> (lane & 7) & 1);
      const uint8_t* row = ring + ((j % kRaw) * 16 + (lane & 7)) * Row<NB>::PITCH;
      uint32_t wk[9], wv[9];
      words(row, present, wk);
      words(row + 8 * Row<NB>::PITCH, present, wv);
      const uint32_t d = __byte_perm(wk[0] >> sh, wv[0] >> sh, 0x5410);  // the scales of K and V
      top |= d & (d << 1);
      // K is free again once its scores are there, V a block later
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        if (j >= kOps) mbar_wait_or_poison(&op_empty[2 * os + kv], ((j / kOps) - 1) & 1, a.err, DEV_TIMEOUT_EMPTY, dead);
        if (used) convert(kv ? wv : wk, dst + os * R::OP + kv * R::OP_K, LO || kv == 0);
        fence_proxy_async_smem();
        __syncwarp();  // also: the ring's rows are read
        if (lane == 0) mbar_arrive(&op_full[2 * os + kv]);
      }
#pragma unroll
      for (int x = 0; x + 1 < kRaw; ++x) rows_at[x] = rows_at[x + 1];
    }
    if (top & 0x40004000u) *big = 1;
    named_bar_sync(1, (8 + kDeqWarps) * 32);  // also: the softmax warps have stored their rows
    redo_rows<NB, LO>(a, smem_raw);
  } else if (warp == kMmaWarp) {
    constexpr uint32_t idesc_s = idesc_h(kBlk, false), idesc_o = idesc_h(DP, true);
    tc::tmem_alloc(tmem_slot, 512);
    set_up();
    const uint32_t tmem = *tmem_slot, base = smem_u32(smem), go = tc::elect_one();
    const int tiles = two ? 2 : 1;
    auto score = [&](int t, int j) {
      mbar_wait_or_poison(&op_full[2 * (j % kOps)], (j / kOps) & 1, a.err, DEV_TIMEOUT_FULL, dead);
      tc::tc_fence_after();
      const uint64_t kd = tc::sw128_desc(base + j % kOps * R::OP);
#pragma unroll
      for (int part = 0; part < 2; ++part)
#pragma unroll
        for (int k = 0; k < DP / 16; ++k)
          tc::mma_ts_go(tmem + kColS + t * kBlk, tmem + kColQ + t * 64 + 8 * k,
                        kd + (uint64_t)(part * (R::PART >> 4) + (k >> 2) * (R::PANEL >> 4) + (k & 3) * 2), idesc_s,
                        (part > 0 || k > 0) ? 1u : 0u, go);
      tc::mma_commit_go(&s_full[t], go);
    };
    // every arrival is waited for before the CTA ends: an operand is only
    // released to one that waits for it, and the warp drains at the end
    auto release = [&](int j, int kv) {
      if (j + kOps < n) tc::mma_commit_go(&op_empty[2 * (j % kOps) + kv], go);
    };
    mbar_wait_or_poison(q_full, 0, a.err, DEV_TIMEOUT_FULL, dead);
    tc::tc_fence_after();
    if (n > 0) {
      for (int t = 0; t < tiles; ++t) score(t, 0);
      release(0, 0);
    }
    for (int j = 0; j < n; ++j) {
      const uint64_t vd = tc::sw128_desc_mn(base + j % kOps * R::OP + R::OP_K, R::PANEL);  // dims across, tokens down
#pragma unroll 1
      for (int t = 0; t < tiles; ++t) {
        mbar_wait_or_poison(&op_full[2 * (j % kOps) + 1], (j / kOps) & 1, a.err, DEV_TIMEOUT_FULL, dead);
        mbar_wait_or_poison(&p_full[t], j & 1, a.err, DEV_TIMEOUT_FULL, dead);
        tc::tc_fence_after();
#pragma unroll
        for (int part = 0; part < (LO ? 2 : 1); ++part)
#pragma unroll
          for (int k = 0; k < kBlk / 16; ++k)
            tc::mma_ts_go(tmem + kColO + t * DP, tmem + kColS + t * kBlk + 8 * k,
                          vd + (uint64_t)(part * (R::PART >> 4) + k * (2048 >> 4)), idesc_o,
                          (j > 0 || part > 0 || k > 0) ? 1u : 0u, go);
        if (j + 1 == n) tc::mma_commit_go(&o_full[t], go);
        if (t + 1 == tiles) release(j, 1);
        if (j + 1 < n) score(t, j + 1);
      }
      if (j + 1 < n) release(j + 1, 0);
    }
    tc::mma_commit_go(drained, go);
    mbar_wait_idle_or_poison(drained, 0, a.err, DEV_TIMEOUT_FULL, dead);
    __syncwarp();
  } else {
    // ---- softmax, a thread per row
    asm volatile("setmaxnreg.inc.sync.aligned.u32 144;");
    const int t = warp >> 2;
    const int my_row = row0 + threadIdx.x;
    const int qrow = my_row < rows ? my_row / a.G * a.Hq + h * a.G + my_row % a.G : -1;
    const int my_len = a.seq_lens[qrow >= 0 ? my_row / a.G : 0];
    // the queries: pieces of 64 bytes of the rows lane / 4 + 8 x, 32 dims per j,
    // all in flight (a row without a query reads the first one)
    uint4 qv[NB][4];
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int r = max(0, __shfl_sync(0xffffffffu, qrow, 8 * x + (lane >> 2)));
#pragma unroll
      for (int j = 0; j < NB; ++j)
        qv[j][x] = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(a.q) + (long long)r * (NB * 32) + 32 * j)[lane & 3];
    }
    set_up();
    const uint32_t tmem = *tmem_slot;
    if (t == 0 || two) {
      const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
      const uint32_t s_addr = tmem + lanes + kColS + t * kBlk, o_addr = tmem + lanes + kColO + t * DP;
      uint8_t* stage = smem + R::OFF_STAGE + warp * 4096;
      const int keys = qrow >= 0 ? max(0, min(min(my_len, a.limit), a.prefix_len)) : 0;
      float sl = a.sl;
      {
        // the row's queries to TMEM (two fp16 per column), dims past D and rows
        // without a query zero, through the stage to the row's thread
        uint32_t w[DP / 2];
#pragma unroll
        for (int j = 0; j < DP / 32; ++j) {
          if (j < NB) {
            __syncwarp();
#pragma unroll
            for (int x = 0; x < 4; ++x) *stage_piece(stage, lane, x) = qv[j < NB ? j : 0][x];
            __syncwarp();
          }
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const uint4 y = j < NB && qrow >= 0 ? *stage_row(stage, lane, x) : make_uint4(0, 0, 0, 0);
            w[16 * j + 4 * x] = y.x, w[16 * j + 4 * x + 1] = y.y, w[16 * j + 4 * x + 2] = y.z, w[16 * j + 4 * x + 3] = y.w;
          }
        }
        if (a.q_bf16) {
          float top = 0.0f;
#pragma unroll
          for (int i = 0; i < DP / 2; ++i)
            top = max3(top, fabsf(__uint_as_float(w[i] << 16)), fabsf(__uint_as_float(w[i] & 0xffff0000u)));
          const int e = min(max((int)(__float_as_uint(top) >> 23) - 127 - 14, -100), 100);
          const float down = __uint_as_float((uint32_t)(127 - e) << 23);
          sl = fmaxf(sl * __uint_as_float((uint32_t)(127 + e) << 23), kMinScale);
#pragma unroll
          for (int i = 0; i < DP / 2; ++i)
            w[i] = pack2<__half>(__uint_as_float(w[i] << 16) * down, __uint_as_float(w[i] & 0xffff0000u) * down);
        }
        __syncwarp();
#pragma unroll
        for (int p = 0; p < R::PANELS; ++p) tc::tmem_st32(tmem + lanes + kColQ + t * 64 + p * 32, w + 32 * p);
        tc::tmem_st_wait();
        tc::tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(q_full);
      }
      float m = -INFINITY;
      F2 l2 = f2(0.0f, 0.0f);
      for (int j = 0; j < n; ++j) {
        mbar_wait_or_poison(&s_full[t], j & 1, a.err, DEV_TIMEOUT_FULL, dead);
        __syncwarp();
        tc::tc_fence_after();
        uint32_t s[kBlk];
        tc::tmem_ld32(s_addr, reinterpret_cast<uint32_t(&)[32]>(s[0]));
        tc::tmem_ld32(s_addr + 32, reinterpret_cast<uint32_t(&)[32]>(s[32]));
        tc::tmem_ld_wait();
        if (a.flip) {
#pragma unroll
          for (int i = 0; i < kBlk; ++i) s[i] ^= a.flip;
        }
        const int lim = keys - (j0 + j) * kBlk;
        const uint64_t present = row_mask[j % kMasks];
        if (__any_sync(0xffffffffu, lim < kBlk) || ~present) {
#pragma unroll
          for (int i = 0; i < kBlk; ++i)
            if (i >= lim || !(present >> i & 1)) s[i] = 0xff800000u;
        }
        const float mn = row_max(s) * sl;
        float f = 1.0f;
        if (mn > m + kLazy) {  // also the row's first keys (m = -inf)
          f = ex2(m - mn);
          m = mn;
          l2 = mul2(l2, f2(f, f));
        }
        if (j > 0 && __any_sync(0xffffffffu, f != 1.0f)) rescale_row(o_addr, DP, f);
        const float off = m == -INFINITY ? 0.0f : kBias - m;
        const F2 sl2 = f2(sl, sl), off2 = f2(off, off);
        F2 sum = f2(0.0f, 0.0f);
        uint32_t p[kBlk / 2];
#pragma unroll
        for (int i = 0; i < kBlk / 2; ++i) {
          const F2 e = fma2(f2(__uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1])), sl2, off2);
          float e0, e1;
          unpack(e, e0, e1);
          e0 = ex2(e0), e1 = ex2(e1);
          sum = add2(sum, f2(e0, e1));
          p[i] = pack2<__half>(e0, e1);
        }
        l2 = add2(l2, sum);
        __syncwarp();
        tc::tmem_st32(s_addr, p);
        tc::tmem_st_wait();
        tc::tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[t]);
      }
      float l, l1;
      unpack(l2, l, l1);
      l += l1;
      if (n > 0) mbar_wait_or_poison(&o_full[t], 0, a.err, DEV_TIMEOUT_FULL, dead);
      __syncwarp();
      tc::tc_fence_after();
      const long long base = (long long)chunk * a.B * a.Hq;
      if (qrow >= 0) a.ml[base + qrow] = make_float2(m - kBias, l);
      const bool none = l == 0.0f;
      float* out[8];  // of the pieces this lane stores, rows lane / 8 + 4 x
#pragma unroll
      for (int x = 0; x < 8; ++x) {
        const int r = __shfl_sync(0xffffffffu, qrow, 4 * x + (lane >> 3));
        out[x] = r >= 0 ? a.part + (base + r) * (NB * 32) + 4 * (lane & 7) : nullptr;
      }
#pragma unroll
      for (int x0 = 0; x0 < NB * 32; x0 += 32) {
        uint32_t o[32];
        tc::tmem_ld32(o_addr + x0, o);
        tc::tmem_ld_wait();
        __syncwarp();
#pragma unroll
        for (int x = 0; x < 8; ++x)
          *stage128_row(stage, lane, x) = none ? make_uint4(0, 0, 0, 0) : make_uint4(o[4 * x], o[4 * x + 1], o[4 * x + 2], o[4 * x + 3]);
        __syncwarp();
        uint4 v[8];
#pragma unroll
        for (int x = 0; x < 8; ++x) v[x] = *stage128_piece(stage, lane, x);
#pragma unroll
        for (int x = 0; x < 8; ++x)
          if (out[x]) *reinterpret_cast<uint4*>(out[x] + x0) = v[x];
      }
    }
    named_bar_arrive(1, (8 + kDeqWarps) * 32);
  }
  tc::tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) tc::tmem_dealloc(*tmem_slot, 512);
}

// ---- combine -------------------------------------------------------------------------
// out = sum_i 2^(m_i - M) O_i / sum_i 2^(m_i - M) l_i over a row's states (the
// prefix chunks, then its segments), M the largest m_i. WR warps share a row:
// warp w takes states w, w + WR, ..., kAtOnce loads in flight, and the first
// one adds the others' sums from shared memory in their order. The grid is at
// most what is resident at once, so that the scan of the lengths is paid once.
// Bound by the states' bytes and the launch: 64 x 32 rows of 128 with 16 prefix
// chunks (17 MB) and their segments take 12 us from cold caches, 10 by themselves.
struct CombineArgs {
  Split split;
  const float* part;
  const float2* ml;
  const float* ppart;  // the prefix chunks' states, [chunk][B * Hq]
  const float2* pml;
  int chunks;
  int Hq, D;
  void* out;
};
constexpr int kAtOnce = 8;  // (float4 per lane)
constexpr int kCta = 256;
constexpr int kCombineCtas = 4;  // per SM

template <typename T, int WR, int VEC>
__global__ void __launch_bounds__(kCta, kCombineCtas) fa_paged_combine_kernel(const CombineArgs a) {
  __shared__ SplitScan<kCta> ss;
  __shared__ float4 s_o[WR > 1 ? kCta / 32 : 1][VEC * 32];
  __shared__ float2 s_ml[kCta / 32];
  scan_units(a.split, ss);
  pdl_wait();
  constexpr int ROWS = kCta / 32 / WR, AT = kAtOnce / VEC;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, w = warp % WR;
  const int brows = a.split.B * a.Hq;
  const int U = ss.scan[kCta];
  const Shares shares(U, a.split.active(U));
  for (int row = blockIdx.x * ROWS + warp / WR; row < brows; row += gridDim.x * ROWS) {
    float4 o[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i) o[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float M = -INFINITY, L = 0.0f;
    const int b = row / a.Hq, h = row - b * a.Hq;
    const int u0 = units_before(a.split, ss, b), u1 = u0 + a.split.units(b);
    const int c0 = u1 > u0 ? shares.worker(u0) : 0, n = u1 > u0 ? shares.worker(u1 - 1) - c0 + 1 : 0;
    const int total = a.chunks + n;
    auto index = [&](int i) {
      return i < a.chunks ? (long long)i * brows + row : ((long long)c0 + b + i - a.chunks) * a.Hq + h;
    };
    for (int i0 = w; i0 < total; i0 += 32 * WR) {
      float2 s = make_float2(-INFINITY, 0.0f);
      const int mine = i0 + lane * WR;
      if (mine < total) s = (mine < a.chunks ? a.pml : a.ml)[index(mine)];
      const int cnt = min(32, (total - i0 + WR - 1) / WR);
      float f = 1.0f, wgt = 0.0f;
#pragma unroll 1
      for (int k0 = 0; k0 < cnt; k0 += AT) {
        float4 v[VEC][AT];
#pragma unroll
        for (int k = 0; k < AT; ++k) {
          const int x = i0 + min(k0 + k, cnt - 1) * WR;  // the last one again past the end, with weight 0
          const float4* p = reinterpret_cast<const float4*>((x < a.chunks ? a.ppart : a.part) + index(x) * a.D);
#pragma unroll
          for (int i = 0; i < VEC; ++i) v[i][k] = p[min(i * 32 + lane, a.D / 4 - 1)];
        }
        if (k0 == 0) {  // under the loads
          const float Mn = fmaxf(M, warp_max(s.x));
          const float base = Mn == -INFINITY ? 0.0f : Mn;
          f = ex2(M - base), wgt = ex2(s.x - base);
          float t = wgt * s.y;
#pragma unroll
          for (int x = 16; x >= 1; x >>= 1) t += __shfl_xor_sync(0xffffffffu, t, x);
          L = L * f + t;
          M = Mn;
#pragma unroll
          for (int i = 0; i < VEC; ++i) o[i].x *= f, o[i].y *= f, o[i].z *= f, o[i].w *= f;
        }
#pragma unroll
        for (int k = 0; k < AT; ++k) {
          const float wk = __shfl_sync(0xffffffffu, wgt, (k0 + k) & 31);
          if (k0 + k < cnt) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
              o[i].x = fmaf(wk, v[i][k].x, o[i].x), o[i].y = fmaf(wk, v[i][k].y, o[i].y);
              o[i].z = fmaf(wk, v[i][k].z, o[i].z), o[i].w = fmaf(wk, v[i][k].w, o[i].w);
            }
          }
        }
      }
    }
    if (WR > 1) {
      named_bar_sync(1 + warp / WR, WR * 32);  // the last row's sums are read
      if (w > 0) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) s_o[WR > 1 ? warp : 0][i * 32 + lane] = o[i];
        if (lane == 0) s_ml[warp] = make_float2(M, L);
      }
      named_bar_sync(1 + warp / WR, WR * 32);
      if (w > 0) continue;
      float top = M;
#pragma unroll
      for (int k = 1; k < WR; ++k) top = fmaxf(top, s_ml[warp + k].x);
      const float base = top == -INFINITY ? 0.0f : top, f = ex2(M - base);
      L *= f;
#pragma unroll
      for (int i = 0; i < VEC; ++i) o[i].x *= f, o[i].y *= f, o[i].z *= f, o[i].w *= f;
#pragma unroll
      for (int k = 1; k < WR; ++k) {
        const float2 s = s_ml[warp + k];
        const float fk = ex2(s.x - base);
        L = fmaf(fk, s.y, L);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          const float4 v = s_o[WR > 1 ? warp + k : 0][i * 32 + lane];
          o[i].x = fmaf(fk, v.x, o[i].x), o[i].y = fmaf(fk, v.y, o[i].y);
          o[i].z = fmaf(fk, v.z, o[i].z), o[i].w = fmaf(fk, v.w, o[i].w);
        }
      }
    }
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
    T* out = static_cast<T*>(a.out) + (long long)row * a.D;
#pragma unroll
    for (int i = 0; i < VEC; ++i)
      if (i * 128 + lane * 4 < a.D)
        *reinterpret_cast<uint2*>(out + i * 128 + lane * 4) =
            make_uint2(pack2<T>(o[i].x * inv, o[i].y * inv), pack2<T>(o[i].z * inv, o[i].w * inv));
  }
}

// ---- pages of other sizes than a multiple of 8 tokens, or a prefix that ends within 8
// tokens where the prefix kernel does not run (D > 128) ------------------------------------
// One warp per (sequence, query head).
constexpr int kWarps = 4;

template <typename T>
__global__ void __launch_bounds__(kWarps * 32) fa_paged_simple_kernel(const FaPagedArgs a) {
  __shared__ float s_q[kWarps][kMaxNB * 32];
  __shared__ float s_p[kWarps][32];
  __shared__ long long s_row[kWarps][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long item = (long long)blockIdx.x * kWarps + warp;
  if (item >= (long long)a.B * a.Hq) return;
  const int b = (int)(item / a.Hq), h = (int)(item % a.Hq), kh = h / (a.Hq / a.Hkv), nb = a.D / 32;
  const int len = (int)min((long long)max(0, min(a.seq_lens[b], a.max_seqlen)), (long long)a.W * a.ps);
  const T* q = static_cast<const T*>(a.q) + item * a.D;
  for (int d = lane; d < a.D; d += 32) s_q[warp][d] = to_f(q[d]) * a.scale;
  __syncwarp();
  const Tokens tokens{a.k, a.v, a.table, a.table + (long long)b * a.W, a.num_pages, (long long)a.Hkv * nb * kQ8,
                      (long long)kh * nb * kQ8, a.ps, a.prefix_len};
  float m, l, acc[kMaxNB];
  attend_tokens<32>(tokens, nb, 0, len, s_q[warp], s_p[warp], s_row[warp], m, l, acc);
  T* out = static_cast<T*>(a.out) + item * a.D;
  const float inv = l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l);  // NaN stays NaN
#pragma unroll
  for (int t = 0; t < kMaxNB; ++t)
    if (t < nb) store_f(out + t * 32 + lane, acc[t] * inv);
}

// Workers per KV head (and group of 16 of its query heads): one CTA's warps per SM in all.
int workers_of(const FaPagedArgs& a, int warps) {
  const int qg = (a.Hq / a.Hkv + 15) / 16;
  return std::max(1, sm_count() * warps / (a.Hkv * qg));
}
// The prefix kernel's pass, for head dimensions up to 128: a third launch that
// costs 5 to 10 us, against the tokens that streaming would read once per
// sequence. Where those are few they are streamed (us with and without it, 8
// KV heads of 128, 300 tokens behind the prefix: 8 sequences behind 1024 18.5
// and 17.1, behind 4096 24.0 and 32.8; 32 behind 256 19.3 and 17.2, behind 1024
// 23.3 and 34.9; heads of 64: 32 behind 256 20.7 and 18.7, behind 1024 20.7 and
// 25.0; 32 KV heads: 8 behind 1024 29.1 and 33.6; one KV head: 32 behind 1024 18.6
// and 15.1, behind 4096, where the rule is 2 us off, 24.8 and 22.4). Streaming
// needs a prefix of whole groups of 8.
constexpr int kPrefixUnits = 40;  // units of repeated reading per SM that it pays from
bool use_prefix(const FaPagedArgs& a) {
  if (a.prefix_len <= 0 || a.D > 128 || a.B <= 1) return false;
  const long long again = (long long)(a.B - 1) * a.prefix_len * a.Hkv;
  return a.prefix_len % 8 || again >= (long long)kPrefixUnits * kUnit * sm_count();
}
// Token chunks of the prefix, so that the grid fills the SMs once, and no more
// of them than the longest one needs (128 blocks over 8 KV heads: 16 chunks of 8
// instead of 18 of 7 or 8, which are two more states per row to merge).
int prefix_groups(const FaPagedArgs& a) {  // (KV head, pair of row tiles)
  const long long rows = (long long)a.B * (a.Hq / a.Hkv);
  return (int)((rows + 2 * kTile - 1) / (2 * kTile)) * a.Hkv;
}
int prefix_chunks(const FaPagedArgs& a) {
  if (!use_prefix(a)) return 0;
  const int blocks = (a.prefix_len + kBlk - 1) / kBlk;
  const int most = std::max(1, std::min(blocks, sm_count() / prefix_groups(a))), longest = (blocks + most - 1) / most;
  return (blocks + longest - 1) / longest;
}
struct Workspace {
  size_t part, ml, ppart, pml, total;  // offsets
};
Workspace workspace_of(const FaPagedArgs& a) {
  const size_t rows = ((size_t)workers_of(a, kStreamWarps) + a.B) * a.Hq, prows = (size_t)prefix_chunks(a) * a.B * a.Hq;
  Workspace w;
  w.part = 0;
  w.ppart = rows * a.D * sizeof(float);
  w.ml = w.ppart + prows * a.D * sizeof(float);
  w.pml = w.ml + rows * sizeof(float2);
  w.total = w.pml + prows * sizeof(float2);
  return w;
}

template <int NB, bool LO>
kq_status_t launch_prefix(const PrefixArgs& a, int grid, cudaStream_t s) {
  auto kernel = fa_paged_prefix_kernel<NB, LO>;
  constexpr int smem = PrefixTraits<NB, LO>::SMEM;
  if (kq_status_t st = ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), smem, "fa_paged_prefix")) return st;
  kernel<<<grid, kPrefixThreads, smem, s>>>(a);
  return check_launch("fa_paged_prefix");
}
template <int NB>
kq_status_t launch_prefix_nb(const PrefixArgs& a, int grid, cudaStream_t s) {
  return a.q_bf16 ? launch_prefix<NB, false>(a, grid, s) : launch_prefix<NB, true>(a, grid, s);
}

// Launches `kernel` as a programmatic dependent of the previous kernel on s
// (plainly where !pdl).
template <typename... Params, typename Arg>
kq_status_t launch_after(void (*kernel)(Params...), int grid, int threads, int smem, bool pdl, cudaStream_t s, const Arg& arg,
                         const char* what) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = pdl ? 1 : 0;
  return check_cuda(cudaLaunchKernelEx(&cfg, kernel, arg), what);
}

template <int NB, bool WIDE, int WARPS>
kq_status_t launch_stream(const StreamArgs& a, bool pdl, cudaStream_t s) {
  auto kernel = fa_paged_stream_kernel<NB, WIDE, WARPS>;
  constexpr int smem = Ring<NB, WARPS>::SMEM;
  if (kq_status_t st = ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), smem, "fa_paged")) return st;
  const int grid = (a.split.workers * a.Hkv * a.QG + WARPS - 1) / WARPS;
  return launch_after(kernel, grid, WARPS * 32, smem, pdl, s, a, "fa_paged_stream");
}
template <int NB>
kq_status_t launch_stream_nb(const StreamArgs& a, bool pdl, cudaStream_t s) {
  if (a.warps == kFewWarps)
    return a.G > 8 ? launch_stream<NB, true, kFewWarps>(a, pdl, s) : launch_stream<NB, false, kFewWarps>(a, pdl, s);
  return a.G > 8 ? launch_stream<NB, true, kStreamWarps>(a, pdl, s) : launch_stream<NB, false, kStreamWarps>(a, pdl, s);
}

// As many warps per row as still take all rows at once, else one (us of whole
// calls: 32 rows of 62 states 10.3 with eight, 18.5 with one; 2048 rows of 26
// states 59.6 with eight, 52.7 with four, 51.4 with two, 53.8 with one; 7168
// rows of 8 states 62.2 with two, 57.8 with one).
template <typename T, int VEC, int WR>
kq_status_t launch_combine_wr(const CombineArgs& a, long long rows, long long most, cudaStream_t s) {
  constexpr int per = kCta / 32 / WR;
  return launch_after(fa_paged_combine_kernel<T, WR, VEC>, (int)std::min(most, (rows + per - 1) / per), kCta, 0, true, s, a,
                      "fa_paged_combine");
}
template <typename T, int VEC>
kq_status_t launch_combine(const CombineArgs& a, cudaStream_t s) {
  const long long rows = (long long)a.split.B * a.Hq, most = (long long)sm_count() * kCombineCtas;
  if (rows <= most) return launch_combine_wr<T, VEC, 8>(a, rows, most, s);
  if (rows <= 2 * most) return launch_combine_wr<T, VEC, 4>(a, rows, most, s);
  if (rows <= 4 * most) return launch_combine_wr<T, VEC, 2>(a, rows, most, s);
  return launch_combine_wr<T, VEC, 1>(a, rows, most, s);
}
template <typename T>
kq_status_t launch_combine_d(const CombineArgs& a, cudaStream_t s) {
  return a.D <= 128 ? launch_combine<T, 1>(a, s) : launch_combine<T, 2>(a, s);
}

}  // namespace

size_t fa_paged_workspace(const FaPagedArgs& a) { return workspace_of(a).total; }

kq_status_t launch_fa_paged(const FaPagedArgs& a, int dtype, cudaStream_t s) {
  const int chunks = prefix_chunks(a);
  // streamed through row 0's table: B > 1 without the prefix kernel
  const int through0 = chunks == 0 && a.B > 1 ? a.prefix_len : 0;
  if (a.ps % 8 || through0 % 8) {
    const long long items = (long long)a.B * a.Hq;
    const unsigned grid = (unsigned)((items + kWarps - 1) / kWarps);
    if (dtype == KQ_F16) fa_paged_simple_kernel<__half><<<grid, kWarps * 32, 0, s>>>(a);
    else fa_paged_simple_kernel<__nv_bfloat16><<<grid, kWarps * 32, 0, s>>>(a);
    return check_launch("fa_paged");
  }
  const Workspace w = workspace_of(a);
  char* ws = static_cast<char*>(a.ws);
  StreamArgs p{};
  p.q = a.q, p.q_bf16 = dtype == KQ_BF16;
  p.k = a.k, p.v = a.v, p.num_pages = a.num_pages;
  p.ps = a.ps, p.W = a.W, p.Hq = a.Hq, p.Hkv = a.Hkv, p.table = a.table, p.prefix_len = through0;
  p.G = a.Hq / a.Hkv;
  p.QG = (p.G + 15) / 16;
  p.split.seq_lens = a.seq_lens, p.split.B = a.B, p.split.start = chunks ? a.prefix_len : 0;
  p.split.limit = (int)std::min<long long>(a.max_seqlen, (long long)a.W * a.ps);
  // Little to stream is bound by latency: fewer warps with deeper rings start
  // sooner (3000 tokens of one sequence, 8 KV heads of 128: 11.0 us with 8
  // warps, 13.7 with 12; 4 x 9000: 21.8 and 25.3); more is bound by issue
  // slots (16 x 3000: 30.1 and 28.1, 16 x 16000: 112 and 102). Heads of 64: 4 x
  // 9000 22.8 and 23.7, 16 x 3000 29.4 and 26.9; 32 KV heads: 1 x 3000 16.6 and
  // 18.6, 4 x 9000 88 and 84; one KV head: 16 x 9000 20.6 and 24.1.
  const long long units = (long long)a.B * a.Hkv * p.QG * ((p.split.limit - p.split.start) / kUnit + 1);
  p.warps = units <= 16ll * kFewWarps * sm_count() ? kFewWarps : kStreamWarps;
  p.split.workers = workers_of(a, p.warps);
  p.sl = a.scale * 1.44269504088896340736f;
  p.part = reinterpret_cast<float*>(ws + w.part), p.ml = reinterpret_cast<float2*>(ws + w.ml);
  kq_status_t st = KQ_OK;
  if (chunks) {
    PrefixArgs x{};
    x.q = a.q, x.q_bf16 = p.q_bf16, x.k = a.k, x.v = a.v, x.num_pages = a.num_pages;
    x.ps = a.ps, x.B = a.B, x.Hq = a.Hq, x.Hkv = a.Hkv, x.G = p.G;
    x.prefix_len = a.prefix_len, x.limit = p.split.limit, x.chunks = chunks;
    x.table = a.table, x.seq_lens = a.seq_lens;
    x.flip = p.sl < 0.0f ? 0x80000000u : 0u;
    x.scale = a.scale;
    x.sl = fmaxf(fabsf(p.sl), kMinScale);
    x.part = reinterpret_cast<float*>(ws + w.ppart), x.ml = reinterpret_cast<float2*>(ws + w.pml);
    x.err = device_error_word();
    const int pgrid = prefix_groups(a) * chunks;
    switch (a.D / 32) {
      case 1: st = launch_prefix_nb<1>(x, pgrid, s); break;
      case 2: st = launch_prefix_nb<2>(x, pgrid, s); break;
      case 3: st = launch_prefix_nb<3>(x, pgrid, s); break;
      default: st = launch_prefix_nb<4>(x, pgrid, s); break;
    }
    if (st) return st;
  }
  const bool pdl = chunks > 0;
  switch (a.D / 32) {
    case 1: st = launch_stream_nb<1>(p, pdl, s); break;
    case 2: st = launch_stream_nb<2>(p, pdl, s); break;
    case 3: st = launch_stream_nb<3>(p, pdl, s); break;
    case 4: st = launch_stream_nb<4>(p, pdl, s); break;
    case 5: st = launch_stream_nb<5>(p, pdl, s); break;
    case 6: st = launch_stream_nb<6>(p, pdl, s); break;
    case 7: st = launch_stream_nb<7>(p, pdl, s); break;
    default: st = launch_stream_nb<8>(p, pdl, s); break;
  }
  if (st) return st;
  CombineArgs ca{p.split, p.part, p.ml, reinterpret_cast<float*>(ws + w.ppart), reinterpret_cast<float2*>(ws + w.pml),
                 chunks, a.Hq, a.D, a.out};
  return dtype == KQ_F16 ? launch_combine_d<__half>(ca, s) : launch_combine_d<__nv_bfloat16>(ca, s);
}

}  // namespace kq
