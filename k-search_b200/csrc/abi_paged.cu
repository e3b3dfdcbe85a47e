// C ABI of the paged-serving operators: argument checks in front of paged.cu,
// fa_prompt.cu and fa_paged.cu.
#include "kq_internal.h"

using namespace kq;

namespace {

bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }

kq_status_t check_dtype(int dtype, const char* what) {
  if (dtype != KQ_F16 && dtype != KQ_BF16) return fail(KQ_ERR_INVALID, "%s: unknown dtype %d", what, dtype);
  return KQ_OK;
}

kq_status_t check_cache_shape(int Hkv, int D, const char* what) {
  if (Hkv <= 0 || D <= 0 || D % 32 || D > 256)
    return fail(KQ_ERR_INVALID, "%s: bad shape Hkv=%d D=%d (D must be a multiple of 32, <= 256)", what, Hkv, D);
  return KQ_OK;
}

struct Span {
  const void* p;
  size_t bytes;
};
bool overlap(const Span& a, const Span& b) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a.p), y = reinterpret_cast<uintptr_t>(b.p);
  return a.bytes > 0 && b.bytes > 0 && x < y + b.bytes && y < x + a.bytes;
}

FaPromptArgs prompt_args(int B, int Tq, int Tk, int Hq, int Hkv, int D) {
  FaPromptArgs a{};
  a.B = B, a.Tq = Tq, a.Tk = Tk, a.Hq = Hq, a.Hkv = Hkv, a.D = D;
  return a;
}

bool prompt_shape_ok(int B, int Tq, int Tk, int Hq, int Hkv, int D) {
  return B >= 0 && Tq >= 0 && Tk >= 0 && Hq > 0 && Hkv > 0 && Hq % Hkv == 0 && D > 0 && D % 8 == 0 && D <= 256;
}

FaPagedArgs paged_args(int B, int Hq, int Hkv, int D, int prefix_len, int max_seqlen) {
  FaPagedArgs a{};
  a.B = B, a.Hq = Hq, a.Hkv = Hkv, a.D = D, a.prefix_len = prefix_len, a.max_seqlen = max_seqlen;
  return a;
}

bool paged_shape_ok(int B, int Hq, int Hkv, int D, int prefix_len, int max_seqlen) {
  return B >= 0 && Hq > 0 && Hkv > 0 && Hq % Hkv == 0 && D > 0 && D % 32 == 0 && D <= 256 && prefix_len >= 0 &&
         max_seqlen >= 0;
}

}  // namespace

extern "C" {

kq_status_t kq_page_plan(const int32_t* cached_lens, const int32_t* new_lens, int B, int32_t* block_tables,
                         int max_blocks, const int32_t* free_pages, int num_free, int page_size, int64_t total_new,
                         int64_t* slots, int32_t* seq_lens, int32_t* cu_new, int32_t* cu_seqlens, int32_t* counts,
                         kq_stream_t stream) {
  if (B < 0 || max_blocks < 0 || num_free < 0 || page_size <= 0 || total_new < 0 || total_new > 0x7fffffff)
    return fail(KQ_ERR_INVALID, "page_plan: bad shape B=%d max_blocks=%d num_free=%d page_size=%d total_new=%lld", B,
                max_blocks, num_free, page_size, (long long)total_new);
  if (!cu_new || !cu_seqlens || !counts || (total_new > 0 && !slots) || (num_free > 0 && !free_pages) ||
      (B > 0 && (!cached_lens || !new_lens || !seq_lens || (max_blocks > 0 && !block_tables))))
    return fail(KQ_ERR_INVALID, "page_plan: null pointer");
  // the kernel's CTAs read the inputs while others already write: no output may
  // lie on them, or on another output, but seq_lens exactly on the lengths it updates
  const size_t w = sizeof(int32_t);
  const Span in[3] = {{cached_lens, B * w}, {new_lens, B * w}, {free_pages, num_free * w}};
  const Span out[6] = {{seq_lens, B * w},        {block_tables, (size_t)B * max_blocks * w}, {slots, total_new * sizeof(int64_t)},
                       {cu_new, (B + (size_t)1) * w}, {cu_seqlens, (B + (size_t)1) * w},          {counts, 2 * w}};
  for (int o = 0; o < 6; ++o) {
    for (int i = 0; i < 3; ++i)
      if (overlap(out[o], in[i]) && !(o == 0 && i < 2 && out[o].p == in[i].p))
        return fail(KQ_ERR_INVALID, "page_plan: an output overlaps an input (only seq_lens may be cached_lens or new_lens)");
    for (int i = 0; i < o; ++i)
      if (overlap(out[o], out[i])) return fail(KQ_ERR_INVALID, "page_plan: two outputs overlap");
  }
  return launch_page_plan(cached_lens, new_lens, B, block_tables, max_blocks, free_pages, num_free, page_size,
                          total_new, slots, seq_lens, cu_new, cu_seqlens, counts, static_cast<cudaStream_t>(stream));
}

kq_status_t kq_page_write_q8_0(int dtype, const void* k, const void* v, int64_t k_row_stride, int64_t k_head_stride,
                               int64_t v_row_stride, int64_t v_head_stride, const int64_t* slots, int64_t T, int Hkv,
                               int D, void* k_cache, void* v_cache, int64_t num_slots, kq_stream_t stream) {
  if (kq_status_t st = check_dtype(dtype, "page_write")) return st;
  if (kq_status_t st = check_cache_shape(Hkv, D, "page_write")) return st;
  if (T < 0 || num_slots < 0) return fail(KQ_ERR_INVALID, "page_write: bad shape T=%lld", (long long)T);
  if (T == 0) return KQ_OK;
  if (!k || !v || !slots || (num_slots > 0 && (!k_cache || !v_cache)))
    return fail(KQ_ERR_INVALID, "page_write: null pointer");
  if (!aligned(k_cache, 2) || !aligned(v_cache, 2) || !aligned(k, 2) || !aligned(v, 2))
    return fail(KQ_ERR_INVALID, "page_write: rows and caches must be 2-byte aligned");
  const int64_t strides[4] = {k_row_stride, k_head_stride, v_row_stride, v_head_stride};
  return launch_page_write_q8_0(dtype, k, v, strides, slots, T, Hkv, D, k_cache, v_cache, num_slots,
                                static_cast<cudaStream_t>(stream));
}

kq_status_t kq_page_read_q8_0(int dtype, const void* k_cache, const void* v_cache, int64_t num_pages, int page_size,
                              int Hkv, int D, const int32_t* block_tables, int max_blocks, const int32_t* cu_seqlens,
                              int B, int64_t total_rows, void* k, void* v, kq_stream_t stream) {
  if (kq_status_t st = check_dtype(dtype, "page_read")) return st;
  if (kq_status_t st = check_cache_shape(Hkv, D, "page_read")) return st;
  if (num_pages < 0 || page_size <= 0 || max_blocks < 0 || B < 0 || total_rows < 0 || total_rows > 0x7fffffff)
    return fail(KQ_ERR_INVALID, "page_read: bad shape num_pages=%lld page_size=%d max_blocks=%d B=%d total_rows=%lld",
                (long long)num_pages, page_size, max_blocks, B, (long long)total_rows);
  if (total_rows == 0) return KQ_OK;
  if (B == 0) return fail(KQ_ERR_INVALID, "page_read: rows without a sequence");
  if (!k || !v || !cu_seqlens || (max_blocks > 0 && !block_tables) || (num_pages > 0 && (!k_cache || !v_cache)))
    return fail(KQ_ERR_INVALID, "page_read: null pointer");
  if (!aligned(k_cache, 16) || !aligned(v_cache, 16) || !aligned(k, 16) || !aligned(v, 16))
    return fail(KQ_ERR_INVALID, "page_read: caches, k and v must be 16-byte aligned");
  return launch_page_read_q8_0(dtype, k_cache, v_cache, num_pages, page_size, Hkv, D, block_tables, max_blocks,
                               cu_seqlens, B, total_rows, k, v, static_cast<cudaStream_t>(stream));
}

size_t kq_fa_prompt_workspace(int B, int Tq, int Tk, int Hq, int Hkv, int D) {
  if (!prompt_shape_ok(B, Tq, Tk, Hq, Hkv, D)) return 0;
  return fa_prompt_workspace(prompt_args(B, Tq, Tk, Hq, Hkv, D));
}

kq_status_t kq_fa_prompt(int dtype, const void* q, const void* k, const void* v, int64_t q_row_stride,
                         int64_t q_head_stride, int64_t k_row_stride, int64_t k_head_stride, int64_t v_row_stride,
                         int64_t v_head_stride, const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k, int B, int Tq,
                         int Tk, int Hq, int Hkv, int D, int causal, float scale, void* out, void* workspace,
                         size_t workspace_bytes, kq_stream_t stream) {
  if (kq_status_t st = check_dtype(dtype, "fa_prompt")) return st;
  if (!prompt_shape_ok(B, Tq, Tk, Hq, Hkv, D))
    return fail(KQ_ERR_INVALID, "fa_prompt: bad shape B=%d Tq=%d Tk=%d Hq=%d Hkv=%d D=%d (D must be a multiple of 8, <= 256)",
                B, Tq, Tk, Hq, Hkv, D);
  if (Tq == 0) return KQ_OK;
  if (B == 0) return fail(KQ_ERR_INVALID, "fa_prompt: rows without a sequence");
  if (!q || !out || !cu_seqlens_q || !cu_seqlens_k || (Tk > 0 && (!k || !v)))
    return fail(KQ_ERR_INVALID, "fa_prompt: null pointer");
  if (!aligned(q, 2) || !aligned(k, 2) || !aligned(v, 2) || !aligned(out, 16))
    return fail(KQ_ERR_INVALID, "fa_prompt: q, k, v must be 2-byte and out 16-byte aligned");
  FaPromptArgs a = prompt_args(B, Tq, Tk, Hq, Hkv, D);
  a.q = q, a.k = k, a.v = v;
  a.q_row = q_row_stride, a.q_head = q_head_stride, a.k_row = k_row_stride, a.k_head = k_head_stride;
  a.v_row = v_row_stride, a.v_head = v_head_stride;
  a.cu_q = cu_seqlens_q, a.cu_k = cu_seqlens_k;
  a.causal = causal ? 1 : 0;
  a.scale = scale;
  a.out = out;
  a.ws = workspace;
  const size_t need = fa_prompt_workspace(a);
  if (need > 0 && (!workspace || workspace_bytes < need || !aligned(workspace, 16)))
    return fail(KQ_ERR_INVALID, "fa_prompt: needs a 16-byte aligned workspace of %zu bytes", need);
  return launch_fa_prompt(a, dtype, static_cast<cudaStream_t>(stream));
}

size_t kq_fa_decode_paged_workspace(int B, int Hq, int Hkv, int D, int prefix_len, int max_seqlen) {
  if (!paged_shape_ok(B, Hq, Hkv, D, prefix_len, max_seqlen)) return 0;
  return fa_paged_workspace(paged_args(B, Hq, Hkv, D, prefix_len, max_seqlen));
}

kq_status_t kq_fa_decode_paged(int dtype, const void* q, const void* k_cache, const void* v_cache, int64_t num_pages,
                               int page_size, const int32_t* block_tables, int max_blocks, const int32_t* seq_lens,
                               int B, int Hq, int Hkv, int D, int prefix_len, int max_seqlen, float scale, void* out,
                               void* workspace, size_t workspace_bytes, kq_stream_t stream) {
  if (kq_status_t st = check_dtype(dtype, "fa_decode_paged")) return st;
  if (!paged_shape_ok(B, Hq, Hkv, D, prefix_len, max_seqlen) || num_pages < 0 || page_size <= 0 || max_blocks < 0)
    return fail(KQ_ERR_INVALID,
                "fa_decode_paged: bad shape B=%d Hq=%d Hkv=%d D=%d prefix_len=%d max_seqlen=%d page_size=%d "
                "max_blocks=%d (D must be a multiple of 32, <= 256)",
                B, Hq, Hkv, D, prefix_len, max_seqlen, page_size, max_blocks);
  if ((long long)prefix_len > (long long)max_blocks * page_size)
    return fail(KQ_ERR_INVALID, "fa_decode_paged: prefix_len=%d is past the block table (%d pages of %d)", prefix_len,
                max_blocks, page_size);
  if (B == 0) return KQ_OK;
  if (!q || !out || !seq_lens || (max_blocks > 0 && !block_tables) || (num_pages > 0 && (!k_cache || !v_cache)))
    return fail(KQ_ERR_INVALID, "fa_decode_paged: null pointer");
  if (!aligned(q, 16) || !aligned(out, 16)) return fail(KQ_ERR_INVALID, "fa_decode_paged: q and out must be 16-byte aligned");
  if (!aligned(k_cache, 16) || !aligned(v_cache, 16))
    return fail(KQ_ERR_INVALID, "fa_decode_paged: caches must be 16-byte aligned");
  FaPagedArgs a = paged_args(B, Hq, Hkv, D, prefix_len, max_seqlen);
  a.q = q, a.out = out;
  a.k = static_cast<const uint8_t*>(k_cache), a.v = static_cast<const uint8_t*>(v_cache);
  a.num_pages = num_pages, a.ps = page_size, a.table = block_tables, a.W = max_blocks, a.seq_lens = seq_lens;
  a.scale = scale;
  a.ws = workspace;
  const size_t need = fa_paged_workspace(a);
  if (need > 0 && (!workspace || workspace_bytes < need || !aligned(workspace, 16)))
    return fail(KQ_ERR_INVALID, "fa_decode_paged: needs a 16-byte aligned workspace of %zu bytes", need);
  return launch_fa_paged(a, dtype, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
