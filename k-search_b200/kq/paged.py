"""Paged serving: block tables and slot maps, the paged q8_0 KV cache, prompt
attention, and decode attention for a batch with a shared prefix.

One serving step with these:

    plan = kq.page_plan(cached_lens, new_lens, block_tables, free_pages, page_size, total_new)
    kq.page_write(k, v, plan.slots, k_cache, v_cache)
    out = kq.flash_prompt_ragged(q, k, v, plan.cu_new)                    # prompts
    out = kq.flash_decode_paged(q, k_cache, v_cache, block_tables, plan.seq_lens, prefix_len=...)  # one token each

Everything runs on the current CUDA stream of the tensors' device and nothing
is read back to the host. Tensors belong to one device. Caches are uint8
[num_pages, page_size, Hkv, D/32, 34] (q8_0 blocks).
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from ._lib import check, lib

DTYPES = {torch.float16: 0, torch.bfloat16: 1}


class PagePlan(NamedTuple):
    slots: torch.Tensor       # int64 [total_new]: cache row of each new token, -1 without one
    seq_lens: torch.Tensor    # int32 [B]: cached + new
    cu_new: torch.Tensor      # int32 [B + 1]: prefix sums of the new lengths
    cu_seqlens: torch.Tensor  # int32 [B + 1]: prefix sums of seq_lens
    counts: torch.Tensor      # int32 [2]: pages the step needs, new tokens without a slot


# The checks run on every call, in front of kernels of a few microseconds: they
# read each attribute once and build messages only to raise.
def _tensor(t, name: str, dtype, device=None) -> torch.Tensor:
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if t.dtype is not dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    if device is not None and t.get_device() != device.index:
        raise ValueError(f"{name} is on {t.device}, expected {device}")
    return t


def _vector(t, name: str, dtype, device, n: int) -> None:
    if isinstance(t, torch.Tensor) and t.dtype is dtype and t.get_device() == device.index and t.numel() == n \
            and t.dim() == 1 and t.is_contiguous():
        return
    _tensor(t, name, dtype, device)
    raise ValueError(f"{name} must be contiguous [{n}], got {list(t.shape)}")


def _numel(t, name: str) -> int:
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    return t.numel()


def _table(t, device, B: int | None) -> torch.Size:
    _tensor(t, "block_tables", torch.int32, device)
    shape = t.shape
    if len(shape) != 2 or (B is not None and shape[0] != B) or not t.is_contiguous():
        raise ValueError(f"block_tables must be contiguous [{'B' if B is None else B}, max_blocks], got {list(shape)}")
    return shape


def _rows(t, name: str, dtype, device=None) -> torch.Size:
    _tensor(t, name, dtype, device)
    shape = t.shape
    if len(shape) != 3:
        raise ValueError(f"{name} must be [tokens, heads, head_dim], got {list(shape)}")
    if t.stride(2) != 1 and shape[2] > 1 and t.numel() > 0:
        raise ValueError(f"{name}'s head dimension must be contiguous")
    return shape


def _float16(t, name: str) -> int:
    dt = DTYPES.get(t.dtype) if isinstance(t, torch.Tensor) else None
    if dt is None:
        raise ValueError(f"{name} must be a float16 or bfloat16 CUDA tensor")
    return dt


def _caches(k_cache, v_cache, device) -> torch.Size:
    """[num_pages, page_size, Hkv, D/32, 34] of a checked cache pair."""
    for t, name in ((k_cache, "k_cache"), (v_cache, "v_cache")):
        _tensor(t, name, torch.uint8, device)
        if t.dim() != 5 or t.size(4) != 34 or not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous uint8 [num_pages, page_size, Hkv, D/32, 34], got {list(t.shape)}")
    shape = k_cache.shape
    if shape != v_cache.shape:
        raise ValueError(f"k_cache {list(shape)} and v_cache {list(v_cache.shape)} differ")
    return shape


_raw_stream, _current_device = torch._C._cuda_getCurrentRawStream, torch._C._cuda_getDevice


def _call(entry: str, device: torch.device, *args) -> None:
    """entry(*args, current stream of `device`) with that device current."""
    before = _current_device()
    if device.index == before:
        status = getattr(lib(), entry)(*args, _raw_stream(before))
    else:
        with torch.cuda.device(device):
            status = getattr(lib(), entry)(*args, _raw_stream(device.index))
    if status:
        check(status, entry)


def page_plan(cached_lens: torch.Tensor, new_lens: torch.Tensor, block_tables: torch.Tensor, free_pages: torch.Tensor,
              page_size: int, total_new: int, out: PagePlan | None = None) -> PagePlan:
    """Block tables and slot map of one serving step, built on the GPU.

    cached_lens, new_lens int32 [B]: tokens already cached and added now, per
    request. block_tables int32 [B, max_blocks] is updated in place: request
    b's new pages come from free_pages int32 [F], in request order, and are
    appended at column ceil(cached / page_size). total_new (host) is the slot
    map's length, sum(new_lens) where nothing pads it. counts[0] > F: the list
    was too short (the missing entries are -1); counts[1] > 0: that many new
    tokens got no slot. ``out``: an earlier plan whose tensors are reused;
    cached_lens may be its seq_lens, which then advance in place. Outputs that
    overlap inputs in any other way are refused."""
    B, F = _numel(cached_lens, "cached_lens"), _numel(free_pages, "free_pages")
    dev = cached_lens.device
    _vector(cached_lens, "cached_lens", torch.int32, dev, B)
    _vector(new_lens, "new_lens", torch.int32, dev, B)
    W = _table(block_tables, dev, B)[1]
    _vector(free_pages, "free_pages", torch.int32, dev, F)
    if out is None:
        slots = cached_lens.new_empty(total_new, dtype=torch.int64)
        seq_lens, cu_new, cu_seqlens, counts = torch.split_with_sizes(cached_lens.new_empty(3 * B + 4),
                                                                      (B, B + 1, B + 1, 2))
        out = PagePlan(slots, seq_lens, cu_new, cu_seqlens, counts)
    else:
        slots, seq_lens, cu_new, cu_seqlens, counts = out
        _vector(slots, "out.slots", torch.int64, dev, total_new)
        _vector(seq_lens, "out.seq_lens", torch.int32, dev, B)
        _vector(cu_new, "out.cu_new", torch.int32, dev, B + 1)
        _vector(cu_seqlens, "out.cu_seqlens", torch.int32, dev, B + 1)
        _vector(counts, "out.counts", torch.int32, dev, 2)
    _call("kq_page_plan", dev, cached_lens.data_ptr(), new_lens.data_ptr(), B, block_tables.data_ptr(), W,
          free_pages.data_ptr(), F, page_size, total_new, slots.data_ptr(), seq_lens.data_ptr(), cu_new.data_ptr(),
          cu_seqlens.data_ptr(), counts.data_ptr())
    return out


def page_write(k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, k_cache: torch.Tensor,
               v_cache: torch.Tensor) -> None:
    """Quantises rows k, v (fp16 or bf16 [T, Hkv, D], any row and head strides)
    into the q8_0 cache rows slots[t] (int64; rows with a negative slot, or one
    past the cache, are skipped)."""
    dt = _float16(k, "k")
    shape = _rows(k, "k", k.dtype)
    dev = k.device
    pages, ps, hkv, nb, _ = _caches(k_cache, v_cache, dev)
    T, h, d = shape
    if _rows(v, "v", k.dtype, dev) != shape or h != hkv or d != nb * 32:
        raise ValueError(f"k and v must be [T, {hkv}, {nb * 32}], got {list(shape)} and {list(v.shape)}")
    _vector(slots, "slots", torch.int64, dev, T)
    ks, vs = k.stride(), v.stride()
    _call("kq_page_write_q8_0", dev, dt, k.data_ptr(), v.data_ptr(), ks[0], ks[1], vs[0], vs[1], slots.data_ptr(), T, hkv,
          d, k_cache.data_ptr(), v_cache.data_ptr(), pages * ps)


def page_read(k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor, cu_seqlens: torch.Tensor,
              total_rows: int, dtype: torch.dtype = torch.float16) -> tuple[torch.Tensor, torch.Tensor]:
    """The sequences' cache rows in packed order: k, v [total_rows, Hkv, D] of
    ``dtype``, row cu_seqlens[b] + i being token i of sequence b. For the
    prompt attention of a chunk that follows cached tokens."""
    dt = DTYPES.get(dtype)
    if dt is None:
        raise ValueError(f"dtype must be float16 or bfloat16, got {dtype}")
    dev = _tensor(k_cache, "k_cache", torch.uint8).device
    pages, ps, hkv, nb, _ = _caches(k_cache, v_cache, dev)
    B, W = _table(block_tables, dev, None)
    _vector(cu_seqlens, "cu_seqlens", torch.int32, dev, B + 1)
    k = k_cache.new_empty((total_rows, hkv, nb * 32), dtype=dtype)
    v = torch.empty_like(k)
    _call("kq_page_read_q8_0", dev, dt, k_cache.data_ptr(), v_cache.data_ptr(), pages, ps, hkv, nb * 32,
          block_tables.data_ptr(), W, cu_seqlens.data_ptr(), B, total_rows, k.data_ptr(), v.data_ptr())
    return k, v


def _out_like(q: torch.Tensor, out) -> torch.Tensor:
    if out is None:
        return torch.empty_like(q, memory_format=torch.contiguous_format)
    _tensor(out, "out", q.dtype, q.device)
    if out.shape != q.shape or not out.is_contiguous():
        raise ValueError(f"out must be contiguous {list(q.shape)}, got {list(out.shape)}")
    return out


def _workspace(nbytes: int, like: torch.Tensor) -> tuple[torch.Tensor | None, int]:
    """Scratch from torch's caching allocator: ordered on the current stream, so
    calls on different streams never share it."""
    if nbytes == 0:
        return None, 0
    ws = like.new_empty(nbytes, dtype=torch.uint8)
    return ws, ws.data_ptr()


def flash_prompt_ragged(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens_q: torch.Tensor,
                        cu_seqlens_k: torch.Tensor | None = None, causal: bool = True, scale: float | None = None,
                        out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of packed prompts -> [Tq, Hq, D]. q [Tq, Hq, D], k, v
    [Tk, Hkv, D] fp16 or bf16 (views of a fused projection are fine: only the
    head dimension has to be contiguous); cu_seqlens_q, cu_seqlens_k int32
    [B+1] on the device (cu_seqlens_k defaults to cu_seqlens_q). causal: row i
    of a sequence sees keys up to i + (len_k - len_q), so a chunk sees the
    context before it; a row without keys is zero, rows that no sequence owns
    are not specified. Prefix sums are cut to the rows that there are. Heads
    above 128 dims, and views whose rows do not start at multiples of 16 bytes,
    take a scalar kernel that is a hundred times slower and more."""
    dt = _float16(q, "q")
    Tq, Hq, D = _rows(q, "q", q.dtype)
    dev = q.device
    kshape = _rows(k, "k", q.dtype, dev)
    Tk, Hkv, Dk = kshape
    if _rows(v, "v", q.dtype, dev) != kshape or Dk != D:
        raise ValueError(f"k and v must be [Tk, Hkv, {D}], got {list(kshape)} and {list(v.shape)}")
    B = _numel(cu_seqlens_q, "cu_seqlens_q") - 1
    _vector(cu_seqlens_q, "cu_seqlens_q", torch.int32, dev, max(B, 0) + 1)
    if cu_seqlens_k is not None:
        _vector(cu_seqlens_k, "cu_seqlens_k", torch.int32, dev, B + 1)
    elif Tq == Tk:
        cu_seqlens_k = cu_seqlens_q
    else:
        raise ValueError(f"cu_seqlens_k is needed where q has {Tq} rows and k {Tk}")
    if scale is None:
        scale = D ** -0.5
    out = _out_like(q, out)
    nbytes = lib().kq_fa_prompt_workspace(B, Tq, Tk, Hq, Hkv, D)
    ws, ptr = _workspace(nbytes, q)
    qs, ks, vs = q.stride(), k.stride(), v.stride()
    _call("kq_fa_prompt", dev, dt, q.data_ptr(), k.data_ptr(), v.data_ptr(), qs[0], qs[1], ks[0], ks[1], vs[0], vs[1],
          cu_seqlens_q.data_ptr(), cu_seqlens_k.data_ptr(), B, Tq, Tk, Hq, Hkv, D, int(causal), scale, out.data_ptr(),
          ptr, nbytes)
    return out


def flash_decode_paged(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor,
                       seq_lens: torch.Tensor, prefix_len: int = 0, max_seqlen: int | None = None,
                       scale: float | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Decode over the paged q8_0 cache, one query token per sequence ->
    [B, Hq, D]. q fp16 or bf16 [B, Hq, D]; block_tables int32 [B, max_blocks];
    seq_lens int32 [B] (device; 0: a padding row, zeros out). The first
    prefix_len tokens are the same pages for every sequence: they are read
    through row 0 of block_tables (also where row 0 is a padding row), once for
    the whole batch where that pays.
    max_seqlen (host) bounds seq_lens, longer sequences are cut to it; it
    defaults to the tables' width, and a bound close to the true lengths gives
    the better work split. Pages of a multiple of 8 tokens are the fast ones:
    others take a scalar kernel, some 50 times slower."""
    dt = _float16(q, "q")
    B, Hq, D = _rows(q, "q", q.dtype)
    dev = q.device
    if not q.is_contiguous():
        raise ValueError("q must be contiguous")
    pages, ps, hkv, nb, _ = _caches(k_cache, v_cache, dev)
    if D != nb * 32:
        raise ValueError(f"q has head dimension {D}, the caches {nb * 32}")
    W = _table(block_tables, dev, B)[1]
    _vector(seq_lens, "seq_lens", torch.int32, dev, B)
    most = min(W * ps, 2 ** 31 - 1)  # a 32-bit argument
    max_seqlen = most if max_seqlen is None else min(int(max_seqlen), most)
    if scale is None:
        scale = D ** -0.5
    out = _out_like(q, out)
    nbytes = lib().kq_fa_decode_paged_workspace(B, Hq, hkv, D, prefix_len, max_seqlen)
    ws, ptr = _workspace(nbytes, q)
    _call("kq_fa_decode_paged", dev, dt, q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), pages, ps,
          block_tables.data_ptr(), W, seq_lens.data_ptr(), B, Hq, hkv, D, prefix_len, max_seqlen, scale, out.data_ptr(),
          ptr, nbytes)
    return out
