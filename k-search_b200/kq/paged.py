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

import ctypes
import math
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


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


def _tensor(t, name: str, dtype, device=None) -> torch.Tensor:
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor")
    if t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")
    return t


def _ints(t, name: str, device, shape) -> torch.Tensor:
    _tensor(t, name, torch.int32, device)
    if t.shape != shape:
        raise ValueError(f"{name} must be {list(shape)}, got {list(t.shape)}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return t


def _rows(t, name: str, dtype, device=None) -> torch.Tensor:
    _tensor(t, name, dtype, device)
    if t.dim() != 3:
        raise ValueError(f"{name} must be [tokens, heads, head_dim], got {list(t.shape)}")
    if t.stride(2) != 1 and t.shape[2] > 1 and t.numel() > 0:
        raise ValueError(f"{name}'s head dimension must be contiguous")
    return t


def _float16(t, name: str) -> int:
    if not isinstance(t, torch.Tensor) or t.dtype not in DTYPES:
        raise ValueError(f"{name} must be a float16 or bfloat16 CUDA tensor")
    return DTYPES[t.dtype]


def _caches(k_cache, v_cache, device) -> tuple[int, int, int, int]:
    """(num_pages, page_size, Hkv, D) of a checked cache pair."""
    for t, name in ((k_cache, "k_cache"), (v_cache, "v_cache")):
        _tensor(t, name, torch.uint8, device)
        if t.dim() != 5 or t.shape[4] != 34 or not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous uint8 [num_pages, page_size, Hkv, D/32, 34], got {list(t.shape)}")
    if k_cache.shape != v_cache.shape:
        raise ValueError(f"k_cache {list(k_cache.shape)} and v_cache {list(v_cache.shape)} differ")
    pages, ps, hkv, nb, _ = k_cache.shape
    return pages, ps, hkv, nb * 32


class _on:
    """Makes the tensors' device current for a launch (nothing to do when it is already)."""

    def __init__(self, device):
        self.device = device
        self.before = torch.cuda.current_device()

    def __enter__(self):
        if self.device.index != self.before:
            torch.cuda.set_device(self.device)
        return torch.cuda.current_stream().cuda_stream

    def __exit__(self, *_):
        if self.device.index != self.before:
            torch.cuda.set_device(self.before)


def page_plan(cached_lens: torch.Tensor, new_lens: torch.Tensor, block_tables: torch.Tensor, free_pages: torch.Tensor,
              page_size: int, total_new: int, out: PagePlan | None = None) -> PagePlan:
    """Block tables and slot map of one serving step, built on the GPU.

    cached_lens, new_lens int32 [B]: tokens already cached and added now, per
    request. block_tables int32 [B, max_blocks] is updated in place: request
    b's new pages come from free_pages int32 [F], in request order, and are
    appended at column ceil(cached / page_size). total_new (host) is the slot
    map's length, sum(new_lens) where nothing pads it. counts[0] > F: the list
    was too short (the missing entries are -1); counts[1] > 0: that many new
    tokens got no slot. ``out``: an earlier plan whose tensors are reused."""
    dev = _tensor(cached_lens, "cached_lens", torch.int32).device
    B = cached_lens.numel()
    _ints(cached_lens, "cached_lens", dev, (B,))
    _ints(new_lens, "new_lens", dev, (B,))
    _tensor(block_tables, "block_tables", torch.int32, dev)
    _need(block_tables.dim() == 2 and block_tables.shape[0] == B and block_tables.is_contiguous(),
          f"block_tables must be contiguous [{B}, max_blocks]")
    F = free_pages.numel() if isinstance(free_pages, torch.Tensor) else -1
    _ints(free_pages, "free_pages", dev, (F,))
    if out is None:
        ints = torch.empty(3 * B + 4, dtype=torch.int32, device=dev)
        out = PagePlan(torch.empty(total_new, dtype=torch.int64, device=dev), ints[:B], ints[B:2 * B + 1],
                       ints[2 * B + 1:3 * B + 2], ints[3 * B + 2:])
    else:
        _tensor(out.slots, "out.slots", torch.int64, dev)
        _need(out.slots.shape == (total_new,) and out.slots.is_contiguous(), f"out.slots must be [{total_new}]")
        _ints(out.seq_lens, "out.seq_lens", dev, (B,))
        _ints(out.cu_new, "out.cu_new", dev, (B + 1,))
        _ints(out.cu_seqlens, "out.cu_seqlens", dev, (B + 1,))
        _ints(out.counts, "out.counts", dev, (2,))
    with _on(dev) as stream:
        check(lib().kq_page_plan(cached_lens.data_ptr(), new_lens.data_ptr(), B, block_tables.data_ptr(),
                                 block_tables.shape[1], free_pages.data_ptr(), F, page_size, total_new,
                                 out.slots.data_ptr(), out.seq_lens.data_ptr(), out.cu_new.data_ptr(),
                                 out.cu_seqlens.data_ptr(), out.counts.data_ptr(), stream), "kq_page_plan")
    return out


def page_write(k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, k_cache: torch.Tensor,
               v_cache: torch.Tensor) -> None:
    """Quantises rows k, v (fp16 or bf16 [T, Hkv, D], any row and head strides)
    into the q8_0 cache rows slots[t] (int64; rows with a negative slot, or one
    past the cache, are skipped)."""
    dt = _float16(k, "k")
    dev = _rows(k, "k", k.dtype).device
    _rows(v, "v", k.dtype, dev)
    pages, ps, hkv, d = _caches(k_cache, v_cache, dev)
    T = k.shape[0]
    _need(k.shape == v.shape and k.shape[1:] == (hkv, d), f"k and v must be [T, {hkv}, {d}], got {list(k.shape)} and {list(v.shape)}")
    _tensor(slots, "slots", torch.int64, dev)
    _need(slots.shape == (T,) and slots.is_contiguous(), f"slots must be contiguous [{T}]")
    with _on(dev) as stream:
        check(lib().kq_page_write_q8_0(dt, k.data_ptr(), v.data_ptr(), k.stride(0), k.stride(1), v.stride(0),
                                       v.stride(1), slots.data_ptr(), T, hkv, d, k_cache.data_ptr(),
                                       v_cache.data_ptr(), pages * ps, stream), "kq_page_write_q8_0")


def page_read(k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor, cu_seqlens: torch.Tensor,
              total_rows: int, dtype: torch.dtype = torch.float16) -> tuple[torch.Tensor, torch.Tensor]:
    """The sequences' cache rows in packed order: k, v [total_rows, Hkv, D] of
    ``dtype``, row cu_seqlens[b] + i being token i of sequence b. For the
    prompt attention of a chunk that follows cached tokens."""
    _need(dtype in DTYPES, f"dtype must be float16 or bfloat16, got {dtype}")
    dev = _tensor(k_cache, "k_cache", torch.uint8).device
    pages, ps, hkv, d = _caches(k_cache, v_cache, dev)
    _tensor(block_tables, "block_tables", torch.int32, dev)
    _need(block_tables.dim() == 2 and block_tables.is_contiguous(), "block_tables must be contiguous [B, max_blocks]")
    B = block_tables.shape[0]
    _ints(cu_seqlens, "cu_seqlens", dev, (B + 1,))
    k = torch.empty((total_rows, hkv, d), dtype=dtype, device=dev)
    v = torch.empty_like(k)
    with _on(dev) as stream:
        check(lib().kq_page_read_q8_0(DTYPES[dtype], k_cache.data_ptr(), v_cache.data_ptr(), pages, ps, hkv, d,
                                      block_tables.data_ptr(), block_tables.shape[1], cu_seqlens.data_ptr(), B,
                                      total_rows, k.data_ptr(), v.data_ptr(), stream), "kq_page_read_q8_0")
    return k, v


def _workspace(nbytes: int, device) -> tuple[torch.Tensor | None, int]:
    """Scratch from torch's caching allocator: ordered on the current stream, so
    calls on different streams never share it."""
    if nbytes == 0:
        return None, 0
    ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
    return ws, ws.data_ptr()


def _out_like(q: torch.Tensor, out) -> torch.Tensor:
    if out is None:
        return torch.empty(q.shape, dtype=q.dtype, device=q.device)
    _tensor(out, "out", q.dtype, q.device)
    _need(out.shape == q.shape and out.is_contiguous(), f"out must be contiguous {list(q.shape)}")
    return out


def flash_prompt_ragged(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cu_seqlens_q: torch.Tensor,
                        cu_seqlens_k: torch.Tensor | None = None, causal: bool = True, scale: float | None = None,
                        out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of packed prompts -> [Tq, Hq, D]. q [Tq, Hq, D], k, v
    [Tk, Hkv, D] fp16 or bf16 (views of a fused projection are fine: only the
    head dimension has to be contiguous); cu_seqlens_q, cu_seqlens_k int32
    [B+1] on the device (cu_seqlens_k defaults to cu_seqlens_q). causal: row i
    of a sequence sees keys up to i + (len_k - len_q), so a chunk sees the
    context before it; a row without keys is zero."""
    dt = _float16(q, "q")
    dev = _rows(q, "q", q.dtype).device
    _rows(k, "k", q.dtype, dev)
    _rows(v, "v", q.dtype, dev)
    Tq, Hq, D = q.shape
    Tk, Hkv = k.shape[0], k.shape[1]
    _need(k.shape == v.shape and k.shape[2] == D, f"k and v must be [Tk, Hkv, {D}], got {list(k.shape)} and {list(v.shape)}")
    _tensor(cu_seqlens_q, "cu_seqlens_q", torch.int32, dev)
    B = cu_seqlens_q.numel() - 1
    _need(B >= 0, "cu_seqlens_q must be [B + 1]")
    _ints(cu_seqlens_q, "cu_seqlens_q", dev, (B + 1,))
    if cu_seqlens_k is None:
        _need(Tq == Tk, f"cu_seqlens_k is needed where q has {Tq} rows and k {Tk}")
        cu_seqlens_k = cu_seqlens_q
    else:
        _ints(cu_seqlens_k, "cu_seqlens_k", dev, (B + 1,))
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    out = _out_like(q, out)
    L = lib()
    nbytes = L.kq_fa_prompt_workspace(B, Tq, Tk, Hq, Hkv, D)
    with _on(dev) as stream:
        ws, ptr = _workspace(nbytes, dev)
        check(L.kq_fa_prompt(dt, q.data_ptr(), k.data_ptr(), v.data_ptr(), q.stride(0), q.stride(1), k.stride(0),
                             k.stride(1), v.stride(0), v.stride(1), cu_seqlens_q.data_ptr(), cu_seqlens_k.data_ptr(),
                             B, Tq, Tk, Hq, Hkv, D, int(causal), ctypes.c_float(scale), out.data_ptr(), ptr, nbytes,
                             stream), "kq_fa_prompt")
    return out


def flash_decode_paged(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor,
                       seq_lens: torch.Tensor, prefix_len: int = 0, max_seqlen: int | None = None,
                       scale: float | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Decode over the paged q8_0 cache, one query token per sequence ->
    [B, Hq, D]. q fp16 or bf16 [B, Hq, D]; block_tables int32 [B, max_blocks];
    seq_lens int32 [B] (device; 0: a padding row, zeros out). The first
    prefix_len tokens are the same pages for every sequence: they are read
    once for the whole batch, through row 0 of block_tables. max_seqlen (host)
    bounds seq_lens, longer sequences are cut to it; it defaults to the
    tables' width."""
    dt = _float16(q, "q")
    dev = _rows(q, "q", q.dtype).device
    _need(q.is_contiguous(), "q must be contiguous")
    pages, ps, hkv, d = _caches(k_cache, v_cache, dev)
    B, Hq, D = q.shape
    _need(D == d, f"q has head dimension {D}, the caches {d}")
    _tensor(block_tables, "block_tables", torch.int32, dev)
    _need(block_tables.dim() == 2 and block_tables.shape[0] == B and block_tables.is_contiguous(),
          f"block_tables must be contiguous [{B}, max_blocks]")
    _ints(seq_lens, "seq_lens", dev, (B,))
    W = block_tables.shape[1]
    max_seqlen = W * ps if max_seqlen is None else min(int(max_seqlen), W * ps)
    if scale is None:
        scale = 1.0 / math.sqrt(D)
    out = _out_like(q, out)
    L = lib()
    nbytes = L.kq_fa_decode_paged_workspace(B, Hq, hkv, D, prefix_len, max_seqlen)
    with _on(dev) as stream:
        ws, ptr = _workspace(nbytes, dev)
        check(L.kq_fa_decode_paged(dt, q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), pages, ps,
                                   block_tables.data_ptr(), W, seq_lens.data_ptr(), B, Hq, hkv, D, prefix_len,
                                   max_seqlen, ctypes.c_float(scale), out.data_ptr(), ptr, nbytes, stream),
              "kq_fa_decode_paged")
    return out
