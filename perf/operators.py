"""Cases that measure the paged-serving operators: page plan, paged q8_0 cache,
prompt attention, and decode attention with a shared prefix.

``run`` computes each in plain torch where ``own`` is false and calls the
kernels' public entry points where it is true. ``exact`` computes the same in
64 bits from the definitions.
"""
from __future__ import annotations

import math
import os
import random
import sys

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
QK = 32           # elements of a q8_0 block
BLOCK_BYTES = 34  # fp16 scale and 32 int8 codes
# query heads, KV heads: the grouped layouts of the 8B and 7B definitions, the
# ungrouped harness form, and generic ones (one KV head, odd group sizes)
HEADS = ((32, 8), (28, 4), (32, 32), (16, 2), (8, 1), (15, 5))


# ---------------------------------------------------------------- cases
def listed():
    return [
        # one decode step of a small batch: every request gets one token
        {"name": "plan_decode", "op": "plan", "B": 8, "T": 8, "context": 2000, "page": 16, "prefix": 0, "mix": 1},
        # admission of a large batch of prompts behind a common system prompt
        {"name": "plan_prompts", "op": "plan", "B": 256, "T": 65536, "context": 0, "page": 32, "prefix": 1024, "mix": 2},
        # a few short follow-up turns written behind short contexts and read back
        {"name": "pages_turns", "op": "pages", "B": 3, "T": 61, "context": 211, "Hkv": 8, "D": 128, "page": 16,
         "dtype": "fp16", "mix": 3},
        # a chunk of long prompts: its rows are written, the whole context comes back for prompt attention
        {"name": "pages_chunk", "op": "pages", "B": 4, "T": 4096, "context": 8192, "Hkv": 8, "D": 128, "page": 64,
         "dtype": "bf16", "mix": 4},
        # a handful of short chat prompts
        {"name": "prompt_short", "op": "prompt", "B": 5, "T": 333, "context": 0, "Hq": 32, "Hkv": 8, "D": 128,
         "dtype": "fp16", "fused": True, "mix": 5},
        # many packed prompts of mixed lengths, an empty one and a one-token one among them
        {"name": "prompt_packed", "op": "prompt", "B": 24, "T": 8000, "context": 0, "Hq": 28, "Hkv": 4, "D": 128,
         "dtype": "bf16", "fused": True, "mix": 6},
        # one long document
        {"name": "prompt_long", "op": "prompt", "B": 1, "T": 8192, "context": 0, "Hq": 32, "Hkv": 8, "D": 128,
         "dtype": "fp16", "fused": False, "mix": 7},
        # the next chunk of a long document: few new rows against a long context
        {"name": "prompt_chunk", "op": "prompt", "B": 1, "T": 256, "context": 24000, "Hq": 32, "Hkv": 8, "D": 128,
         "dtype": "bf16", "fused": False, "mix": 8},
        # one interactive user, no shared prefix: latency counts
        {"name": "decode_single", "op": "decode", "B": 1, "prefix": 0, "suffix": 3000, "Hq": 32, "Hkv": 8, "D": 128,
         "page": 16, "dtype": "fp16", "mix": 9},
        # a batch of chats behind one long system prompt
        {"name": "decode_chats", "op": "decode", "B": 64, "prefix": 8192, "suffix": 700, "Hq": 32, "Hkv": 8, "D": 128,
         "page": 32, "dtype": "fp16", "mix": 10},
        # a large batch sampling from one document
        {"name": "decode_samples", "op": "decode", "B": 256, "prefix": 4096, "suffix": 300, "Hq": 28, "Hkv": 4, "D": 128,
         "page": 16, "dtype": "bf16", "mix": 11},
        # long separate conversations that share little
        {"name": "decode_long", "op": "decode", "B": 16, "prefix": 512, "suffix": 16000, "Hq": 32, "Hkv": 8, "D": 128,
         "page": 64, "dtype": "fp16", "mix": 12},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(("plan", "pages", "prompt", "prompt", "decode", "decode"))
    mix = rng.randrange(1 << 20)
    page = rng.choice((16, 32, 64, 128))
    dtype = rng.choice(("fp16", "bf16"))
    hq, hkv = rng.choice(HEADS)
    d = rng.choice((128, 128, 64, 96))
    if op == "plan":
        b = _log_int(rng, 1, 256)
        t = b if rng.random() < 0.4 else _log_int(rng, b, 65536)
        return {"op": op, "B": b, "T": t, "context": _log_int(rng, 1, 4000), "page": page,
                "prefix": page * rng.randrange(0, 9), "mix": mix}
    if op == "pages":
        return {"op": op, "B": _log_int(rng, 1, 8), "T": _log_int(rng, 1, 4096), "context": _log_int(rng, 1, 2048),
                "Hkv": hkv, "D": d, "page": page, "dtype": dtype, "mix": mix}
    if op == "prompt":
        if rng.random() < 0.3:  # the next chunk of one or a few requests
            return {"op": op, "B": _log_int(rng, 1, 3), "T": _log_int(rng, 1, 1024), "context": _log_int(rng, 64, 8000),
                    "Hq": hq, "Hkv": hkv, "D": d, "dtype": dtype, "fused": False, "mix": mix}
        t = _log_int(rng, 16, 8000)
        return {"op": op, "B": _log_int(rng, 1, min(t, 48)), "T": t, "context": 0, "Hq": hq, "Hkv": hkv, "D": d,
                "dtype": dtype, "fused": rng.random() < 0.5, "mix": mix}
    b = _log_int(rng, 1, 256)
    prefix = 0 if rng.random() < 0.2 else page * _log_int(rng, 1, 8192 // page)
    return {"op": op, "B": b, "prefix": prefix, "suffix": _log_int(rng, 1, min(8000, 1000000 // (b * hkv))), "Hq": hq, "Hkv": hkv,
            "D": d, "page": page, "dtype": dtype, "mix": mix}


def _split(rng, total, parts):
    """`total` cut into `parts` lengths at random places; some may be 0."""
    cuts = sorted(rng.randint(0, total) for _ in range(parts - 1))
    return [b - a for a, b in zip([0] + cuts, cuts + [total])]


def _lengths(case):
    """(cached, new) lengths of every request, from the case alone."""
    rng = random.Random(case["mix"])
    b = case["B"]
    if case["op"] == "decode":  # the padding rows of a batch of fixed size hold no token
        top = case["suffix"]
        new = [top if b == 1 else rng.randint(max(1, top // 8), top) for _ in range(b)]
        total = [case["prefix"] + n for n in new]
        if b >= 16:
            total[rng.randrange(b)] = 0
        return total, new
    new = [1] * b if case["T"] == b else _split(rng, case["T"], b)
    if b >= 6 and case["T"] > b:  # an empty request and a one-token one
        i, j, k = rng.sample(range(b), 3)
        new[k] += new[i] + new[j]
        new[i], new[j] = 0, 1
        new[k] -= 1
        if new[k] < 0:
            new[j], new[k] = 0, 0
            new[i] = case["T"] - sum(new)
    ctx = case["context"]
    if case["op"] == "prompt":
        return [0 if ctx == 0 else ctx if b == 1 else rng.randint(ctx // 2, ctx) for _ in range(b)], new
    return [case.get("prefix", 0) + (ctx if b == 1 else rng.randint(0, ctx)) for _ in range(b)], new


def _ceil(a, b):
    return -(-a // b)


# ---------------------------------------------------------------- inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _rows(g, t, h, d, dtype, scale=1.0):
    """Activations with channels of different size, as projections leave them."""
    x = torch.randn((t, h, d), generator=g, device="cuda")
    x *= torch.exp(0.4 * torch.randn((1, h, d), generator=g, device="cuda")) * scale
    return x.to(dtype)


def _random_pages(g, pages, page, hkv, d):
    """A pool of q8_0 pages as earlier writes left it."""
    c = torch.empty((pages, page, hkv, d // QK, BLOCK_BYTES), dtype=torch.uint8, device="cuda")
    amax = 2.0 + 0.5 * torch.randn((pages, page, hkv, d // QK, 1), generator=g, device="cuda").abs()
    c[..., :2] = (amax / 127).to(torch.float16).view(torch.uint8)
    x = torch.randn((pages, page, hkv, d // QK, QK), generator=g, device="cuda")
    c[..., 2:] = (x * 50).round_().clamp_(-127, 127).to(torch.int8).view(torch.uint8)
    return c


def _table(g, counts, width, pages, shared=0):
    """Block tables over randomly placed pages; the first `shared` pages are common. Returns (tables, free pages)."""
    perm = torch.randperm(pages, generator=g, device="cuda").to(torch.int32).cpu()
    table = torch.full((len(counts), width), -1, dtype=torch.int32)
    table[:, :shared] = perm[:shared]
    at = shared
    for b, n in enumerate(counts):
        own_pages = max(0, n - shared)
        table[b, shared:shared + own_pages] = perm[at:at + own_pages]
        at += own_pages
    return table.cuda(), perm[at:].contiguous().cuda()


def prepare(case, seed):
    g = _gen(seed)
    cached, new = _lengths(case)
    op = case["op"]
    if op == "prompt":
        dt, hq, hkv, d = DTYPES[case["dtype"]], case["Hq"], case["Hkv"], case["D"]
        lk = [a + b for a, b in zip(cached, new)]
        tq, tk = sum(new), sum(lk)
        if case["fused"]:  # views of one projection's output
            qkv = _rows(g, tq, hq + 2 * hkv, d, dt)
            q, k, v = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
        else:
            q, k, v = _rows(g, tq, hq, d, dt), _rows(g, tk, hkv, d, dt), _rows(g, tk, hkv, d, dt)
        cu_q = _ints([sum(new[:i]) for i in range(len(new) + 1)])
        cu_k = _ints([sum(lk[:i]) for i in range(len(lk) + 1)])
        return {"op": op, "q": q, "k": k, "v": v, "cu_q": cu_q, "cu_k": cu_k}
    page = case["page"]
    if op == "decode":
        dt, hq, hkv, d = DTYPES[case["dtype"]], case["Hq"], case["Hkv"], case["D"]
        width = _ceil(max(cached), page)
        counts = [_ceil(n, page) for n in cached]
        shared = case["prefix"] // page
        pages = shared + sum(max(0, n - shared) for n in counts) + 8
        table, _ = _table(g, counts, width, pages, shared)
        return {"op": op, "q": _rows(g, case["B"], hq, d, dt), "k": _random_pages(g, pages, page, hkv, d),
                "v": _random_pages(g, pages, page, hkv, d), "table": table, "lens": _ints(cached),
                "prefix": case["prefix"], "max_len": max(cached)}
    counts = [_ceil(n, page) for n in cached]
    need = [_ceil(a + b, page) for a, b in zip(cached, new)]
    shared = case.get("prefix", 0) // page
    width = max(1, max(need)) + 1
    pages = shared + sum(n - shared for n in need) + 16
    if op == "plan":
        table, free = _table(g, counts, width, pages, shared)
        return {"op": op, "cached": _ints(cached), "new": _ints(new), "table": table, "free": free, "page": page,
                "T": sum(new)}
    table, _ = _table(g, need, width, pages)
    dt, hkv, d = DTYPES[case["dtype"]], case["Hkv"], case["D"]
    slots, lens = [], [a + b for a, b in zip(cached, new)]
    host = table.cpu()
    for b in range(case["B"]):
        pos = torch.arange(cached[b], lens[b])
        slots.append(host[b, pos // page].long() * page + pos % page)
    return {"op": op, "k": _rows(g, sum(new), hkv, d, dt), "v": _rows(g, sum(new), hkv, d, dt),
            "slots": torch.cat(slots).cuda(), "kc": _random_pages(g, pages, page, hkv, d),
            "vc": _random_pages(g, pages, page, hkv, d), "table": table,
            "cu": _ints([sum(lens[:i]) for i in range(len(lens) + 1)]), "rows": sum(lens)}


# ---------------------------------------------------------------- one pass
def _kq():
    at = os.path.join(os.getcwd(), "k-search_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    import kq

    return kq


def run(state):
    if own:
        return _run_own(state)
    return {"plan": _plain_plan, "pages": _plain_pages, "prompt": _plain_prompt, "decode": _plain_decode}[state["op"]](state)


def _run_own(s):
    kq = _kq()
    if s["op"] == "plan":
        p = kq.page_plan(s["cached"], s["new"], s["table"], s["free"], s["page"], s["T"])
        return {"slots": p.slots, "seq_lens": p.seq_lens, "cu_new": p.cu_new, "cu_seqlens": p.cu_seqlens,
                "counts": p.counts, "table": s["table"]}
    if s["op"] == "pages":
        kq.page_write(s["k"], s["v"], s["slots"], s["kc"], s["vc"])
        k, v = kq.page_read(s["kc"], s["vc"], s["table"], s["cu"], s["rows"], dtype=s["k"].dtype)
        return {"k": k, "v": v}
    if s["op"] == "prompt":
        return kq.flash_prompt_ragged(s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"])
    return kq.flash_decode_paged(s["q"], s["k"], s["v"], s["table"], s["lens"], prefix_len=s["prefix"],
                                 max_seqlen=s["max_len"])


def _cumulative(lens):
    return torch.cat([lens.new_zeros(1), lens.cumsum(0, dtype=torch.int32)])


def _plain_plan(s):
    cached, new, table, free, page = s["cached"], s["new"], s["table"], s["free"], s["page"]
    width = table.shape[1]
    lens = cached + new
    have = ((cached + page - 1) // page).clamp(max=width)
    need = ((lens + page - 1) // page).clamp(max=width)
    take = need - have
    start = take.cumsum(0) - take
    col = torch.arange(width, device="cuda")
    fresh = (col >= have[:, None]) & (col < need[:, None])
    index = start[:, None] + col - have[:, None]
    pages = torch.where(index < free.numel(), free[index.clamp(0, max(0, free.numel() - 1))], -1)
    table.copy_(torch.where(fresh, pages, table))
    cu_new = _cumulative(new)
    tok = torch.arange(s["T"], device="cuda", dtype=torch.int32)
    row = torch.searchsorted(cu_new[1:], tok, right=True)
    pos = cached[row] + tok - cu_new[row]
    at = table[row, (pos // page).clamp(max=width - 1)].long()
    slots = torch.where((at >= 0) & (pos // page < width), at * page + pos % page, -1)
    counts = torch.stack([take.sum(), (slots < 0).sum()]).to(torch.int32)
    return {"slots": slots, "seq_lens": lens, "cu_new": cu_new, "cu_seqlens": _cumulative(lens), "counts": counts,
            "table": table}


def _dequantise(blocks):
    d = blocks[..., :2].contiguous().view(torch.float16).float()
    x = d * blocks[..., 2:].contiguous().view(torch.int8).float()
    return x.flatten(-2)


def _quantise(x):
    """fp16 or bf16 [T, H, D] -> q8_0 blocks [T, H, D/32, 34]."""
    x = x.float().unflatten(-1, (-1, QK))
    amax = x.abs().amax(-1, keepdim=True)
    d = torch.where(amax > 0, amax / torch.full_like(amax, 127.0), torch.ones_like(amax))
    q = (x / d).round().clamp(-128, 127).to(torch.int8)
    return torch.cat([d.to(torch.float16).view(torch.uint8), q.view(torch.uint8)], -1)


def _plain_pages(s):
    out = {}
    page = s["kc"].shape[1]
    tok = torch.arange(s["rows"], device="cuda", dtype=torch.int32)
    row = torch.searchsorted(s["cu"][1:], tok, right=True)
    pos = tok - s["cu"][row]
    slot = s["table"][row, pos // page].long() * page + pos % page
    for name, x, cache in (("k", s["k"], s["kc"]), ("v", s["v"], s["vc"])):
        flat = cache.flatten(0, 1)
        flat[s["slots"]] = _quantise(x)
        out[name] = _dequantise(flat[slot]).to(x.dtype)
    return out


def _softmax_product(scores, v):
    """softmax over the last axis times v; a row that is masked throughout gives zeros."""
    m = scores.amax(-1, keepdim=True).clamp(min=-3e38)
    p = scores.sub_(m).exp_()
    total = p.sum(-1, keepdim=True)
    return torch.where(total > 0, (p @ v) / total.clamp(min=1e-30), 0.0)


def _plain_prompt(s):
    q, k, v, cu_q, cu_k = s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"]
    (tq, hq, d), (tk, hkv, _) = q.shape, k.shape
    iq, ik = (torch.arange(n, device="cuda", dtype=torch.int32) for n in (tq, tk))
    bq, bk = torch.searchsorted(cu_q[1:], iq, right=True), torch.searchsorted(cu_k[1:], ik, right=True)
    last = iq - cu_q[bq] + (cu_k[bq + 1] - cu_k[bq]) - (cu_q[bq + 1] - cu_q[bq])  # each row's last key
    hidden = (bq[:, None] != bk) | (ik - cu_k[bk] > last[:, None])
    qs = (q.float() * (1 / math.sqrt(d))).view(tq, hkv, hq // hkv, d).permute(1, 2, 0, 3)
    scores = qs @ k.float().permute(1, 2, 0).unsqueeze(1)
    scores.masked_fill_(hidden, float("-inf"))
    out = _softmax_product(scores, v.float().transpose(0, 1).unsqueeze(1))
    return out.permute(2, 0, 1, 3).reshape(tq, hq, d).to(q.dtype)


def _plain_decode(s):
    q, table, lens, prefix = s["q"], s["table"], s["lens"], s["prefix"]
    b, hq, d = q.shape
    page, hkv = s["k"].shape[1], s["k"].shape[2]
    n = prefix // page
    qs = (q.float() * (1 / math.sqrt(d))).view(b, hkv, hq // hkv, d)
    shared, apart = table[0, :n].long(), table[:, n:].long().clamp(min=0)
    # the shared pages once for the whole batch, then each sequence's own pages
    kp, vp = (_dequantise(c[shared]).flatten(0, 1).transpose(0, 1) for c in (s["k"], s["v"]))
    ks, vs = (_dequantise(c[apart]).flatten(1, 2).transpose(1, 2) for c in (s["k"], s["v"]))
    sp = (qs.transpose(0, 1).flatten(1, 2) @ kp.transpose(1, 2)).unflatten(1, (b, -1)).transpose(0, 1)
    ss = qs @ ks.transpose(2, 3)
    tok = torch.arange(prefix + ss.shape[-1], device="cuda")
    scores = torch.cat([sp, ss], -1).masked_fill_((tok >= lens[:, None])[:, None, None], float("-inf"))
    m = scores.amax(-1, keepdim=True).clamp(min=-3e38)
    p = (scores - m).exp_()
    total = p.sum(-1, keepdim=True)
    o = (p[..., :prefix].transpose(0, 1).flatten(1, 2) @ vp).unflatten(1, (b, -1)).transpose(0, 1) + p[..., prefix:] @ vs
    return torch.where(total > 0, o / total.clamp(min=1e-30), 0.0).reshape(b, hq, d).to(q.dtype)


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    cached, new = _lengths(case)
    op = case["op"]
    if op == "plan":
        page = case["page"]
        fresh = sum(_ceil(a + b, page) - _ceil(a, page) for a, b in zip(cached, new))
        return {"bytes": 8 * len(new) + 8 * sum(new) + 8 * fresh + 12 * len(new) + 16, "flops": 0}
    if op == "pages":
        hd = case["Hkv"] * case["D"]
        t, rows = sum(new), sum(cached) + sum(new)
        row = hd // QK * BLOCK_BYTES
        return {"bytes": 2 * t * (2 * hd + row) + 8 * t + 2 * rows * 2 * hd + 2 * (rows - t) * row, "flops": 0}
    hq, hkv, d = case["Hq"], case["Hkv"], case["D"]
    if op == "prompt":
        tk = sum(cached) + sum(new)
        pairs = sum(n * c + n * (n + 1) // 2 for c, n in zip(cached, new))
        return {"bytes": 4 * sum(new) * hq * d + 4 * tk * hkv * d, "flops": 4 * hq * d * pairs}
    own_tokens = sum(max(0, n - case["prefix"]) for n in cached)
    row = 2 * hkv * (d // QK) * BLOCK_BYTES
    return {"bytes": row * (case["prefix"] + own_tokens) + 4 * case["B"] * hq * d, "flops": 4 * hq * d * sum(cached)}


# ---------------------------------------------------------------- the same in 64 bits
def _values64(blocks):
    d = blocks[..., 0:2].contiguous().view(torch.float16).double()
    return (blocks[..., 2:].contiguous().view(torch.int8).double() * d).reshape(*blocks.shape[:-2], -1)


def _attend64(q, k, v, first_len):
    """One KV head: q [R, D], k, v [L, D]; row r sees its first first_len[r] keys."""
    w = q.double() @ k.T / math.sqrt(q.shape[-1])
    seen = torch.arange(k.shape[0], device=q.device)[None, :] < first_len[:, None]
    w = torch.where(seen, w, torch.full_like(w, -math.inf))
    top = torch.where(seen.any(1), w.max(1).values, torch.zeros_like(w[:, 0]))
    e = torch.exp(w - top[:, None])
    z = e.sum(1, keepdim=True)
    return torch.where(z > 0, e @ v / torch.where(z > 0, z, 1.0), 0.0)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "plan":
        return None
    cached, new = _lengths(case)
    if op == "pages":
        page, out = case["page"], {}
        table = s["table"].cpu()
        for name, x, cache in (("k", s["k"], s["kc"]), ("v", s["v"], s["vc"])):
            x = x.double().reshape(x.shape[0], x.shape[1], -1, QK)
            amax = x.abs().amax(-1, keepdim=True)
            d = torch.where(amax > 0, amax / 127, torch.ones_like(amax))
            written = (torch.round(x / d) * d.to(torch.float16).double()).flatten(2)
            parts, at = [], 0
            for b in range(case["B"]):
                pages = table[b, :_ceil(cached[b], page)].long().cuda()
                parts.append(_values64(cache[pages]).flatten(0, 1)[:cached[b]])
                parts.append(written[at:at + new[b]].reshape(new[b], case["Hkv"], case["D"]))
                at += new[b]
            out[name] = torch.cat(parts)
        return out
    hq, hkv = case["Hq"], case["Hkv"]
    g = hq // hkv
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    if op == "prompt":
        aq = ak = 0
        for c, n in zip(cached, new):
            for h in range(hkv if n else 0):
                k, v = s["k"][ak:ak + c + n, h].double(), s["v"][ak:ak + c + n, h].double()
                for i in range(h * g, h * g + g):
                    out[aq:aq + n, i] = _attend64(s["q"][aq:aq + n, i], k, v, c + 1 + torch.arange(n, device="cuda"))
            aq, ak = aq + n, ak + c + n
        return out
    page, table = case["page"], s["table"].cpu()
    for b, n in enumerate(cached):
        if n == 0:
            continue
        pages = table[b, :_ceil(n, page)].long().cuda()
        k, v = (_values64(c[pages]).flatten(0, 1)[:n] for c in (s["k"], s["v"]))
        full = torch.full((g,), n, device="cuda")
        for h in range(hkv):
            out[b, h * g:h * g + g] = _attend64(s["q"][b, h * g:h * g + g], k[:, h], v[:, h], full)
    return out
