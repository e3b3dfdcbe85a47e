"""GPU parity of the paged-serving operators against plain 64-bit forms.

Tolerance of the attention outputs, per element, with u the type's unit
roundoff (2^-11 fp16, 2^-8 bf16), ref the exact value and A = sum_j p_j |v_j|
/ sum_j p_j: the output's rounding gives u |ref|; the weights p_j are rounded
to the type before the product with V (u A) and the block scale folded into
them may round once more (u A); the scores and exponentials in fp32 give
relative errors of p of a few 2^-24 (D + |s|) each, bounded by 2e-5 (4 + |s|max)
for the sizes here. Nothing else is rounded to fewer than 32 bits.
"""
import math
import random

import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


# ---------------------------------------------------------------- helpers
def rows(g, t, h, d, dtype, scale=1.0):
    return (torch.randn((t, h, d), generator=g, device="cuda") * scale).to(dtype)


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def prefix_sums(lens):
    out = [0]
    for n in lens:
        out.append(out[-1] + n)
    return out


def random_cache(g, pages, ps, hkv, d):
    nb = d // 32
    c = torch.empty((pages, ps, hkv, nb, 34), dtype=torch.uint8, device="cuda")
    scale = (0.005 + 0.03 * torch.rand((pages, ps, hkv, nb, 1), generator=g, device="cuda")).to(torch.float16)
    c[..., :2] = scale.view(torch.uint8)
    c[..., 2:] = torch.randint(-127, 128, (pages, ps, hkv, nb, 32), generator=g, device="cuda").to(torch.int8).view(torch.uint8)
    return c


def values(blocks):
    """q8_0 blocks [..., H, NB, 34] -> float64 [..., H, D]."""
    d = blocks[..., :2].contiguous().view(torch.float16).double()
    return (d * blocks[..., 2:].contiguous().view(torch.int8).double()).flatten(-2)


def attend(q, k, v, seen, scale):
    """q [R, D], k, v [L, D] float64, seen bool [R, L] -> (out, A, largest |s|)."""
    s = q @ k.T * scale
    s = s.masked_fill(~seen, -math.inf)
    m = s.amax(1, keepdim=True) if s.shape[1] else s.new_full((s.shape[0], 1), -math.inf)
    m = torch.where(torch.isfinite(m), m, 0.0)
    p = torch.exp(s - m)
    l = p.sum(1, keepdim=True)
    l = torch.where(l > 0, l, 1.0)
    top = s.masked_fill(~seen, 0.0).abs().max().item() if s.numel() else 0.0
    return p @ v / l, p @ v.abs() / l, top


def check_out(got, ref, spread, top, dtype, what=""):
    u = U[dtype]
    tol = u * ref.abs() + 2 * u * spread + 2e-5 * (4 + top) * spread + (2.0 ** -24 if dtype == torch.float16 else 0)
    err = (got.double() - ref).abs()
    bad = err > tol
    assert torch.isfinite(got).all(), f"{what}: not finite"
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((err / tol.clamp(min=1e-30)).max()):.2f} x bound"


# ---------------------------------------------------------------- page_plan
def plan_ref(cached, new, table, free, ps, total):
    W = len(table[0]) if table else 0
    table = [list(r) for r in table]
    used, slots, dropped = 0, [], 0
    for b in range(len(cached)):
        c, n = max(0, cached[b]), max(0, new[b])
        have, need = min(-(-c // ps), W), min(-(-(c + n) // ps), W)
        for col in range(have, need):
            table[b][col] = free[used] if used < len(free) else -1
            used += 1
        for i in range(n):
            col = (c + i) // ps
            page = table[b][col] if col < W else -1
            slots.append(page * ps + (c + i) % ps if page >= 0 else -1)
    placed = sum(s >= 0 for s in slots[:total])
    dropped = len(slots) - placed
    slots = (slots + [-1] * total)[:total]
    return table, slots, used, dropped


PLANS = [
    # B, cached top, new top, page, width, free, total - sum(new)
    (1, 0, 1, 16, 4, 10, 0), (1, 17, 1, 16, 4, 10, 0), (3, 40, 0, 16, 5, 0, 0), (7, 50, 30, 1, 100, 500, 0),
    (8, 500, 1, 16, 40, 100, 0), (33, 100, 90, 7, 64, 2000, 13), (64, 300, 200, 32, 20, 100, 0),
    (600, 30, 20, 16, 4, 4000, 0), (1500, 9, 5, 4, 4, 900, -100), (5, 2000, 9000, 16, 700, 5000, 0),
    (2, 60, 60, 16, 3, 50, 0), (4, 10, 10, 16, 0, 5, 0),
]


@pytest.mark.parametrize("B,ctop,ntop,ps,W,F,extra", PLANS)
def test_page_plan(cuda, B, ctop, ntop, ps, W, F, extra):
    import kq
    rng = random.Random(B * 131 + ps)
    cached = [rng.randint(0, ctop) for _ in range(B)]
    new = [rng.randint(0, ntop) for _ in range(B)]
    if B > 3:
        cached[1], new[2], new[3] = 0, 0, -5
        cached[3] = -2
    table = [[rng.randrange(1000) for _ in range(W)] for _ in range(B)]
    if B > 4 and W > 1:  # a partly filled page that has no entry
        cached[4] = ps + ps // 2
        table[4][1] = -1
        new[4] = max(new[4], 1)
    free = rng.sample(range(1000, 20000), F)
    total = max(0, sum(max(0, n) for n in new) + extra)
    tt = ints(table).reshape(B, W)
    for out in (None, "again"):
        plan = kq.page_plan(ints(cached), ints(new), tt, ints(free), ps, total, out=None if out is None else plan)  # noqa: F821
        rt, rs, used, dropped = plan_ref(cached, new, table, free, ps, total)
        assert tt.tolist() == rt
        assert plan.slots.tolist() == rs
        c, n = [max(0, x) for x in cached], [max(0, x) for x in new]
        assert plan.seq_lens.tolist() == [x + y for x, y in zip(c, n)]
        assert plan.cu_new.tolist() == prefix_sums(n)
        assert plan.cu_seqlens.tolist() == prefix_sums([x + y for x, y in zip(c, n)])
        assert plan.counts.tolist() == [used, dropped]


def test_page_plan_no_requests(cuda):
    import kq
    e = ints([])
    plan = kq.page_plan(e, e, torch.empty((0, 4), dtype=torch.int32, device=cuda), e, 16, 3)
    assert plan.slots.tolist() == [-1] * 3 and plan.cu_new.tolist() == [0] and plan.counts.tolist() == [0, 0]


# ---------------------------------------------------------------- page_write, page_read
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T,H,D,ps", [(1, 1, 32, 1), (5, 3, 96, 5), (77, 8, 128, 16), (300, 4, 64, 32), (9, 2, 256, 16),
                                      (33, 7, 160, 3)])
def test_page_write_read(cuda, dtype, T, H, D, ps):
    import kq
    g = gen(T + D)
    pages = -(-T // ps) + 3
    fused = rows(g, T, 3 * H, D, dtype, 2.0)
    k, v = fused[:, H:2 * H], fused[:, 2 * H:]
    k[0, 0, :32] = 0                         # an all-zero block
    if T > 2:
        v[2, H - 1, 5] = 6e4                 # one large value sets its block's scale
    kc, vc = random_cache(g, pages, ps, H, D), random_cache(g, pages, ps, H, D)
    before = kc.clone(), vc.clone()
    perm = torch.randperm(pages, generator=g, device="cuda")
    pos = torch.arange(T, device="cuda")
    slots = perm[pos // ps] * ps + pos % ps
    skip = torch.zeros(T, dtype=torch.bool, device="cuda")
    if T > 4:
        skip[3], skip[4] = True, True
    given = slots.clone()
    given[skip] = -1
    if T > 4:
        given[4] = pages * ps                # past the cache: skipped, not written
    kq.page_write(k, v, given, kc, vc)
    for x, cache, old in ((k, kc, before[0]), (v, vc, before[1])):
        want = kq.quantize_rows(x.float().reshape(T * H, D).contiguous(), "q8_0").view(T, H, D // 32, 34)
        ref = old.flatten(0, 1).clone()
        ref[slots[~skip]] = want[~skip]
        assert torch.equal(cache.flatten(0, 1), ref)
    # read two sequences back, the second through an invalid page in the middle
    na = T // 3
    lens = [na, T - na]
    width = -(-T // ps) + 1
    table = torch.full((2, width), -1, dtype=torch.int32, device="cuda")
    npg = -(-T // ps)
    table[:, :npg] = perm[:npg].to(torch.int32)
    bad = None
    if lens[1] > ps:
        bad = 1
        table[1, 1] = pages + 7
    rk, rv = kq.page_read(kc, vc, table, ints(prefix_sums(lens)), T + 2, dtype=dtype)
    for got, cache in ((rk, kc), (rv, vc)):
        flat = values(cache.flatten(0, 1))
        pos = torch.cat([torch.arange(n, device="cuda") for n in lens])
        ref = flat[perm[pos // ps] * ps + pos % ps]
        if bad is not None:
            hit = (pos // ps == bad) & (torch.arange(T, device="cuda") >= na)
            ref[hit] = 0
        assert torch.equal(got[:T], ref.float().to(dtype))
        assert not got[T:].any()


def test_page_offsets_past_32_bits(cuda):
    """A cache of more than 2^32 bytes: its last rows are written, read and attended to."""
    import kq
    H, D, ps = 8, 128, 64
    pages = (1 << 32) // (ps * H * 136) + 2
    kc = torch.zeros((pages, ps, H, 4, 34), dtype=torch.uint8, device=cuda)
    vc = torch.zeros_like(kc)
    g = gen(1)
    k, v, q = rows(g, ps, H, D, torch.float16), rows(g, ps, H, D, torch.float16), rows(g, 1, 16, D, torch.float16)
    slots = torch.arange((pages - 1) * ps, pages * ps, device=cuda)
    kq.page_write(k, v, slots, kc, vc)
    table = ints([[pages - 1]])
    rk, rv = kq.page_read(kc, vc, table, ints([0, ps]), ps)
    assert (rk.float() - k.float()).abs().max() < 0.03 and (rv.float() - v.float()).abs().max() < 0.03
    for prefix in (0, ps):
        out = kq.flash_decode_paged(q, kc, vc, table, ints([ps]), prefix_len=prefix)
        for h in range(16):
            ref, spread, top = attend(q[0, h:h + 1].double(), values(kc[-1])[:, h // 2], values(vc[-1])[:, h // 2],
                                      torch.ones((1, ps), dtype=torch.bool, device=cuda), D ** -0.5)
            check_out(out[0, h:h + 1], ref, spread, top, torch.float16, f"head {h} prefix {prefix}")
    # two sequences in the same page, whose shared tokens go through the prefix's pass
    out = kq.flash_decode_paged(q.repeat(2, 1, 1), kc, vc, table.repeat(2, 1), ints([ps, ps]), prefix_len=ps - 3)
    for h in range(16):
        ref, spread, top = attend(q[0, h:h + 1].double(), values(kc[-1])[:, h // 2], values(vc[-1])[:, h // 2],
                                  torch.ones((1, ps), dtype=torch.bool, device=cuda), D ** -0.5)
        for b in range(2):
            check_out(out[b, h:h + 1], ref, spread, top, torch.float16, f"sequence {b} head {h}")


# ---------------------------------------------------------------- prompt attention
def prompt_ref(q, k, v, lq, lk, causal, scale):
    out, spread, top = torch.zeros(q.shape, dtype=torch.float64, device="cuda"), torch.zeros(q.shape, dtype=torch.float64, device="cuda"), 0.0
    g = q.shape[1] // k.shape[1]
    aq = ak = 0
    for n, m in zip(lq, lk):
        i, j = torch.arange(n, device="cuda")[:, None], torch.arange(m, device="cuda")[None, :]
        seen = j <= i + (m - n) if causal else torch.ones((n, m), dtype=torch.bool, device="cuda")
        for h in range(q.shape[1] if n else 0):
            o, a, t = attend(q[aq:aq + n, h].double(), k[ak:ak + m, h // g].double(), v[ak:ak + m, h // g].double(), seen, scale)
            out[aq:aq + n, h], spread[aq:aq + n, h], top = o, a, max(top, t)
        aq, ak = aq + n, ak + m
    return out, spread, top


PROMPTS = [
    # lens q, lens k (None: the same), Hq, Hkv, D
    ([1], None, 1, 1, 64), ([1], None, 32, 8, 128), ([1, 1, 1], None, 4, 4, 128), ([2, 0, 5], None, 8, 2, 64),
    ([127], None, 4, 1, 128), ([128], None, 4, 1, 128), ([129], None, 4, 1, 128), ([257], None, 2, 2, 128),
    ([300, 0, 1, 77, 512], None, 28, 4, 128), ([33, 95, 64], None, 15, 5, 128), ([700], None, 3, 1, 96),
    ([40, 200], None, 6, 2, 80), ([50, 60], None, 2, 1, 256), ([31, 70], None, 4, 2, 8), ([1000], None, 16, 2, 64),
    # chunks that follow a context, single tokens against long ones, keys fewer than rows
    ([64], [1000], 32, 8, 128), ([1, 1, 1], [777, 1, 128], 32, 8, 128), ([16, 3], [2048, 515], 28, 4, 128),
    ([100, 50, 20], [40, 0, 300], 8, 2, 128), ([5], [3], 1, 1, 128), ([200], [4000], 8, 1, 64),
    ([60, 0, 9], [0, 200, 9], 4, 2, 64), ([1], [9000], 16, 2, 128), ([130], [131], 64, 1, 128), ([3], [40], 127, 1, 64),
    ([20], [300], 130, 1, 64),
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lq,lk,Hq,Hkv,D", PROMPTS)
def test_prompt(cuda, dtype, lq, lk, Hq, Hkv, D):
    import kq
    lk = lk or lq
    g = gen(sum(lq) + Hq)
    q, k, v = rows(g, sum(lq), Hq, D, dtype, 1.5), rows(g, sum(lk), Hkv, D, dtype), rows(g, sum(lk), Hkv, D, dtype)
    for causal in (True, False):
        got = kq.flash_prompt_ragged(q, k, v, ints(prefix_sums(lq)), ints(prefix_sums(lk)), causal=causal)
        ref, spread, top = prompt_ref(q, k, v, lq, lk, causal, D ** -0.5)
        check_out(got, ref, spread, top, dtype, f"causal={causal}")


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("offset", [0, 1, 8])
def test_prompt_strided_views(cuda, D, offset):
    """q, k, v as views of one projection, at aligned and unaligned places; heads before tokens."""
    import kq
    g = gen(offset)
    lens, Hq, Hkv = [70, 130], 8, 2
    T, width = sum(lens), (Hq + 2 * Hkv) * D
    flat = torch.randn(T * (width + 16) + 16, generator=g, device="cuda").to(torch.float16)
    buf = flat[offset:offset + T * (width + 16)].view(T, width + 16)[:, :width].unflatten(1, (-1, D))
    q, k, v = buf[:, :Hq], buf[:, Hq:Hq + Hkv], buf[:, Hq + Hkv:]
    cu = ints(prefix_sums(lens))
    ref, spread, top = prompt_ref(q, k, v, lens, lens, True, 0.2)
    check_out(kq.flash_prompt_ragged(q, k, v, cu, scale=0.2), ref, spread, top, torch.float16)
    kt = k.transpose(0, 1).contiguous().transpose(0, 1)  # [Hkv, T, D] in memory
    check_out(kq.flash_prompt_ragged(q.contiguous(), kt, v, cu, scale=0.2), ref, spread, top, torch.float16)


@pytest.mark.parametrize("case", ["growing", "huge", "equal", "one_key", "negative_scale"])
def test_prompt_score_ranges(cuda, case):
    """Scores whose running maximum rises at every key block, that are far apart, all equal, or all very negative."""
    import kq
    g = gen(3)
    T, Hq, Hkv, D, dtype = 600, 4, 2, 128, torch.float16
    q, k, v = rows(g, T, Hq, D, dtype), rows(g, T, Hkv, D, dtype), rows(g, T, Hkv, D, dtype)
    scale = D ** -0.5
    if case == "growing":
        q = q.abs()
        k = (k.abs() * torch.linspace(0.05, 2.0, T, device="cuda")[:, None, None]).to(dtype)
    elif case == "huge":
        q, k = (q.float() * 8).to(dtype), (k.float() * 8).to(dtype)
    elif case == "equal":
        q = torch.zeros_like(q)
    elif case == "one_key":
        k[300] = 30.0 * q[450, :2]
    else:
        scale = -0.3
    cu = ints([0, T])
    ref, spread, top = prompt_ref(q, k, v, [T], [T], True, scale)
    check_out(kq.flash_prompt_ragged(q, k, v, cu, scale=scale), ref, spread, top, dtype, case)


def test_prompt_rows_outside_are_not_read(cuda):
    """What lies behind a sequence's keys (another sequence's infinities and NaN) stays out of its rows."""
    import kq
    g = gen(5)
    lens, H, D = [100, 40, 60], 4, 128
    q, k, v = (rows(g, sum(lens), H, D, torch.float16) for _ in range(3))
    k[100:140], v[100:140] = float("nan"), float("inf")
    cu = ints(prefix_sums(lens))
    got = kq.flash_prompt_ragged(q, k, v, cu)
    keep = torch.cat([torch.arange(100), torch.arange(140, 200)]).cuda()
    ref, spread, top = prompt_ref(q[keep], k[keep], v[keep], [100, 60], [100, 60], True, D ** -0.5)
    check_out(got[keep], ref, spread, top, torch.float16)
    assert torch.isnan(got[100:140]).all()


# ---------------------------------------------------------------- paged decode
def paged_case(g, lens, prefix, ps, hkv, d, spare=3, one_table=False):
    """Random caches and tables whose first pages are shared. A page that the prefix fills only partly is
    shared too, so every sequence's tokens of that page are the shared ones."""
    shared = -(-prefix // ps)
    width = max(1, -(-max(lens) // ps), shared) + 1
    need = [max(0, -(-n // ps) - shared) for n in lens]
    pages = shared + sum(need) + spare
    perm = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(lens), width), -1, dtype=torch.int32, device="cuda")
    table[:, :shared] = perm[:shared]
    at = shared
    for b, n in enumerate(need):
        table[b, shared:shared + n] = perm[at:at + n]
        at += n
    return random_cache(g, pages, ps, hkv, d), random_cache(g, pages, ps, hkv, d), table


def decode_ref(q, kc, vc, table, lens, scale, prefix=0):
    B, Hq, D = q.shape
    ps, hkv = kc.shape[1], kc.shape[2]
    g = Hq // hkv
    out, spread, top = torch.zeros(q.shape, dtype=torch.float64, device="cuda"), torch.zeros(q.shape, dtype=torch.float64, device="cuda"), 0.0
    for b, n in enumerate(lens):
        if n == 0:
            continue
        pages = table[b, :-(-n // ps)].long()
        k, v = (values(c[pages]).flatten(0, 1)[:n] for c in (kc, vc))
        if prefix:
            first = table[0, :-(-prefix // ps)].long()
            k, v = (torch.cat([values(c[first]).flatten(0, 1)[:min(n, prefix)], x[prefix:]]) for c, x in ((kc, k), (vc, v)))
        seen = torch.ones((g, n), dtype=torch.bool, device="cuda")
        seen &= (pages >= 0).repeat_interleave(ps)[:n]
        for h in range(hkv):
            o, a, t = attend(q[b, h * g:(h + 1) * g].double(), k[:, h], v[:, h], seen, scale)
            out[b, h * g:(h + 1) * g], spread[b, h * g:(h + 1) * g], top = o, a, max(top, t)
    return out, spread, top


DECODES = [
    # lens, prefix, page, Hq, Hkv, D
    ([1], 0, 16, 32, 8, 128), ([0], 0, 16, 8, 8, 128), ([3000], 0, 16, 32, 8, 128), ([17, 0, 33, 1], 0, 16, 28, 4, 128),
    ([5, 6, 7], 0, 3, 15, 5, 96), ([100, 200], 0, 64, 16, 1, 64), ([60, 80, 100], 0, 16, 8, 2, 256),
    ([40, 1], 0, 16, 4, 4, 32), ([129, 257, 64], 0, 32, 6, 2, 160), ([300, 5], 0, 16, 40, 1, 128),
    ([50] * 70, 0, 16, 32, 32, 128),
    # shared prefixes: whole pages, pages partly shared, sequences that end inside or before it
    ([64, 65, 100], 64, 16, 32, 8, 128), ([300, 128, 200, 129], 128, 32, 28, 4, 128), ([1000] * 5, 1000, 16, 32, 8, 128),
    ([90, 40, 0, 200], 80, 16, 8, 2, 64), ([500, 30, 700, 600, 480], 475, 16, 15, 5, 96), ([65] * 3, 64, 64, 8, 1, 128),
    ([260 + 3 * i for i in range(40)], 256, 16, 32, 8, 128), ([2100, 2048, 2300], 2048, 128, 4, 4, 128),
    ([130, 140], 128, 16, 8, 2, 256), ([150] * 33, 96, 16, 28, 4, 64), ([200, 210], 128, 16, 128, 1, 128),
    ([35] * 300, 32, 16, 4, 2, 32), ([515, 700], 512, 16, 48, 2, 128),
    # prefixes that many sequences share, or that end within 8 tokens: a pass of their own
    ([640 + 3 * i for i in range(40)], 640, 16, 32, 8, 128), ([330] * 299 + [7], 320, 16, 4, 2, 32),
    ([2048 + 40 * i for i in range(14)], 2048, 128, 28, 4, 64), ([1030] * 100 + [500, 0], 1024, 32, 8, 1, 96),
    ([700 + i for i in range(30)], 699, 24, 15, 5, 64), ([129, 200], 127, 16, 4, 4, 32),
    # rows for every number of warps that merge a row, odd counts among them
    ([90 + i for i in range(53)], 0, 16, 15, 5, 64), ([200] * 111, 0, 16, 15, 3, 128), ([70 + i for i in range(127)], 48, 16, 21, 7, 160),
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lens,prefix,ps,Hq,Hkv,D", DECODES)
def test_decode(cuda, dtype, lens, prefix, ps, Hq, Hkv, D):
    import kq
    g = gen(sum(lens) + prefix)
    kc, vc, table = paged_case(g, lens, prefix, ps, Hkv, D)
    q = rows(g, len(lens), Hq, D, dtype)
    ref, spread, top = decode_ref(q, kc, vc, table, lens, D ** -0.5)
    for bound in (None, max(lens)):
        got = kq.flash_decode_paged(q, kc, vc, table, ints(lens), prefix_len=prefix, max_seqlen=bound)
        check_out(got, ref, spread, top, dtype, f"max_seqlen={bound}")


@pytest.mark.parametrize("D,ps", [(128, 16), (64, 8), (256, 16), (96, 24), (32, 5)])
@pytest.mark.parametrize("prefix", [40, 43, 200])
def test_decode_copied_last_page(cuda, D, ps, prefix):
    """A prefix that ends inside a page: every sequence holds its own copy of that page, and only the
    first sequence's copy has the prefix's tokens (the others' are NaN there)."""
    import kq
    g = gen(prefix + D)
    lens = [prefix + n for n in (30, 7, 100, 1, 55)]
    kc, vc, table = paged_case(g, lens, prefix - prefix % ps, ps, 2, D)
    nan = torch.tensor([float("nan")], dtype=torch.float16, device=cuda).view(torch.uint8)
    for b in range(1, len(lens)):
        for c in (kc, vc):
            c[table[b, prefix // ps].item(), :prefix % ps, ..., :2] = nan
    q = rows(g, len(lens), 8, D, torch.float16)
    ref, spread, top = decode_ref(q, kc, vc, table, lens, D ** -0.5, prefix)
    check_out(kq.flash_decode_paged(q, kc, vc, table, ints(lens), prefix_len=prefix), ref, spread, top, torch.float16)


@pytest.mark.parametrize("prefix", [0, 128, 131])
@pytest.mark.parametrize("case", ["growing", "huge", "equal", "scales"])
def test_decode_score_ranges(cuda, prefix, case):
    import kq
    g = gen(7)
    lens, ps, Hq, Hkv, D = [900, 300, 640], 16, 8, 2, 128
    kc, vc, table = paged_case(g, lens, prefix, ps, Hkv, D)
    q = rows(g, 3, Hq, D, torch.float16)
    scale = D ** -0.5
    if case == "growing":   # the maximum rises along the sequence
        q = q.abs()
        kc[..., 2:] &= 127
        for b, n in enumerate(lens):
            for j in range(-(-n // ps)):
                kc[table[b, j].item(), ..., :2] = torch.tensor([0.0005 * (j + 1)], dtype=torch.float16, device=cuda).view(torch.uint8)
    elif case == "huge":
        q = (q.float() * 20).to(torch.float16)
    elif case == "equal":
        q = torch.zeros_like(q)
    else:                   # value scales from fp16's smallest numbers to large ones
        s = torch.tensor([6e-8, 1e-6, 3e-3, 500.0], dtype=torch.float16, device=cuda)
        vc[..., :2] = s[torch.randint(0, 4, vc.shape[:-1], generator=g, device="cuda")].unsqueeze(-1).view(torch.uint8)
    ref, spread, top = decode_ref(q, kc, vc, table, lens, scale)
    got = kq.flash_decode_paged(q, kc, vc, table, ints(lens), prefix_len=prefix)
    if case == "scales":    # outputs past fp16's range are infinite on both sides
        fits = ref.abs() < 6.5e4
        got, ref, spread = got[fits], ref[fits], spread[fits]
    check_out(got, ref, spread, top, torch.float16, case)


@pytest.mark.parametrize("scale", [-0.3, 0.0, 1.7])
@pytest.mark.parametrize("prefix", [0, 131])
def test_decode_scales(cuda, prefix, scale):
    import kq
    g = gen(17)
    lens = [400, 0, 140, 90]
    kc, vc, table = paged_case(g, lens, prefix, 16, 2, 128)
    q = rows(g, len(lens), 8, 128, torch.float16, 0.3)
    ref, spread, top = decode_ref(q, kc, vc, table, lens, scale)
    got = kq.flash_decode_paged(q, kc, vc, table, ints(lens), prefix_len=prefix, scale=scale)
    check_out(got, ref, spread, top, torch.float16)


@pytest.mark.parametrize("prefix", [64, 61])
def test_decode_hidden_pages(cuda, prefix):
    """A page id outside the cache hides its tokens, in the prefix and behind it."""
    import kq
    g = gen(11)
    lens, ps = [200, 170], 16
    kc, vc, table = paged_case(g, lens, prefix, ps, 2, 128)
    table[:, 1] = -1
    table[0, 7] = kc.shape[0] + 5
    q = rows(g, 2, 8, 128, torch.float16)
    got = kq.flash_decode_paged(q, kc, vc, table, ints(lens), prefix_len=prefix)
    seen = table.clone()
    seen[0, 7] = -1
    ref, spread, top = decode_ref(q, kc, vc, seen, lens, 128 ** -0.5)
    check_out(got, ref, spread, top, torch.float16)


@pytest.mark.parametrize("prefix", [64, 61])
def test_decode_unowned_cache_rows_do_not_matter(cuda, prefix):
    """NaN scales in rows behind a sequence's end, and in pages nobody owns, change nothing."""
    import kq
    g = gen(12)
    lens, ps = [100, 70, 0, 69], 16
    kc, vc, table = paged_case(g, lens, prefix, ps, 4, 128)
    q = rows(g, 4, 16, 128, torch.float16)
    ref, spread, top = decode_ref(q, kc, vc, table, lens, 128 ** -0.5)
    used = torch.zeros(kc.shape[:2], dtype=torch.bool, device=cuda)
    for b, n in enumerate(lens):
        for j in range(n):
            used[table[b, j // ps].item(), j % ps] = True
    nan = torch.tensor([float("nan")], dtype=torch.float16, device=cuda).view(torch.uint8)
    for c in (kc, vc):
        c[~used] = torch.cat([nan, torch.full((32,), 255, dtype=torch.uint8, device=cuda)])
    got = kq.flash_decode_paged(q, kc, vc, table, ints(lens), prefix_len=prefix)
    check_out(got, ref, spread, top, torch.float16)


def test_decode_max_seqlen_cuts(cuda):
    import kq
    g = gen(13)
    kc, vc, table = paged_case(g, [300, 90], 32, 16, 2, 128)
    q = rows(g, 2, 4, 128, torch.bfloat16)
    got = kq.flash_decode_paged(q, kc, vc, table, ints([300, 90]), prefix_len=32, max_seqlen=100)
    ref, spread, top = decode_ref(q, kc, vc, table, [100, 90], 128 ** -0.5)
    check_out(got, ref, spread, top, torch.bfloat16)


# ---------------------------------------------------------------- streams, graphs, one step together
def test_two_streams(cuda):
    """Calls on two streams at once: neither sees the other's scratch."""
    import kq
    g = gen(21)
    sets = []
    for i in range(2):
        lens = [700 + 100 * i, 300, 512]
        kc, vc, table = paged_case(g, lens, 256, 16, 8, 128)
        q = rows(g, 3, 32, 128, torch.float16)
        p = [rows(g, 40, 32, 128, torch.float16), rows(g, 3000, 8, 128, torch.float16), rows(g, 3000, 8, 128, torch.float16)]
        sets.append((q, kc, vc, table, ints(lens), p))

    def both(s):
        return [kq.flash_decode_paged(*s[:5], prefix_len=256), kq.flash_prompt_ragged(*s[5], ints([0, 40]), ints([0, 3000]))]

    alone = [both(s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(both(sets[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for outs in got[i]:
            for a, b in zip(outs, alone[i]):
                assert torch.equal(a, b)


def test_serving_step_in_a_graph(cuda):
    """Plan, write and decode captured once and replayed on new lengths."""
    import kq
    g = gen(22)
    B, ps, Hq, Hkv, D, prefix, W = 5, 16, 8, 2, 128, 32, 12
    kc, vc = random_cache(g, 80, ps, Hkv, D), random_cache(g, 80, ps, Hkv, D)
    table = torch.full((B, W), -1, dtype=torch.int32, device=cuda)
    table[:, :2] = ints([3, 4])
    cached, new, free = ints([32] * B), ints([1] * B), torch.arange(10, 70, dtype=torch.int32, device=cuda)
    k, v, q = rows(g, B, Hkv, D, torch.float16), rows(g, B, Hkv, D, torch.float16), rows(g, B, Hq, D, torch.float16)
    plan = kq.page_plan(cached, new, table, free, ps, B)
    out = torch.empty_like(q)

    def step():
        kq.page_plan(cached, new, table, free, ps, B, out=plan)
        kq.page_write(k, v, plan.slots, kc, vc)
        kq.flash_decode_paged(q, kc, vc, table, plan.seq_lens, prefix_len=prefix, out=out)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for t in range(20):  # positions 32 .. 51: a new page at 32 and at 48
        cached.fill_(32 + t)
        k.copy_(rows(g, B, Hkv, D, torch.float16))
        v.copy_(rows(g, B, Hkv, D, torch.float16))
        free.copy_(torch.roll(free, -B) if (32 + t) % ps == 0 and t else free)
        graph.replay()
        assert plan.counts.tolist() == [B if (32 + t) % ps == 0 else 0, 0]
        ref, spread, top = decode_ref(q, kc, vc, table, [33 + t] * B, D ** -0.5)
        check_out(out, ref, spread, top, torch.float16, f"token {t}")


def test_prompt_after_cached_chunk(cuda):
    """A prompt in two chunks through the cache: written, read back, attended to."""
    import kq
    g = gen(23)
    ps, Hq, Hkv, D, W = 16, 8, 2, 128, 40
    kc, vc = random_cache(g, 60, ps, Hkv, D), random_cache(g, 60, ps, Hkv, D)
    table = torch.full((2, W), -1, dtype=torch.int32, device=cuda)
    free = torch.randperm(60, generator=g, device="cuda").to(torch.int32)
    cached, at = ints([0, 0]), 0
    lens = [0, 0]
    for new in ([100, 37], [130, 60]):
        T = sum(new)
        q, k, v = rows(g, T, Hq, D, torch.float16), rows(g, T, Hkv, D, torch.float16), rows(g, T, Hkv, D, torch.float16)
        plan = kq.page_plan(cached, ints(new), table, free[at:].contiguous(), ps, T)
        at += plan.counts[0].item()
        lens = [a + b for a, b in zip(lens, new)]
        kq.page_write(k, v, plan.slots, kc, vc)
        ck, cv = kq.page_read(kc, vc, table, plan.cu_seqlens, sum(lens))
        got = kq.flash_prompt_ragged(q, ck, cv, plan.cu_new, plan.cu_seqlens)
        ref, spread, top = prompt_ref(q, ck, cv, new, lens, True, D ** -0.5)
        check_out(got, ref, spread, top, torch.float16)
        cached = plan.seq_lens.clone()


# ---------------------------------------------------------------- empty calls and refusals
def test_empty_calls(cuda):
    import kq
    e = ints([])
    q = torch.empty((0, 8, 128), dtype=torch.float16, device=cuda)
    k = torch.empty((0, 2, 128), dtype=torch.float16, device=cuda)
    assert kq.flash_prompt_ragged(q, k, k, ints([0])).shape == (0, 8, 128)
    assert kq.flash_prompt_ragged(q, k, k, ints([0, 0, 0])).shape == (0, 8, 128)
    kc = torch.zeros((2, 16, 2, 4, 34), dtype=torch.uint8, device=cuda)
    assert kq.flash_decode_paged(q, kc, kc.clone(), torch.empty((0, 3), dtype=torch.int32, device=cuda), e).shape == (0, 8, 128)
    kq.page_write(k, k, torch.empty(0, dtype=torch.int64, device=cuda), kc, kc.clone())
    a, b = kq.page_read(kc, kc, torch.zeros((1, 2), dtype=torch.int32, device=cuda), ints([0, 0]), 0)
    assert a.shape == (0, 2, 128) and b.shape == a.shape
    # rows without any key
    q1 = torch.randn((3, 4, 128), device=cuda).half()
    assert not kq.flash_prompt_ragged(q1, k, k, ints([0, 3]), ints([0, 0])).any()


def test_refusals(cuda):
    import kq
    h = torch.float16
    q, k = torch.zeros((4, 8, 128), dtype=h, device=cuda), torch.zeros((4, 2, 128), dtype=h, device=cuda)
    kc = torch.zeros((3, 16, 2, 4, 34), dtype=torch.uint8, device=cuda)
    cu, table, lens = ints([0, 4]), torch.zeros((4, 2), dtype=torch.int32, device=cuda), ints([1, 2, 3, 4])
    slots = torch.zeros(4, dtype=torch.int64, device=cuda)
    refused = [
        lambda: kq.flash_prompt_ragged(q.float(), k, k, cu),
        lambda: kq.flash_prompt_ragged(q.cpu(), k, k, cu),
        lambda: kq.flash_prompt_ragged(q, k.bfloat16(), k, cu),
        lambda: kq.flash_prompt_ragged(q, k, k[:, :1], cu),
        lambda: kq.flash_prompt_ragged(q, k[..., :64], k[..., :64], cu),
        lambda: kq.flash_prompt_ragged(q.transpose(1, 2), k, k, cu),
        lambda: kq.flash_prompt_ragged(q, k, k, cu.long()),
        lambda: kq.flash_prompt_ragged(q, k, k, cu, ints([0, 2, 4])),
        lambda: kq.flash_prompt_ragged(q, k[:3], k[:3], cu),
        lambda: kq.flash_prompt_ragged(q, k, k, cu, out=q.float()),
        lambda: kq.flash_decode_paged(q.transpose(0, 1), kc, kc, table, lens),
        lambda: kq.flash_decode_paged(q, kc[..., :33], kc[..., :33], table, lens),
        lambda: kq.flash_decode_paged(q, kc, kc[:2], table, lens),
        lambda: kq.flash_decode_paged(q[..., :64].contiguous(), kc, kc, table, lens),
        lambda: kq.flash_decode_paged(q, kc, kc, table[:3], lens),
        lambda: kq.flash_decode_paged(q, kc, kc, table.long(), lens),
        lambda: kq.flash_decode_paged(q, kc, kc, table, lens[:3]),
        lambda: kq.page_write(k, k[:3], slots, kc, kc),
        lambda: kq.page_write(k, k, slots.int(), kc, kc),
        lambda: kq.page_write(k.float(), k.float(), slots, kc, kc),
        lambda: kq.page_write(q, q, slots, kc, kc),
        lambda: kq.page_read(kc, kc, table, cu, 4),
        lambda: kq.page_read(kc, kc, table, ints([0] * 5), 4, dtype=torch.float32),
        lambda: kq.page_plan(lens, lens[:2], table, lens, 16, 4),
        lambda: kq.page_plan(lens.long(), lens, table, lens, 16, 4),
        lambda: kq.page_plan(lens, lens, table.t(), lens, 16, 4),
    ]
    for i, call in enumerate(refused):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was not refused")
    denied = [
        lambda: kq.flash_prompt_ragged(torch.zeros((4, 9, 128), dtype=h, device=cuda), k, k, cu),         # 9 heads over 2
        lambda: kq.flash_prompt_ragged(q[..., :12], k[..., :12], k[..., :12], cu),                       # D % 8
        lambda: kq.flash_decode_paged(torch.zeros((4, 9, 128), dtype=h, device=cuda), kc, kc, table, lens),
        lambda: kq.flash_decode_paged(q, kc, kc, table, lens, prefix_len=33),                            # past the table
        lambda: kq.flash_decode_paged(q, kc, kc, table, lens, prefix_len=-1),
        lambda: kq.page_plan(lens, lens, table, lens, 0, 4),
    ]
    for i, call in enumerate(denied):
        with pytest.raises(kq.KQError) as e:
            call()
        assert e.value.status == 1, i
    torch.cuda.synchronize()
    assert kq.device_error() == 0
