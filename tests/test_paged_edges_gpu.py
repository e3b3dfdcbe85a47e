"""Paged-serving operators where they can go wrong: lengths updated in place, padded free lists, scales and
scores at the ends of their ranges, infinities and NaN in masked places, prefix sums that run past the rows,
and the paths that only large batches take. Bounds as in test_paged_gpu, unless a test derives its own."""
import importlib.util
import math
import random
from pathlib import Path

import pytest
import torch

from test_paged_gpu import U, check_out, decode_ref, gen, ints, paged_case, plan_ref, prefix_sums, prompt_ref, rows

pytestmark = pytest.mark.gpu


def half_bytes(value):
    return torch.tensor([value], dtype=torch.float16, device="cuda").view(torch.uint8)


# ---------------------------------------------------------------- page_plan
@pytest.mark.parametrize("B,top,ps,W,extra", [(1, 60, 16, 40, 0), (8, 1, 16, 20, 0), (16, 400, 16, 250, 0), (3, 9000, 32, 2000, 5),
                                              (700, 12, 4, 40, 0), (1500, 3, 16, 8, -40)])
@pytest.mark.parametrize("which", ["cached", "new"])
def test_plan_updates_lengths_in_place(cuda, B, top, ps, W, extra, which):
    """A plan whose seq_lens are the next plan's cached (or new) lengths, reused as its output, step after step."""
    import kq
    rng = random.Random(B)
    lens = [rng.randint(0, top) for _ in range(B)]
    other = [rng.randint(0, top) for _ in range(B)]
    table, tt = [[-1] * W for _ in range(B)], ints([[-1] * W] * B)
    plan, free = None, list(range(7, 7 + B * W))
    for step in range(5):
        c, n = (lens, other) if which == "cached" else (other, lens)
        total = sum(n) + extra
        a = ints(lens) if plan is None else plan.seq_lens
        pair = (a, ints(other)) if which == "cached" else (ints(other), a)
        if plan is not None and plan.slots.numel() != total:
            plan = plan._replace(slots=torch.empty(total, dtype=torch.int64, device=cuda))
        plan = kq.page_plan(*pair, tt, ints(free), ps, total, out=plan)
        table, slots, used, dropped = plan_ref(c, n, table, free, ps, total)
        lens = [x + y for x, y in zip(c, n)]
        assert plan.seq_lens.tolist() == lens, step
        assert tt.tolist() == table and plan.slots.tolist() == slots, step
        assert plan.cu_new.tolist() == prefix_sums(n) and plan.cu_seqlens.tolist() == prefix_sums(lens), step
        assert plan.counts.tolist() == [used, dropped], step
        free = free[used:] + free[:used]
        other = [rng.randint(0, top) for _ in range(B)]
        if which == "new":  # the sums are the next step's new tokens: start over behind nothing
            other = [0] * B


@pytest.mark.parametrize("B,top,ps,W", [(1, 40, 16, 4), (7, 300, 16, 20), (40, 900, 32, 30), (600, 40, 16, 4)])
def test_plan_counts_tokens_of_absent_free_pages(cuda, B, top, ps, W):
    """A free list of fixed size whose unused entries are -1: the tokens of those pages count as not placed."""
    import kq
    rng = random.Random(B)
    cached, new = [rng.randint(0, top) for _ in range(B)], [rng.randint(0, top) for _ in range(B)]
    table = [[rng.randrange(1000) for _ in range(W)] for _ in range(B)]
    need = sum(max(0, min(-(-(c + n) // ps), W) - min(-(-c // ps), W)) for c, n in zip(cached, new))
    free = [1000 + i if rng.random() < 0.7 else -1 for i in range(need)] + [-1] * 5
    for total in (sum(new), sum(new) * 2 // 3, sum(new) + 9):
        tt = ints(table)
        plan = kq.page_plan(ints(cached), ints(new), tt, ints(free), ps, total)
        rt, rs, used, dropped = plan_ref(cached, new, table, free, ps, total)
        assert tt.tolist() == rt and plan.slots.tolist() == rs
        assert plan.counts.tolist() == [used, dropped]


# ---------------------------------------------------------------- decode: scales and scores
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("scale", [0.0, -0.0, 1e-38, -0.2])
@pytest.mark.parametrize("prefix", [0, 125, 128])
def test_decode_zero_queries(cuda, dtype, scale, prefix):
    """Zero and tiny query rows with a scale of 0 beside ordinary ones: hidden tokens stay hidden."""
    import kq
    g = gen(31)
    lens = [prefix + 60, 90, 0, prefix + 3]
    kc, vc, table = paged_case(g, lens, prefix, 16, 2, 128)
    q = rows(g, len(lens), 8, 128, dtype)
    q[:, ::3] = 0
    q[1:, 1] *= 2.0 ** -12
    if dtype == torch.bfloat16:
        q[0, 1] *= 2.0 ** -100
    ref, spread, top = decode_ref(q, kc, vc, table, lens, scale)
    check_out(kq.flash_decode_paged(q, kc, vc, table, ints(lens), prefix_len=prefix, scale=scale), ref, spread, top, dtype)


4
def check_decode(got, ref, spread, top, dtype, what=""):
    """Decode rounds a weight times its block scale to fp16 (and V's operand, of half the output's precision at
    most, once more), scores stay in fp32, the output is rounded to the type: u |ref| + 3 2^-11 A + the scores' part."""
    tol = U[dtype] * ref.abs() + 3 * 2.0 ** -11 * spread + 2e-5 * (4 + top) * spread + (2.0 ** -24 if dtype == torch.float16 else 0)
    err = (got.double() - ref).abs()
    assert torch.isfinite(got).all(), f"{what}: not finite"
    assert (err <= tol).all(), f"{what}: {int((err > tol).sum())} of {err.numel()} off, worst {float((err / tol.clamp(min=1e-30)).max()):.2f} x bound"


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("strength", [8.0, 16.0, 31.0])
@pytest.mark.parametrize("prefix", [0, 2045])
def test_decode_outlier_channel(cuda, dtype, strength, prefix):
    """One large channel of Q and K, as projections have it: scores of 30 to 120 that differ by little."""
    import kq
    g = gen(41)
    lens, ps, Hq, Hkv, D = [2100, 2300, 2045], 16, 8, 2, 128
    kc, vc, table = paged_case(g, lens, prefix, ps, Hkv, D)
    n = kc.shape[0] * ps
    k = torch.randn((n, Hkv, D), generator=g, device="cuda")
    k[..., 5] = 40.0 + 2.0 * torch.randn((n, Hkv), generator=g, device="cuda")
    kq.page_write(k.to(dtype), k.to(dtype), torch.arange(n, device="cuda"), kc, kc.clone())
    q = torch.randn((3, Hq, D), generator=g, device="cuda")
    q[..., 5] = strength
    q = q.to(dtype)
    ref, spread, top = decode_ref(q, kc, vc, table, lens, D ** -0.5)
    got = kq.flash_decode_paged(q, kc, vc, table, ints(lens), prefix_len=prefix)
    check_decode(got, ref, spread, top, dtype)


@pytest.mark.parametrize("prefix", [0, 128, 131])
@pytest.mark.parametrize("case", ["growing", "huge", "equal"])
def test_decode_score_ranges_bf16(cuda, prefix, case):
    import kq
    g = gen(43)
    lens, ps, Hq, Hkv, D = [900, 300, 640], 16, 8, 2, 128
    kc, vc, table = paged_case(g, lens, prefix, ps, Hkv, D)
    q = rows(g, 3, Hq, D, torch.bfloat16)
    if case == "growing":
        q = q.abs()
        kc[..., 2:] &= 127
        for b, n in enumerate(lens):
            for j in range(-(-n // ps)):
                kc[table[b, j].item(), ..., :2] = half_bytes(0.0005 * (j + 1))
    elif case == "huge":
        q = (q.float() * 20).to(torch.bfloat16)
    else:
        q = torch.zeros_like(q)
    ref, spread, top = decode_ref(q, kc, vc, table, lens, D ** -0.5)
    got = kq.flash_decode_paged(q, kc, vc, table, ints(lens), prefix_len=prefix)
    check_decode(got, ref, spread, top, torch.bfloat16, case)


5
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D,G,prefix", [(128, 4, 0), (128, 4, 61), (256, 2, 0), (96, 9, 0), (32, 16, 0)])
@pytest.mark.parametrize("d,gap", [(5e-4, 12.0), (2e-3, 11.0), (3e-2, 10.0), (1e-6, 3.0), (6e-8, 0.0), (1e-6, -1.0)])
def test_decode_small_value_scales(cuda, dtype, D, G, prefix, d, gap):
    """Small values behind one token that takes nearly all the weight and whose value is zero; the others share
    one score and one scale, so that a weight's rounding error would not average out. gap -1: random scores."""
    import kq
    g = gen(51)
    lens, ps, Hkv = [900, 333], 16, 2
    kc, vc, table = paged_case(g, lens, prefix, ps, Hkv, D)
    q = torch.ones((2, G * Hkv, D), dtype=dtype, device=cuda)
    vc[..., :2] = half_bytes(d)
    if gap >= 0:
        kc[..., 2:] = 0
        for b in range(2):
            first = kc[table[b, 0].item(), 0]
            first[..., 2:] = 100
            first[..., :2] = half_bytes(gap / (D ** 0.5 * 100))
            vc[table[b, 0].item(), 0, ..., 2:] = 0
    else:
        q = rows(g, 2, G * Hkv, D, dtype)
    ref, spread, top = decode_ref(q, kc, vc, table, lens, D ** -0.5)
    got = kq.flash_decode_paged(q, kc, vc, table, ints(lens), prefix_len=prefix)
    check_decode(got, ref, spread, top, dtype)


6
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("which", ["k", "v", "both"])
@pytest.mark.parametrize("prefix,D,Hkv,G", [(0, 128, 2, 4), (203, 128, 2, 4), (203, 64, 1, 15), (77, 96, 3, 1), (0, 256, 2, 9)])
def test_decode_large_scales(cuda, dtype, which, prefix, D, Hkv, G):
    """Block scales up to the largest fp16 number, among ordinary ones, whichever kernel reads them."""
    import kq
    g = gen(61)
    lens = [300, 210, 77, 500]
    kc, vc, table = paged_case(g, lens, prefix, 16, Hkv, D)
    scales = torch.tensor([0.01, 0.5, 600.0, 1500.0, 30000.0, 65504.0], dtype=torch.float16, device=cuda)
    for c, name in ((kc, "k"), (vc, "v")):
        if which in (name, "both"):
            pick = torch.randint(0, 6, c.shape[:-1], generator=g, device="cuda")
            pick[torch.rand(pick.shape, generator=g, device="cuda") < 0.7] = 0
            c[..., :2] = scales[pick].unsqueeze(-1).view(torch.uint8)
    big = 127 * 65504.0
    q = rows(g, len(lens), G * Hkv, D, dtype, 4.0 / big * D ** 0.5 if which != "v" else 1.0)
    # outputs that the type holds: fp16's reach up to 65504
    if dtype == torch.float16 and which != "k":
        vc[..., 2:] = torch.where(vc[..., 2:].view(torch.int8) > 0, 1, -1).to(torch.int8).view(torch.uint8)
    scale = D ** -0.5 if which == "v" else 1.0 / D
    if which != "v" and dtype == torch.float16:  # fp16 queries this small are subnormal: exact inputs all the same
        q = rows(g, len(lens), G * Hkv, D, dtype, 2.0 ** -18)
        scale = 2.0 ** -5
    ref, spread, top = decode_ref(q, kc, vc, table, lens, scale)
    got = kq.flash_decode_paged(q, kc, vc, table, ints(lens), prefix_len=prefix, scale=scale)
    if dtype == torch.float16:
        fits = ref.abs() < 6.5e4
        assert fits.any()
        got, ref, spread = got[fits], ref[fits], spread[fits]
    check_decode(got, ref, spread, top, dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("bad", [float("inf"), float("nan"), 60000.0])
@pytest.mark.parametrize("prefix", [200, 203])
def test_decode_hidden_prefix_tokens(cuda, dtype, bad, prefix):
    """Sequences that end inside the prefix do not see what its later tokens hold."""
    import kq
    g = gen(62)
    lens = [prefix + 50, 70, prefix, 1, 129, 0] + [100] * 40
    kc, vc, table = paged_case(g, lens, prefix, 16, 2, 128)
    q = rows(g, len(lens), 8, 128, dtype)
    ref, spread, top = decode_ref(q, kc, vc, table, lens, 128 ** -0.5)
    at = 150
    for c in (kc, vc):
        c[table[0, at // 16].item(), at % 16, :, 1, :2] = half_bytes(bad)
    got = kq.flash_decode_paged(q, kc, vc, table, ints(lens), prefix_len=prefix)
    short = [b for b, n in enumerate(lens) if n <= at]
    check_decode(got[short], ref[short], spread[short], top, dtype)


0
def test_decode_table_wider_than_32_bits(cuda):
    """A table whose pages could hold 2^32 tokens: the default bound on the lengths does not wrap."""
    import kq
    g = gen(91)
    ps, W = 1 << 15, 1 << 17
    kc, vc, _ = paged_case(g, [ps], 0, ps, 1, 32, spare=0)
    table = torch.zeros((1, W), dtype=torch.int32, device=cuda)
    q = rows(g, 1, 2, 32, torch.float16)
    ref, spread, top = decode_ref(q, kc, vc, table[:, :1], [1000], 32 ** -0.5)
    check_out(kq.flash_decode_paged(q, kc, vc, table, ints([1000])), ref, spread, top, torch.float16)


LARGE = [
    # lens, prefix, page, Hq, Hkv, D: more units than the 8-warp kernel is used for
    ([500 + 10 * i for i in range(64)], 0, 16, 32, 8, 128), ([260 + i for i in range(300)], 0, 32, 8, 4, 64),
    ([600 + i for i in range(64)], 0, 16, 24, 8, 96), ([600 + i for i in range(64)], 0, 24, 8, 8, 32),
    ([640 + i for i in range(64)], 0, 16, 16, 8, 160), ([640 + i for i in range(64)], 0, 16, 8, 8, 192),
    ([640 + i for i in range(64)], 0, 64, 16, 8, 224), ([640 + i for i in range(64)], 0, 16, 32, 8, 256),
    ([2500] * 40 + [2600 + i for i in range(24)], 0, 16, 32, 2, 128), ([1600 + i for i in range(72)], 0, 16, 40, 1, 64),
    ([1600] * 64 + [0, 1, 17], 0, 32, 45, 3, 96), ([2600 + i for i in range(64)], 0, 128, 18, 2, 32),
    ([2500 + i for i in range(64)], 0, 16, 32, 2, 256), ([2500 + i for i in range(64)], 0, 16, 24, 2, 160),
    ([1024 + 500 + 10 * i for i in range(48)] + [0, 900, 1024], 1024, 16, 32, 8, 128),
    ([515 + 1450 + i for i in range(70)], 515, 32, 45, 3, 96), ([256 + 640 + i for i in range(64)], 256, 16, 16, 8, 160),
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lens,prefix,ps,Hq,Hkv,D", LARGE)
def test_decode_large_batches(cuda, dtype, lens, prefix, ps, Hq, Hkv, D):
    """Enough to stream for the kernel with twelve warps, at every head size and with groups up to three sixteens."""
    import kq
    g = gen(sum(lens) + D)
    units = len(lens) * Hkv * (-(-(Hq // Hkv) // 16)) * ((max(lens) - prefix) // 16 + 1)
    assert units > 16 * 8 * torch.cuda.get_device_properties(0).multi_processor_count
    kc, vc, table = paged_case(g, lens, prefix, ps, Hkv, D)
    q = rows(g, len(lens), Hq, D, dtype)
    ref, spread, top = decode_ref(q, kc, vc, table, lens, D ** -0.5)
    check_out(kq.flash_decode_paged(q, kc, vc, table, ints(lens), prefix_len=prefix, max_seqlen=max(lens)), ref, spread, top, dtype)


# ---------------------------------------------------------------- prompts
7
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lq,lk,Hq,Hkv,D,at", [
    ([300], None, 4, 1, 128, (299, 130, 37)), ([300], None, 2, 2, 64, (255, 1)), ([1100], [1101], 2, 2, 128, (255, 700, 1100)),
    ([1100], [1101], 4, 2, 64, (511, 128)), ([70, 200, 33], None, 28, 4, 128, (69, 150, 302)),
    ([40], [3000], 8, 2, 128, (2999, 2970, 2961)), ([200], [4000], 8, 8, 128, (3999, 3850)), ([90], None, 6, 2, 80, (50, 89)),
    ([1500], None, 15, 5, 96, (1, 640, 1499)), ([64], None, 2, 1, 256, (40,)),
])
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_prompt_hidden_values(cuda, dtype, lq, lk, Hq, Hkv, D, at, bad):
    """An infinity or NaN in K or V reaches the rows that see its key, and no row before them."""
    import kq
    lk = lk or lq
    g = gen(71)
    q, k, v = rows(g, sum(lq), Hq, D, dtype), rows(g, sum(lk), Hkv, D, dtype), rows(g, sum(lk), Hkv, D, dtype)
    ref, spread, top = prompt_ref(q, k, v, lq, lk, True, D ** -0.5)
    cq, ck = prefix_sums(lq), prefix_sums(lk)
    for where in ("v", "k"):
        bk, bv = k.clone(), v.clone()
        hidden = torch.ones(sum(lq), dtype=torch.bool, device=cuda)
        for j in at:
            (bv if where == "v" else bk)[j, :, 3::7] = bad
            b = max(i for i in range(len(lk)) if ck[i] <= j)
            first = cq[b] + max(0, j - ck[b] - (lk[b] - lq[b]))  # the first row that sees the key
            hidden[first:cq[b + 1]] = False
        got = kq.flash_prompt_ragged(q, bk, bv, ints(cq), ints(ck))
        check_out(got[hidden], ref[hidden], spread[hidden], top, dtype, where)
        dims = got[~hidden][..., 3::7] if where == "v" else got[~hidden]
        if where == "v" or math.isnan(bad):
            assert not torch.isfinite(dims).any(), where
        if where == "v":
            rest = [d for d in range(D) if d % 7 != 3]
            check_out(got[~hidden][..., rest], ref[~hidden][..., rest], spread[~hidden][..., rest], top, dtype, "other dims")


8
@pytest.mark.parametrize("D,offset", [(128, 0), (64, 0), (256, 0), (128, 1)])
def test_prompt_prefix_sums_past_the_rows(cuda, D, offset):
    """Prefix sums outside the rows given are cut to them: nothing outside is read or written."""
    import kq
    g = gen(81)
    Tq, Tk, Hq, Hkv, dtype = 200, 200, 4, 2, torch.float16
    flat = torch.randn(Tk * Hkv * D + 8, generator=g, device="cuda").to(dtype)
    k = flat[offset:offset + Tk * Hkv * D].view(Tk, Hkv, D)
    q, v = rows(g, Tq, Hq, D, dtype), rows(g, Tk, Hkv, D, dtype)
    guarded = torch.full((3 * Tq, Hq, D), 7.0, dtype=dtype, device=cuda)
    out = guarded[Tq:2 * Tq]
    for causal in (True, False):
        # the last sequence claims more than there is
        got = kq.flash_prompt_ragged(q, k, v, ints([0, 90, 2 ** 31 - 1]), ints([0, 90, 2 ** 31 - 1]), causal=causal, out=out)
        ref, spread, top = prompt_ref(q, k, v, [90, 110], [90, 110], causal, D ** -0.5)
        check_out(got, ref, spread, top, dtype, f"causal={causal}")
        # a first entry above zero, and one below
        got = kq.flash_prompt_ragged(q, k, v, ints([60, 200]), ints([60, 200]), causal=causal, out=out)
        ref, spread, top = prompt_ref(q[60:], k[60:], v[60:], [140], [140], causal, D ** -0.5)
        check_out(got[60:], ref, spread, top, dtype, f"behind 60 rows, causal={causal}")
        kq.flash_prompt_ragged(q, k, v, ints([-500, 100, 200]), ints([-9, 100, 2 ** 30]), causal=causal, out=out)
    torch.cuda.synchronize()
    assert (guarded[:Tq] == 7).all() and (guarded[2 * Tq:] == 7).all() and kq.device_error() == 0


QUEUES = [
    # lens q, lens k, Hq, Hkv, D: several times the CTAs that fit at once, of one tile and of two
    ([1, 0, 400, 33, 900, 128, 1, 0, 700, 257, 64, 811, 1, 500, 90, 0, 640], None, 32, 8, 128),
    ([0, 300, 1, 1000, 129, 77, 0, 640, 31, 2, 900, 450], None, 28, 4, 128),
    ([700, 1, 0, 900, 600, 333, 800, 127], None, 32, 32, 64),
    ([1024, 1, 2000, 0, 3000, 1500], None, 32, 8, 128), ([2500, 0, 1, 1800, 1300], None, 28, 7, 64),
    ([900, 1, 0, 700, 1200], [2000, 500, 0, 700, 2900], 30, 10, 96),
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lq,lk,Hq,Hkv,D", QUEUES)
def test_prompt_queues(cuda, dtype, lq, lk, Hq, Hkv, D):
    """Many more jobs than CTAs fit at once: each takes several, empty and one-token sequences among them."""
    import kq
    lk = lk or lq
    tiles = 2 if sum(lk) // len(lk) >= 1024 else 1
    rows_per_cta = 128 // (Hq // Hkv) * tiles
    resident = torch.cuda.get_device_properties(0).multi_processor_count * (1 if tiles == 2 else 2)
    assert sum(-(-n // rows_per_cta) for n in lq) * Hkv > 1.9 * resident
    g = gen(sum(lq) + D)
    q, k, v = rows(g, sum(lq), Hq, D, dtype, 1.5), rows(g, sum(lk), Hkv, D, dtype), rows(g, sum(lk), Hkv, D, dtype)
    for causal in (True, False):
        ref, spread, top = prompt_ref(q, k, v, lq, lk, causal, D ** -0.5)
        for _ in range(3):  # which CTA takes which job differs from call to call
            got = kq.flash_prompt_ragged(q, k, v, ints(prefix_sums(lq)), ints(prefix_sums(lk)), causal=causal)
            check_out(got, ref, spread, top, dtype, f"causal={causal}")
    assert kq.device_error() == 0


@pytest.mark.parametrize("dtype,kw", [
    (torch.float16, dict(requests=7, system=320, prompt=90, Hq=16, Hkv=4, page_size=16)),
    (torch.bfloat16, dict(requests=40, system=1024, prompt=90, Hq=28, Hkv=4, page_size=32)),
])
def test_example_prompt_outputs(cuda, dtype, kw):
    """What the serving example's prompts and its system prompt return, against their definition."""
    import kq
    path = Path(__file__).resolve().parents[1] / "k-search_b200" / "examples" / "paged_serving.py"
    spec = importlib.util.spec_from_file_location("paged_serving", path)
    ex = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ex)
    D, E, ps, R = 128, 256, kw["page_size"], kw["requests"]
    g = gen(5)
    layer = ex.Layer(E, kw["Hq"], kw["Hkv"], D, dtype, cuda)
    new = [1 + kw["prompt"] * (b + 1) // R for b in range(R)]
    pages = kw["system"] // ps + sum(-(-n // ps) for n in new)
    server = ex.Server(layer, R, pages, ps, -(-(kw["system"] + max(new)) // ps), cuda)
    x = torch.randn((kw["system"], E), generator=g, device="cuda").to(dtype)
    got = server.system_prompt(x)
    ref, spread, top = prompt_ref(*layer.qkv(x), [kw["system"]], [kw["system"]], True, D ** -0.5)
    check_out(got, ref, spread, top, dtype, "system prompt")
    x = torch.randn((sum(new), E), generator=g, device="cuda").to(dtype)
    got = server.prompts(x, new)
    lens = [kw["system"] + n for n in new]
    keys, values = kq.page_read(server.k_cache, server.v_cache, server.tables, ints(prefix_sums(lens)), sum(lens), dtype)
    ref, spread, top = prompt_ref(layer.qkv(x)[0], keys, values, new, lens, True, D ** -0.5)
    check_out(got, ref, spread, top, dtype, "prompts")


@pytest.mark.parametrize("lq,lk,D", [([300, 70], None, 128), ([1200], None, 64), ([30], [2500], 128), ([40], None, 256)])
def test_prompt_in_place(cuda, lq, lk, D):
    """The output on the queries themselves: the same rows; next to a hidden NaN the true row or NaN, never another."""
    import kq
    lk = lk or lq
    g = gen(101)
    q, k, v = rows(g, sum(lq), 8, D, torch.float16), rows(g, sum(lk), 2, D, torch.float16), rows(g, sum(lk), 2, D, torch.float16)
    cq, ck = ints(prefix_sums(lq)), ints(prefix_sums(lk))
    ref, spread, top = prompt_ref(q, k, v, lq, lk, True, D ** -0.5)
    x = q.clone()
    check_out(kq.flash_prompt_ragged(x, k, v, cq, ck, out=x), ref, spread, top, torch.float16)
    v[lk[0] - 1, :, 5] = float("nan")
    x = q.clone()
    got = kq.flash_prompt_ragged(x, k, v, cq, ck, out=x)
    seen = torch.isfinite(got)
    assert not seen[lq[0] - 1, :, 5].any()
    check_out(got[seen], ref[seen], spread[seen], top, torch.float16)
