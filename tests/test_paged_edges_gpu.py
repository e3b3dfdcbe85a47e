"""Paged-serving operators where they can go wrong: lengths updated in place, padded free lists, scales and
scores at the ends of their ranges, infinities and NaN in masked places, prefix sums that run past the rows,
and the paths that only large batches take. Bounds as in test_paged_gpu, unless a test derives its own."""
import random

import pytest
import torch

from test_paged_gpu import ints, plan_ref, prefix_sums

pytestmark = pytest.mark.gpu


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
