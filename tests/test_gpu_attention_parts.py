"""B200: sequences that are cut along the cache and joined again, where lengths and starts are not what they should be."""
import math

import pytest
import torch

from on_device_sd_b200 import _lib, paged_attention
from test_gpu_attention import BF16, F16, F32, Case, reference, tolerance

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("starts, served", [
    ([0, 1, -3, 2, 9], [0, 3]),             # two entries that fit nothing between two that do
    ([0, 4, 2, 2, 9], [0, 3]),              # one that runs backwards: its neighbours' rows 2 and 3 are computed for both
    ([0, 1, 1000, 3, 9], [0, 3]),
    ([3, 5, 9, 1 << 30, -(1 << 30)], [0, 1]),
])
@pytest.mark.parametrize("context", [700, 5000])
def test_starts_that_do_not_fit_leave_their_neighbours_alone(dtype, starts, served, context):
    """Spans that do not fit are skipped; every other sequence gets its output although it is cut and the starts are not sorted."""
    spans = [max(0, b - a) for a, b in zip(starts, starts[1:])]
    c = Case(dtype, 8, 2, 64, 16, [1] * 4, [context, context - 100, context // 2, context - 7], seed=60)
    g = torch.Generator("cuda").manual_seed(61)
    c.q = torch.randn(9, 8, 64, generator=g, device="cuda").to(dtype)
    out = torch.full_like(c.q, 5.0)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    lse_keep = paged_attention(c.q, c.kc, c.vc, c.tables, c.lens, query_start=torch.tensor(starts, dtype=torch.int32, device="cuda"), max_query_len=2,
                               out=out, return_lse=True, status=status)[1]
    assert status.item() == _lib.DEV_BAD_LENGTH
    claimed = torch.zeros(9, dtype=torch.int64)
    for b in served:
        claimed[starts[b]: starts[b + 1]] += 1
    for b in served:
        one = dict(spans=[spans[b]], contexts=[c.contexts[b]], starts=[starts[b]])
        want, wl, mean_abs, all_abs, err = reference(c.q, c.kc, c.vc, c.tables[b: b + 1], one["spans"], one["contexts"], one["starts"], c.scale)
        tol = tolerance(want, mean_abs, all_abs, err, c.contexts[b], dtype)
        for t in range(starts[b], starts[b + 1]):
            if claimed[t] == 1:
                assert ((out[t].double() - want[t]).abs() <= tol[t]).all(), (b, t)
                assert torch.isfinite(lse_keep[t]).all()
    assert (out[claimed == 0] == 5.0).all(), "rows of no sequence stay as they were"


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_rows_between_the_sequences_of_a_cut_call(dtype):
    """Rows before the first sequence, behind the last, and sequences without rows or keys among long ones."""
    spans, contexts = [0, 3, 0, 1, 6, 0, 2], [4000, 3000, 0, 0, 900, 50, 2]
    c = Case(dtype, 12, 2, 128, 24, spans, contexts, seed=62, extra_rows=5)
    out = torch.full_like(c.q, 5.0)
    _, lse = c.run(out=out, return_lse=True)
    c.check(out, lse)
    assert (out[c.starts[-1]:] == 5.0).all()


@pytest.mark.parametrize("batch, span, context, heads", [(128, 8, 700, (32, 4, 64)), (1000, 1, 300, (8, 8, 64)), (300, 1, 1500, (4, 1, 32)), (2, 1, 60000, (32, 8, 64)),
                                                         (40, 1, 3000, (4, 1, 64)), (33, 4, 900, (4, 2, 32)), (100, 1, 2000, (8, 1, 256))])
def test_cut_batches_of_all_sizes(batch, span, context, heads):
    """From far more units than CTAs to far fewer; the same call gives the same bits."""
    hq, hk, d = heads
    g = torch.Generator().manual_seed(batch)
    spans = [span if span == 1 else int(torch.randint(0, span + 1, (1,), generator=g)) for _ in range(batch)]
    contexts = [max(n, int(torch.randint(1, context, (1,), generator=g))) for n in spans]
    c = Case(BF16, hq, hk, d, 64, spans, contexts, seed=63)
    out, lse = c.run(return_lse=True)
    if batch * context <= 120000:
        c.check(out, lse)
    else:                                   # a part of the batch against the definition
        pick = list(range(0, batch, 16))
        want, wl, mean_abs, all_abs, err = reference(c.q, c.kc, c.vc, c.tables[pick], [spans[b] for b in pick], [contexts[b] for b in pick],
                                                     [c.starts[b] for b in pick], c.scale)
        tol = tolerance(want, mean_abs, all_abs, err, max(contexts), BF16)
        for b in pick:
            for t in range(c.starts[b], c.starts[b + 1]):
                assert ((out[t].double() - want[t]).abs() <= tol[t]).all()
    again, lse2 = c.run(return_lse=True)
    assert torch.equal(out, again) and torch.equal(lse, lse2)


def test_lengths_written_just_before_the_call():
    """Lengths and starts come from kernels of the same stream right in front of a cut call, again and again: the attention
    and the join both have to see the new ones."""
    c = Case(BF16, 32, 4, 64, 16, [2, 1, 3], [6000, 6000, 6000], seed=64)
    g = torch.Generator().manual_seed(65)
    plans = []
    for _ in range(12):
        n = [int(torch.randint(0, 4, (1,), generator=g)) for _ in range(3)]
        n[2] = min(n[2], 6 - n[0] - n[1]) if n[0] + n[1] <= 6 else 0
        starts = [0, n[0], n[0] + n[1], n[0] + n[1] + n[2]]
        plans.append((torch.tensor(starts, dtype=torch.int32, device="cuda"), torch.randint(700, 6001, (3,), generator=g).to(torch.int32).cuda(), starts))
    alone = []
    for s, l, _ in plans:
        c.qstart.copy_(s)
        c.lens.copy_(l)
        torch.cuda.synchronize()
        alone.append(c.run(out=torch.zeros_like(c.q), max_query_len=3))
        torch.cuda.synchronize()
    outs = [torch.zeros_like(c.q) for _ in plans]
    torch.cuda.synchronize()
    for _ in range(5):
        for (s, l, _), o in zip(plans, outs):
            c.qstart.copy_(s)
            c.lens.copy_(l)
            c.run(out=o, max_query_len=3)
    torch.cuda.synchronize()
    for (s, l, starts), o, a in zip(plans, outs, alone):
        assert torch.equal(o[: starts[-1]], a[: starts[-1]])
