"""B200: probabilities at both ends of the cache type's range."""
import math

import pytest
import torch

from on_device_sd_b200 import paged_attention
from test_gpu_attention import BF16, F16, F32, Case, half_step

pytestmark = pytest.mark.gpu


def far_tail_tolerance(want, keys, dtype):
    # p: half a step of its type; in fp16 also half of its smallest number, 2^-25, where the largest p is at least 2^8 (the
    # reference of the exponent lies that far below the maximum): 2^-33 for every key.  Sums in fp32: a key group adds up
    # a quarter of the keys, one after the other (a key, or the 16 of a stage, at a time), each time off by half a step of
    # the running sum, 2^-24; other groups and parts are joined in a few hundred steps; so (keys / 4 + 256) half steps
    # for the numerator and as many for the denominator.  Then the output's rounding, in fp16 at least 2^-25.
    f = (half_step(dtype) if dtype != F32 else 0.0) * want.abs() + 2 * (keys / 4 + 256) * 2.0 ** -24 * want.abs()
    f = f + (2.0 ** -33 * keys if dtype == F16 else 0.0)
    return f + half_step(dtype) * (want.abs() + f) + (2.0 ** -25 if dtype == F16 else 1e-30)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("bits", [4, 12, 16, 20, 24, 26, 28])
@pytest.mark.parametrize("sink_at", [0, 9000])
@pytest.mark.parametrize("rows, batch", [(1, 1), (4, 1), (1, 300), (4, 300)])
def test_many_improbable_keys_beside_one_that_takes_nearly_all(dtype, bits, sink_at, rows, batch):
    """One key (the first, as in models with an attention sink, or one in the middle) outweighs each other key by 2^bits; what the
    others add up to is still there.  rows: query heads a kv head, times a span of 5.  One sequence is cut into many parts;
    of 300 (which hold the same pages) most are not, so that many keys meet the sink in one part."""
    d, hk, n, span = 64, 1, 20001, 5
    kc = torch.zeros(-(-n // 64), 64, hk, d, dtype=dtype, device="cuda")
    vc = torch.zeros_like(kc)
    kc.view(-1, hk, d)[sink_at, 0, 0] = bits
    vc.view(-1, hk, d)[:n] = 1.0
    vc.view(-1, hk, d)[sink_at, 0, : d // 2] = 0.0                    # the tail alone, and the tail beside the sink
    q = torch.zeros(batch * span, rows, d, dtype=dtype, device="cuda")
    q[..., 0] = 16.0
    scale = math.log(2.0) / 16.0                                      # the sink's score is bits * ln 2, the others' 0
    tables = torch.arange(kc.shape[0], dtype=torch.int32, device="cuda").expand(batch, -1)
    lens = torch.full((batch,), n, dtype=torch.int32, device="cuda")
    out, lse = paged_attention(q, kc, vc, tables, lens, query_start=torch.arange(0, batch * span + 1, span, dtype=torch.int32, device="cuda"),
                               max_query_len=span, scale=scale, return_lse=True)
    out, lse = out.view(batch, span, rows, d), lse.view(batch, span, rows)
    for i in range(span):
        tail = (n - span + i) * 2.0 ** -bits
        want = torch.full((rows, d), tail / (1 + tail), dtype=torch.float64, device="cuda")
        want[:, d // 2:] = 1.0
        tol = far_tail_tolerance(want, float(n), dtype)
        err = (out[:, i].double() - want).abs().amax(0)
        assert (err <= tol).all(), (err / tol).max().item()
        total = bits * math.log(2.0) + math.log1p(tail)
        assert (lse[:, i].double() - total).abs().max().item() <= (n / 4 + 256) * 2.0 ** -24 + 2.0 ** -22 * total


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("per_stage", [0.5, 3.0, 7.9, 8.1, 15.9, 16.1, 40.0])
@pytest.mark.parametrize("falling", [False, True])
def test_scores_that_rise_along_the_cache(dtype, per_stage, falling):
    """The maximum grows by less and by more than the exponent's reference is allowed to lag, over a cut sequence."""
    d, n = 64, 2000
    c = Case(dtype, 4, 1, d, 16, [1, 3], [n, n - 300], seed=70)
    step = torch.arange(c.tables.shape[1] * 16, device="cuda").double() // 16 * per_stage * math.log(2.0)
    if falling:
        step = step.flip(0)
    step = torch.where(step > 60000, 60000.0, step)
    c.q[:] = 0
    c.q[..., 0] = 1.0
    for b in range(2):
        j = torch.arange(c.contexts[b], device="cuda")
        c.kc[c.tables[b].long()[j // 16], j % 16, 0, 0] = step[j].to(dtype)
    out, lse = c.run(return_lse=True, scale=1.0)
    c.check(out, lse, scale=1.0)


@pytest.mark.parametrize("heads", [(4, 1, 64), (8, 2, 128), (2, 2, 256), (4, 1, 32)])
def test_large_scores_and_values_in_fp16(heads):
    """Scores in the hundreds, and values next to the type's largest: p is as large as 2^15 while sums stay in range."""
    hq, hk, d = heads
    c = Case(F16, hq, hk, d, 16, [1, 2, 20], [300, 500, 900], seed=71)
    c.q.mul_(40)
    out, lse = c.run(return_lse=True)
    c.check(out, lse)
    c = Case(F16, hq, hk, d, 16, [1, 9], [777, 3000], seed=72)
    c.q.zero_()
    c.vc.clamp_(-1, 1).mul_(65000)
    out, lse = c.run(return_lse=True)
    c.check(out, lse)
