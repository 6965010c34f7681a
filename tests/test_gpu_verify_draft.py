"""B200: verification of drafted tokens against the rule in 64 bits on the host."""
import math

import numpy as np
import pytest
import torch

from on_device_sd_b200 import _lib, verify_draft

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def rule(tokens, target, draft, accept, sample, starts, width):
    """Sequence by sequence in numpy's float64."""
    tokens, accept, sample = tokens.tolist(), accept.double().tolist(), sample.double().tolist()
    target = target.double().cpu().numpy()
    draft = None if draft is None else draft.double().cpu().numpy()
    out = np.full((len(sample), width + 1), -1, np.int64)
    taken = []
    for b, u in enumerate(sample):
        base, n = starts[b], starts[b + 1] - starts[b]
        j = 0
        while j < n:
            x = tokens[base + j]
            ok = 0 <= x < target.shape[1] and target[base + b + j, x] > accept[base + j] * (1.0 if draft is None else draft[base + j, x])
            if not ok:
                break
            out[b, j] = x
            j += 1
        p = target[base + b + j]
        r = p.copy()
        if j < n:
            if draft is not None:
                r = p - draft[base + j]
            elif 0 <= tokens[base + j] < len(r):
                r[tokens[base + j]] = 0
        r = np.where(r > 0, r, 0)
        if j < n and not r.sum() > 0:
            r = np.where(p > 0, p, 0)
        c = np.cumsum(r)
        if c[-1] > 0:
            past = np.nonzero(c > u * c[-1])[0]
            out[b, j] = past[0] if len(past) else np.nonzero(r > 0)[0][-1]
        taken.append(j)
    return torch.from_numpy(out), torch.tensor(taken, dtype=torch.int32)


def make(counts, vocab, dtype, sampled, seed, noise=0.7):
    g = torch.Generator("cuda").manual_seed(seed)
    total, batch = sum(counts), len(counts)
    logits = 2.5 * torch.randn(total + batch, vocab, generator=g, device="cuda")
    starts = [0]
    for n in counts:
        starts.append(starts[-1] + n)
    rows = torch.tensor([starts[b] + b + j for b, n in enumerate(counts) for j in range(n)], dtype=torch.int64, device="cuda")
    dl = logits[rows] + noise * torch.randn(total, vocab, generator=g, device="cuda")
    draft = torch.softmax(dl, -1)
    tokens = (draft.argmax(-1) if not sampled else torch.multinomial(draft, 1, generator=g).flatten()) if total else rows
    return dict(tokens=tokens, target=torch.softmax(logits, -1).to(dtype), draft=draft.to(dtype) if sampled else None,
                accept=torch.rand(total, generator=g, device="cuda"), sample=torch.rand(batch, generator=g, device="cuda"), starts=starts)


def run(c, width, **kw):
    return verify_draft(c["tokens"], c["target"], c["draft"], c["accept"], c["sample"],
                        draft_start=torch.tensor(c["starts"], dtype=torch.int32, device="cuda"), max_draft_len=width, **kw)


def check(c, width):
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out, n = run(c, width, status=status)
    want, wn = rule(c["tokens"], c["target"], c["draft"], c["accept"], c["sample"], c["starts"], width)
    assert torch.equal(n.cpu(), wn) and torch.equal(out.cpu(), want)
    assert status.item() == 0
    return out, n


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("sampled", [True, False])
@pytest.mark.parametrize("vocab", [1, 2, 7, 127, 128, 1000, 4099, 32000, 151936])
def test_matches_the_rule(dtype, sampled, vocab):
    counts = [4, 0, 1, 3, 5, 2, 0, 5, 5, 4, 1]
    check(make(counts, vocab, dtype, sampled, seed=vocab), 5)


@pytest.mark.parametrize("counts, width", [([0], 0), ([0, 0], 3), ([1], 1), ([40], 40), ([600], 700), ([3] * 200, 3)])
def test_spans_of_all_lengths(counts, width):
    c = make(counts, 777, F32, True, seed=5, noise=0.05)
    check(c, width)
    c["accept"].zero_()                                     # everything with a probability is accepted
    out, n = check(c, width)
    assert n.tolist() == counts


def test_numbers_at_their_ends():
    """u = 0 takes the first token with any weight, u next to 1 the last; equal distributions accept every draft."""
    c = make([3, 3, 3, 3], 5000, F32, True, seed=6)
    c["draft"] = c["target"][[0, 1, 2, 4, 5, 6, 8, 9, 10, 12, 13, 14]].clone()
    c["sample"].copy_(torch.tensor([0.0, 1 - 2.0 ** -24, 0.5, 0.0]))
    c["target"][3, :100] = 0.0                              # the row behind the first span starts with nothing
    c["target"][7, 4000:] = 0.0
    out, n = check(c, 3)
    assert n.tolist() == [3, 3, 3, 3] and out[0, 3] == 100 and out[1, 3] == 3999 and out[3, 3] == 0


def test_certain_and_impossible_drafts():
    vocab = 300
    target = torch.zeros(6, vocab, device="cuda")
    for r, x in enumerate((5, 6, 7, 8, 9, 10)):
        target[r, x] = 1.0
    tokens = torch.tensor([5, 6, 299, 9], device="cuda")    # the third drafted token has no probability at all
    c = dict(tokens=tokens, target=target, draft=None, accept=torch.zeros(4, device="cuda"), sample=torch.full((2,), 0.99, device="cuda"), starts=[0, 3, 4])
    out, n = check(c, 3)
    assert out.tolist() == [[5, 6, 7, -1], [9, 10, -1, -1]] and n.tolist() == [2, 1]


def test_nothing_left_of_the_difference_falls_back_to_the_target():
    vocab = 1000
    p = torch.softmax(torch.randn(2, vocab, device="cuda"), -1)
    q = p[:1] * 1.5                                          # larger everywhere (unnormalised): no remainder
    c = dict(tokens=torch.tensor([3], device="cuda"), target=p, draft=q, accept=torch.full((1,), 0.9, device="cuda"),
             sample=torch.tensor([0.37], device="cuda"), starts=[0, 1])
    out, n = check(c, 1)
    assert n.item() == 0 and out[0, 0] >= 0


def test_rows_with_gaps_and_views():
    """Row strides wider than the vocabulary, bases that are not 16-byte aligned."""
    for offset, pad in ((0, 8), (1, 5), (3, 0)):
        c = make([2, 4, 0, 3], 1003, F32, True, seed=8 + offset)
        for key in ("target", "draft"):
            rows, v = c[key].shape
            store = torch.full((rows * (v + pad) + offset,), 9.0, device="cuda")
            view = store[offset:].view(rows, v + pad)[:, :v]
            view.copy_(c[key])
            c[key] = view
        check(c, 4)


def test_16_bit_rows_of_odd_length():
    for dtype in (BF16, F16):
        check(make([5, 2, 0, 4], 32001, dtype, True, seed=9), 5)


def test_bad_tokens_probabilities_and_spans_are_reported():
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    c = make([2, 2, 1], 500, F32, True, seed=10)
    c["accept"].zero_()
    good, _ = run(c, 2)
    c["tokens"][1], c["tokens"][2] = 500, -1
    out, n = run(c, 2, status=status)
    assert status.item() == _lib.DEV_BAD_TOKEN and n.tolist() == [1, 0, 1] and torch.equal(out[2], good[2])
    want, wn = rule(c["tokens"], c["target"], c["draft"], c["accept"], c["sample"], c["starts"], 2)
    assert torch.equal(out.cpu(), want) and torch.equal(n.cpu(), wn)
    status.zero_()
    c = make([1, 1], 500, F32, False, seed=11)
    c["target"][0] = math.nan
    c["target"][2] = -1.0
    out, n = run(c, 1, status=status)
    assert status.item() == _lib.DEV_BAD_PROBS and out[0, 0] == -1 and n.tolist() == [0, 0]
    status.zero_()
    c = make([2, 2, 2], 500, F32, True, seed=12)
    ok, _ = run(c, 2)
    for starts in ([0, 2, 1, 3], [0, 2, 99, 4], [-1, 2, 4, 6]):
        c["starts"] = starts
        out, n = run(c, 2, status=status)
        assert status.item() & _lib.DEV_BAD_LENGTH
        status.zero_()
    c["starts"] = [0, 2, 4, 6]
    out, n = run(c, 1, status=status)                        # spans longer than announced
    assert (out == -1).all() and (n == 0).all() and status.item() == _lib.DEV_BAD_LENGTH


def test_infinite_probabilities_do_not_hang():
    c = make([1, 1, 0], 4000, F32, True, seed=13)
    c["target"][0, 17] = math.inf
    c["target"][4, :] = math.inf
    c["sample"][0] = math.nan
    out, n = run(c, 1)
    torch.cuda.synchronize()
    assert ((out >= -1) & (out < 4000)).all()


def test_refusals():
    c = make([2, 1], 100, F32, True, seed=14)
    with pytest.raises(TypeError):
        run(dict(c, tokens=c["tokens"].int()), 2)
    with pytest.raises(TypeError):
        run(dict(c, draft=c["draft"].half()), 2)
    with pytest.raises(ValueError):
        run(dict(c, draft=c["draft"][:1]), 2)
    with pytest.raises(ValueError):
        run(dict(c, accept=c["accept"][:1]), 2)
    with pytest.raises(ValueError):
        run(dict(c, starts=[0, 1]), 2)
    with pytest.raises(ValueError):
        run(c, -1)
    with pytest.raises(ValueError):
        run(dict(c, target=c["target"].t().contiguous().t()), 2)


def test_captured_and_replayed_with_new_numbers():
    c = make([4, 3, 0, 5], 9000, BF16, True, seed=15)
    starts = torch.tensor(c["starts"], dtype=torch.int32, device="cuda")
    gr = torch.cuda.CUDAGraph()
    run(c, 5)
    torch.cuda.synchronize()
    with torch.cuda.graph(gr):
        out, n = verify_draft(c["tokens"], c["target"], c["draft"], c["accept"], c["sample"], draft_start=starts, max_draft_len=5)
    for _ in range(5):
        c["accept"].uniform_()
        c["sample"].uniform_()
        gr.replay()
        torch.cuda.synchronize()
        want, wn = rule(c["tokens"], c["target"], c["draft"], c["accept"], c["sample"], c["starts"], 5)
        assert torch.equal(out.cpu(), want) and torch.equal(n.cpu(), wn)


def test_accepted_tokens_follow_the_target():
    """Rejection sampling keeps the target's distribution: first tokens of 200000 one-token spans over 6 tokens.  A count is
    binomial; 6 standard deviations."""
    B, vocab = 200000, 6
    g = torch.Generator("cuda").manual_seed(16)
    p = torch.tensor([0.05, 0.3, 0.1, 0.25, 0.1, 0.2], device="cuda")
    q = torch.tensor([0.3, 0.1, 0.2, 0.1, 0.25, 0.05], device="cuda")
    tokens = torch.multinomial(q, B, replacement=True, generator=g)
    out, _ = verify_draft(tokens, p.expand(2 * B, vocab).contiguous(), q.expand(B, vocab).contiguous(), torch.rand(B, generator=g, device="cuda"),
                          torch.rand(B, generator=g, device="cuda"), draft_start=torch.arange(B + 1, dtype=torch.int32, device="cuda"), max_draft_len=1)
    freq = torch.bincount(out[:, 0], minlength=vocab).double()
    assert ((freq - B * p.double()).abs() <= 6 * (B * p.double() * (1 - p.double())).sqrt()).all()
