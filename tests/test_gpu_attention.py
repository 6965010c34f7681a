"""B200: the paged cache write and the attention over the cache against their definitions in 64 bits."""
import math

import pytest
import torch

from on_device_sd_b200 import _lib, paged_attention, rope_store_kvcache, rotary_table, store_kvcache

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


# ---------------------------------------------------------------------------------------------------------
# the cache write
# ---------------------------------------------------------------------------------------------------------
def store_reference(x, w, pos, table, eps):
    """(z, bound on |z| before rounding) of the norm and the rotation in 64 bits."""
    x = x.double()
    d = x.shape[-1]
    y = x if w is None else x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * w.double()
    cos, sin = table[pos][:, None, : d // 2].double(), table[pos][:, None, d // 2:].double()
    a, b = y[..., : d // 2], y[..., d // 2:]
    z = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    size = torch.cat((a.abs() * cos.abs() + b.abs() * sin.abs(), b.abs() * cos.abs() + a.abs() * sin.abs()), -1)
    return z, size


def store_tolerance(z, size, d, dtype):
    # fp32: the sum of squares (d terms, halved by the root), eps, the root and two products for y; two products and a sum
    # for z: (d/2 + 6) half steps of 2^-24 on the sizes of the terms; then one rounding to the output type
    # (2^-25 is half of fp16's smallest number, the rounding error of its smallest values)
    f = (d / 2 + 6) * 2.0 ** -24 * size
    return f + half_step(dtype) * (z.abs() + f) + 2.0 ** -25


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("T, hq, hk, d, page, norm, idx", [
    (1, 32, 4, 128, 256, True, torch.int64), (5, 4, 2, 32, 16, False, torch.int32), (33, 8, 1, 64, 24, True, torch.int64),
    (130, 7, 7, 256, 1, True, torch.int32), (700, 32, 8, 128, 16, False, torch.int64), (1500, 5, 1, 64, 7, True, torch.int32),
])
def test_store_matches_definition(dtype, T, hq, hk, d, page, norm, idx):
    g = torch.Generator("cuda").manual_seed(T * 7 + d)
    blocks = T // page + 3
    qkv = torch.randn(T, (hq + 2 * hk) * d + 64, generator=g, device="cuda").to(dtype)     # rows wider than what is used
    q, k, v = (x.view(T, -1, d) for x in qkv[:, : (hq + 2 * hk) * d].split((hq * d, hk * d, hk * d), -1))
    kc = torch.randn(blocks, page, hk, d, generator=g, device="cuda").to(dtype)
    vc = torch.randn(blocks, page, hk, d, generator=g, device="cuda").to(dtype)
    k0, v0 = kc.clone(), vc.clone()
    slots = torch.randperm(blocks * page, generator=g, device="cuda")[:T].to(idx)
    if T > 3:
        slots[2] = -1
    limit = 60000
    pos = torch.randint(0, limit, (T,), generator=g, device="cuda").to(idx)
    pos[0] = limit - 1
    table = rotary_table(d, limit, device="cuda")
    wq = (1 + 0.2 * torch.randn(d, generator=g, device="cuda")).to(dtype) if norm else None
    wk = (1 + 0.2 * torch.randn(d, generator=g, device="cuda")).to(dtype) if norm else None
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = rope_store_kvcache(q, k, v, pos, table, kc, vc, slots, q_norm_weight=wq, k_norm_weight=wk, eps=1e-6, status=status)
    assert status.item() == 0
    z, size = store_reference(q, wq, pos.long(), table, 1e-6)
    assert ((out.double() - z).abs() <= store_tolerance(z, size, d, dtype)).all()
    zk, sk = store_reference(k, wk, pos.long(), table, 1e-6)
    used = slots >= 0
    where = slots[used].long()
    got = kc.view(-1, hk, d)[where].double()
    assert ((got - zk[used]).abs() <= store_tolerance(zk, sk, d, dtype)[used]).all()
    assert torch.equal(vc.view(-1, hk, d)[where], v[used])
    k0.view(-1, hk, d)[where] = kc.view(-1, hk, d)[where]
    v0.view(-1, hk, d)[where] = vc.view(-1, hk, d)[where]
    assert torch.equal(k0, kc) and torch.equal(v0, vc), "slots that no token names stay as they were"
    # in place, and keys and values alone
    again = qkv.clone()
    q2 = again[:, : hq * d].view(T, hq, d)
    kc2, vc2 = kc.clone(), vc.clone()
    assert rope_store_kvcache(q2, k, v, pos, table, kc2, vc2, slots, q_norm_weight=wq, k_norm_weight=wk, eps=1e-6, out=q2) is q2
    assert torch.equal(q2, out) and torch.equal(kc2, kc)
    store_kvcache(k, v, kc2, vc2, slots)
    assert torch.equal(kc2.view(-1, hk, d)[where], k[used]) and torch.equal(vc2, vc)


def test_store_wide_and_narrow_forms_agree():
    """Past a size the kernel takes four heads per lane group: the same rows give the same bits."""
    d, hq, hk, T = 128, 32, 4, 3000
    g = torch.Generator("cuda").manual_seed(3)
    qkv = torch.randn(T, (hq + 2 * hk) * d, generator=g, device="cuda").to(BF16)
    q, k, v = (x.view(T, -1, d) for x in qkv.split((hq * d, hk * d, hk * d), -1))
    w = torch.rand(d, generator=g, device="cuda").to(BF16)
    table = rotary_table(d, T, device="cuda")
    pos = slots = torch.arange(T, device="cuda")
    cache = [torch.zeros(T, 1, hk, d, dtype=BF16, device="cuda") for _ in range(4)]
    big = rope_store_kvcache(q, k, v, pos, table, cache[0], cache[1], slots, q_norm_weight=w, k_norm_weight=w)
    for i in range(0, T, 250):
        s = slice(i, i + 250)
        part = rope_store_kvcache(q[s], k[s], v[s], pos[s], table, cache[2], cache[3], slots[s], q_norm_weight=w, k_norm_weight=w)
        assert torch.equal(part, big[s])
    assert torch.equal(cache[0], cache[2]) and torch.equal(cache[1], cache[3])


def test_store_one_norm_only_and_strided_caches():
    d, hq, hk, T = 64, 4, 2, 9
    g = torch.Generator("cuda").manual_seed(4)
    q, k, v = (torch.randn(T, h, d, generator=g, device="cuda").to(F16) for h in (hq, hk, hk))
    w = torch.rand(d, generator=g, device="cuda").to(F16)
    table = rotary_table(d, 64, device="cuda")
    pos = torch.arange(T, device="cuda")
    # both caches in one tensor, heads before slots in memory
    both = torch.zeros(2, 5, hk, 8, d, dtype=F16, device="cuda")
    kc, vc = both[0].transpose(1, 2), both[1].transpose(1, 2)
    out = rope_store_kvcache(q, k, v, pos, table, kc, vc, pos + 11, q_norm_weight=w)
    z, size = store_reference(q, w, pos, table, 1e-6)
    assert ((out.double() - z).abs() <= store_tolerance(z, size, d, F16)).all()
    zk, sk = store_reference(k, None, pos, table, 1e-6)
    got = kc.reshape(-1, hk, d)[11: 11 + T].double()
    assert ((got - zk).abs() <= store_tolerance(zk, sk, d, F16)).all()
    assert torch.equal(vc.reshape(-1, hk, d)[11: 11 + T], v)


def test_store_reports_bad_slots_and_positions():
    d, hq, hk, T, page, blocks = 64, 4, 2, 6, 4, 2
    g = torch.Generator("cuda").manual_seed(5)
    q, k, v = (torch.randn(T, h, d, generator=g, device="cuda").to(BF16) for h in (hq, hk, hk))
    table = rotary_table(d, 10, device="cuda")
    kc = torch.full((blocks, page, hk, d), 7.0, dtype=BF16, device="cuda")
    vc = kc.clone()
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    pos = torch.tensor([0, 1, 10, -1, 4, 5], device="cuda")
    slots = torch.tensor([0, 8, 2, 3, -2, 5], device="cuda")
    out = rope_store_kvcache(q, k, v, pos, table, kc, vc, slots, status=status)
    assert status.item() == _lib.DEV_BAD_SLOT | _lib.DEV_BAD_POSITION
    assert (out[2] == 0).all() and (out[3] == 0).all() and (out[1] != 0).any()
    flat = kc.view(-1, hk, d)
    assert (flat[[1, 2, 3, 4, 6, 7]] == 7.0).all() and torch.equal(vc.view(-1, hk, d)[5], v[5])
    status.zero_()
    store_kvcache(k, v, kc, vc, torch.tensor([1 << 40, -1, -1, -1, -1, -1], device="cuda"), status=status)
    assert status.item() == _lib.DEV_BAD_SLOT


# ---------------------------------------------------------------------------------------------------------
# the attention
# ---------------------------------------------------------------------------------------------------------
def reference(q, kc, vc, tables, spans, contexts, starts, scale):
    """out, lse and, per element, sum_j w_j |v_j|, sum_j |v_j| and the rounding error of the scores in units of 2^-24 (64 bits)."""
    T, hq, d = q.shape
    page, hk = kc.shape[1:3]
    out = torch.zeros(T, hq, d, dtype=torch.float64, device=q.device)
    lse = torch.full((T, hq), -math.inf, dtype=torch.float64, device=q.device)
    mean_abs, all_abs, score_err = torch.zeros_like(out), torch.zeros_like(out), torch.zeros(T, hq, 1, dtype=torch.float64, device=q.device)
    for b, (n, c) in enumerate(zip(spans, contexts)):
        j = torch.arange(c, device=q.device)
        blk = tables[b].long()[j // page] if c else j
        for i in range(n):
            t, m = starts[b] + i, c - n + i + 1
            if m <= 0:
                continue
            for g in range(hk):
                h = slice(g * (hq // hk), (g + 1) * (hq // hk))
                kk, vv = kc[blk[:m], (j % page)[:m], g].double(), vc[blk[:m], (j % page)[:m], g].double()
                s = q[t, h].double() @ kk.T * scale
                lse[t, h] = torch.logsumexp(s, -1)
                w = torch.exp(s - lse[t, h][:, None])
                out[t, h] = w @ vv
                mean_abs[t, h] = w @ vv.abs()
                all_abs[t, h] = vv.abs().sum(0)
                score_err[t, h, 0] = ((q[t, h].double().abs() @ kk.abs().T * scale) * (d + 1) + 4 * s.abs()).amax(-1)
    return out, lse, mean_abs, all_abs, score_err


def tolerance(out, mean_abs, all_abs, score_err, keys, dtype):
    # p: rounded to the cache's type (half a step; in fp16 also half of its smallest number, against a largest p of 1), and
    # wrong by the score's error and the exponential's two units; sums over at most `keys` terms; the same again for l;
    # then the output's rounding
    e = 2.0 ** -24
    u = half_step(dtype) if dtype != F32 else 0.0
    p = u + 2 * score_err * e + 2 * (keys + 64) * e
    body = p * mean_abs + (2.0 ** -25 if dtype == F16 else 0.0) * all_abs
    # an fp16 output below its smallest normal number is off by 2^-25
    return body + half_step(dtype) * (out.abs() + body) + (2.0 ** -25 if dtype == F16 else 1e-30)


class Case:
    def __init__(self, dtype, hq, hk, d, page, spans, contexts, seed=0, extra_rows=0, poison=True):
        g = torch.Generator("cuda").manual_seed(seed)
        self.spans, self.contexts, self.dtype = spans, contexts, dtype
        need = [(c + page - 1) // page for c in contexts]
        blocks = sum(need) + 2
        fill = math.nan if poison else 0.0
        self.kc = torch.full((blocks, page, hk, d), fill, dtype=dtype, device="cuda")      # what no sequence holds is NaN
        self.vc = self.kc.clone()
        order = torch.randperm(blocks, generator=g, device="cuda").to(torch.int32)
        self.tables = torch.full((len(spans), max(need + [1]) + 1), blocks - 1, dtype=torch.int32, device="cuda")
        at = 0
        for b, (n, c) in enumerate(zip(need, contexts)):
            self.tables[b, :n] = order[at: at + n]
            at += n
            j = torch.arange(c, device="cuda")
            blk = self.tables[b].long()[j // page]
            self.kc[blk, j % page] = torch.randn(c, hk, d, generator=g, device="cuda").to(dtype)
            self.vc[blk, j % page] = torch.randn(c, hk, d, generator=g, device="cuda").to(dtype)
        self.starts = [0]
        for n in spans:
            self.starts.append(self.starts[-1] + n)
        T = self.starts[-1] + extra_rows
        wide = torch.randn(T, hq + 2 * hk, d, generator=g, device="cuda").to(dtype)
        self.q = wide[:, :hq]                                                               # rows of a fused projection
        self.lens = torch.tensor(contexts, dtype=torch.int32, device="cuda")
        self.qstart = torch.tensor(self.starts, dtype=torch.int32, device="cuda")
        self.scale = d ** -0.5

    def run(self, **kw):
        kw.setdefault("query_start", self.qstart)
        if kw["query_start"] is not None:
            kw.setdefault("max_query_len", max(self.spans + [0]))
        return paged_attention(self.q, self.kc, self.vc, self.tables, self.lens, **kw)

    def check(self, out, lse=None, scale=None):
        scale = scale or self.scale
        want, wl, mean_abs, all_abs, score_err = reference(self.q, self.kc, self.vc, self.tables, self.spans, self.contexts, self.starts, scale)
        n = self.starts[-1]
        tol = tolerance(want, mean_abs, all_abs, score_err, max(self.contexts + [1]), self.dtype)
        err = (out.double() - want).abs()
        assert (err[:n] <= tol[:n]).all(), (err[:n] / tol[:n]).max()
        if lse is not None:
            finite = torch.isfinite(wl[:n])
            assert torch.equal(torch.isfinite(lse[:n]), finite) and (lse[:n][~finite] == -math.inf).all()
            e = 2.0 ** -24 * (2 * score_err[:n, :, 0] + 2 * (max(self.contexts + [1]) + 64) + 4 * wl[:n].abs())
            assert ((lse[:n].double() - wl[:n]).abs()[finite] <= e[finite]).all()


HEADS = [(32, 4, 128), (16, 8, 64), (4, 2, 32), (8, 1, 256), (7, 7, 128), (12, 1, 64)]


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("hq, hk, d", HEADS)
@pytest.mark.parametrize("page", [1, 24, 256])
def test_attention_ragged_spans(dtype, hq, hk, d, page):
    spans = [1, 0, 5, 3, 1, 8, 2, 1, 4, 1]
    contexts = [1, 9, 5, 64, 65, 500, 1, 0, 130, 257]         # shorter than its span, empty, across tiles
    c = Case(dtype, hq, hk, d, page, spans, contexts, seed=d + page, extra_rows=3)
    out = torch.full_like(c.q, 3.0)
    got, lse = c.run(out=out, return_lse=True)
    assert got is out
    c.check(out, lse)
    assert (out[c.starts[-1]:] == 3.0).all(), "rows behind the last sequence stay as they were"


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("hq, hk, d, contexts", [
    (32, 4, 128, [33]), (32, 8, 128, [5000]), (8, 1, 256, [700, 1, 2000]), (4, 4, 64, [1, 15, 16, 17, 63, 64, 65, 255, 256, 257, 1000]), (32, 1, 32, [3001]),
])
def test_attention_single_tokens(dtype, hq, hk, d, contexts):
    c = Case(dtype, hq, hk, d, 16, [1] * len(contexts), contexts, seed=9)
    out, lse = c.run(query_start=None, return_lse=True)
    c.check(out, lse)
    # a table that is wider than the sequences, and one cut to them, hold the same pages
    same = paged_attention(c.q, c.kc, c.vc, c.tables[:, : (max(contexts) + 15) // 16], c.lens)
    c.check(same)
    assert torch.equal(c.run(query_start=None), out), "the same call gives the same bits"
    scaled = c.run(query_start=None, scale=0.3)
    c.check(scaled, scale=0.3)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_attention_many_sequences_and_long_spans(dtype):
    g = torch.Generator().manual_seed(1)
    spans = torch.randint(0, 4, (300,), generator=g).tolist()
    contexts = torch.randint(0, 150, (300,), generator=g).tolist()
    c = Case(dtype, 4, 2, 64, 16, spans, contexts, seed=11)
    out, lse = c.run(return_lse=True)
    c.check(out, lse)
    c = Case(dtype, 8, 1, 128, 32, [40, 1, 23], [300, 900, 23], seed=12)       # more rows than a tile holds
    for longest in (40, 1, 7, None):                                           # the hint only picks the tile
        out, lse = c.run(max_query_len=longest, return_lse=True)
        c.check(out, lse)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("heads", [(8, 2, 128), (8, 1, 64)])
def test_keys_a_row_does_not_see_do_not_reach_it(dtype, bad, heads):
    hq, hk, d = heads
    spans, contexts = [6, 3, 9], [100, 3, 640]
    c = Case(dtype, hq, hk, d, 16, spans, contexts, seed=13)
    clean = c.run().clone()
    for b, (n, ctx) in enumerate(zip(spans, contexts)):
        j = ctx - 2                                                            # the last two keys: seen by the last two rows
        for k in (j, j + 1):
            blk = c.tables[b, k // 16].long()
            c.vc[blk, k % 16] = bad
            c.kc[blk, k % 16] = bad
    out = c.run()
    for b, n in enumerate(spans):
        s = c.starts[b]
        a, w = out[s: s + n - 2].double(), clean[s: s + n - 2].double()
        assert torch.isfinite(a).all()
        # the other path adds keys one by one: fp32 sums of the same products, then one rounding
        assert ((a - w).abs() <= 2 * half_step(dtype) * w.abs() + 1e-4).all()
        assert not torch.isfinite(out[s + n - 1]).any(), "a row that sees them shows it"


def test_nan_queries_stay_in_their_rows():
    c = Case(BF16, 8, 2, 128, 16, [2, 1], [50, 400], seed=14)
    clean = c.run().clone()
    c.q[1, 3] = math.nan
    out = c.run()
    assert torch.isnan(out[1, 3]).all()
    keep = torch.ones(3, 8, dtype=torch.bool, device="cuda")
    keep[1, 3] = False
    assert torch.equal(out[keep], clean[keep])


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_large_scores_and_shared_maxima(dtype):
    """Scores in the hundreds (one key takes all) and all keys alike (the mean of the values)."""
    c = Case(dtype, 4, 1, 64, 16, [1, 2], [300, 500], seed=15)
    c.q.mul_(40)
    out, lse = c.run(return_lse=True)
    c.check(out, lse)
    c = Case(dtype, 4, 1, 64, 16, [1], [777], seed=16)
    c.q.zero_()
    out, lse = c.run(return_lse=True)
    c.check(out, lse)


def test_bad_pages_and_lengths_are_reported_and_not_followed():
    c = Case(BF16, 8, 2, 128, 16, [1, 1, 1, 1], [100, 100, 40, 20], seed=17)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    clean = c.run(status=status).clone()
    assert status.item() == 0
    c.tables[1, 3] = 1 << 30
    c.tables[1, 4] = -5
    out = c.run(status=status)
    assert status.item() == _lib.DEV_BAD_PAGE
    assert torch.equal(out[[0, 2, 3]], clean[[0, 2, 3]])
    status.zero_()
    c.lens[2], c.lens[3] = 1 << 29, -7
    c.tables[2] = c.tables[2, 0]
    out = c.run(status=status)
    assert status.item() & _lib.DEV_BAD_LENGTH and torch.equal(out[0], clean[0])
    assert (out[3] == 0).all()
    status.zero_()
    # spans that run past the rows, backwards, or start before them are skipped
    out = torch.full_like(c.q, 5.0)
    c.run(out=out, query_start=torch.tensor([0, 1, -3, 2, 9], dtype=torch.int32, device="cuda"), status=status)
    assert status.item() & _lib.DEV_BAD_LENGTH and torch.equal(out[0], clean[0]) and (out[3] == 5.0).all()


def test_no_pages_and_no_rows():
    c = Case(BF16, 8, 2, 128, 16, [1, 1], [0, 0], seed=18)
    out, lse = paged_attention(c.q, c.kc, c.vc, c.tables[:, :0], c.lens, return_lse=True)
    assert (out == 0).all() and (lse == -math.inf).all()
    empty = paged_attention(c.q[:0], c.kc, c.vc, c.tables[:0], c.lens[:0])
    assert empty.shape == (0, 8, 128)
    assert paged_attention(c.q[:0], c.kc, c.vc, c.tables, c.lens, query_start=torch.zeros(3, dtype=torch.int32, device="cuda")).shape[0] == 0


def test_refuses_what_does_not_fit():
    c = Case(BF16, 8, 2, 128, 16, [1, 1], [30, 40], seed=19)
    ok = (c.q, c.kc, c.vc, c.tables, c.lens)
    with pytest.raises(ValueError, match="one token per sequence"):
        paged_attention(c.q[:1], *ok[1:])
    with pytest.raises(TypeError):
        paged_attention(c.q.float(), *ok[1:])
    with pytest.raises(TypeError):
        paged_attention(*ok[:3], c.tables.long(), c.lens)
    with pytest.raises(ValueError):
        paged_attention(*ok, query_start=torch.zeros(2, dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError):
        paged_attention(c.q, c.kc, c.vc[:1], c.tables, c.lens)
    with pytest.raises(ValueError, match="no CPU path"):
        paged_attention(*ok[:4], c.lens.cpu())
    with pytest.raises(ValueError):
        paged_attention(*ok, status=torch.zeros(1, device="cuda"))
    with pytest.raises(_lib.B200MoEError, match="scale"):
        paged_attention(*ok, scale=0.0)
    shifted = torch.zeros(2 * 8 * 128 + 4, dtype=BF16, device="cuda")[4:].view(2, 8, 128)
    with pytest.raises(_lib.B200MoEError, match="aligned"):
        paged_attention(shifted, *ok[1:])
    with pytest.raises(_lib.B200MoEError, match="head_dim"):
        paged_attention(c.q[..., :96], c.kc[..., :96], c.vc[..., :96], c.tables, c.lens)
    with pytest.raises(ValueError, match="expanded"):
        paged_attention(*ok, out=torch.zeros(1, 8, 128, dtype=BF16, device="cuda").expand(2, 8, 128))
    kv = torch.zeros(2, 2, 128, dtype=BF16, device="cuda")
    flat = torch.zeros(1, 16, 2, 128, dtype=BF16, device="cuda").expand(3, 16, 2, 128)
    with pytest.raises(ValueError, match="expanded"):
        store_kvcache(kv, kv, flat, flat, torch.tensor([0, 40], device="cuda"))
    odd = torch.zeros(2, 7, 128, dtype=BF16, device="cuda")
    with pytest.raises(_lib.B200MoEError, match="multiple"):
        paged_attention(odd, *ok[1:])


def test_strided_caches_tables_and_outputs():
    """Caches that are halves of one tensor with heads in front of the slots, a table that is a view, an output with gaps."""
    c = Case(BF16, 8, 2, 64, 16, [1, 3, 2], [50, 300, 129], seed=20)
    want, wl = c.run(return_lse=True)
    blocks, page, hk, d = c.kc.shape
    both = torch.empty(blocks, 2, hk, page, d, dtype=BF16, device="cuda")
    both[:, 0].copy_(c.kc.transpose(1, 2))
    both[:, 1].copy_(c.vc.transpose(1, 2))
    table = torch.full((3, c.tables.shape[1] + 9), -1, dtype=torch.int32, device="cuda")
    table[:, 4: 4 + c.tables.shape[1]] = c.tables
    gaps = torch.full((6, 10, 64), 2.0, dtype=BF16, device="cuda")
    out, lse = paged_attention(c.q, both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2), table[:, 4: 4 + c.tables.shape[1]], c.lens,
                               query_start=c.qstart, max_query_len=3, out=gaps[:, 1:9], return_lse=True)
    assert torch.equal(out, want) and torch.equal(lse, wl)
    assert (gaps[:, 0] == 2.0).all() and (gaps[:, 9] == 2.0).all()


def test_offsets_past_32_bits():
    """A cache of more than 2^31 elements: the sequence's pages lie at both ends of it."""
    page, hk, d = 256, 8, 128
    blocks = (1 << 31) // (page * hk * d) + 40
    kc = torch.empty(blocks, page, hk, d, dtype=BF16, device="cuda")
    vc = torch.empty(blocks, page, hk, d, dtype=BF16, device="cuda")
    g = torch.Generator("cuda").manual_seed(21)
    pages = [blocks - 1, 0, blocks - 3, 5]
    ctx = 4 * page - 37
    c = Case(BF16, 32, hk, d, page, [2], [ctx], seed=21)
    for i, b in enumerate(pages):
        kc[b], vc[b] = (torch.randn(page, hk, d, generator=g, device="cuda").to(BF16) for _ in range(2))
    c.kc, c.vc = kc, vc
    c.tables = torch.tensor([pages], dtype=torch.int32, device="cuda")
    out, lse = c.run(return_lse=True)
    c.check(out, lse)
    slots = torch.tensor([(blocks - 1) * page + 9, 3], device="cuda")
    k, v = (torch.randn(2, hk, d, generator=g, device="cuda").to(BF16) for _ in range(2))
    store_kvcache(k, v, kc, vc, slots)
    assert torch.equal(kc[blocks - 1, 9], k[0]) and torch.equal(vc[0, 3], v[1])


def test_streams_and_graphs():
    """Two captured graphs and an eager call run side by side on three streams; each has its own workspace."""
    cases = [Case(BF16, 32, 4, 128, 256, [1] * 4, [4000, 100, 9000, 2000], seed=s) for s in (30, 31, 32)]
    want = [c.run(query_start=None).clone() for c in cases]
    graphs, outs = [], []
    for c in cases[:2]:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(c.run(query_start=None))
        graphs.append(gr)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    eager = []
    for _ in range(20):
        for s, gr in zip(streams, graphs):
            with torch.cuda.stream(s):
                gr.replay()
        with torch.cuda.stream(streams[2]):
            eager.append(cases[2].run(query_start=None))
    torch.cuda.synchronize()
    assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])
    assert all(torch.equal(e, want[2]) for e in eager)
    # a replay sees new lengths
    cases[0].lens.copy_(torch.tensor([17, 0, 8000, 1], dtype=torch.int32))
    graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], cases[0].run(query_start=None))


def test_store_then_attention_follow_each_other():
    """The cache write, then the attention that reads it, many times in one stream: each launch may start before its
    predecessor has drained, and has to see what that one wrote."""
    hq, hk, d, page = 32, 4, 128, 16
    g = torch.Generator("cuda").manual_seed(33)
    table = rotary_table(d, 4096, device="cuda")
    kc = torch.zeros(20, page, hk, d, dtype=BF16, device="cuda")
    vc = torch.zeros_like(kc)
    tables = torch.randperm(20, generator=g, device="cuda").to(torch.int32).view(1, 20)
    qkv = torch.randn(300, hq + 2 * hk, d, generator=g, device="cuda").to(BF16)
    outs = []
    for t in range(300):
        q, k, v = qkv[t: t + 1].split((hq, hk, hk), 1)
        slot = tables[0, t // page].long() * page + t % page
        pos = torch.full((1,), t, device="cuda")
        qr = rope_store_kvcache(q, k, v, pos, table, kc, vc, slot.view(1))
        outs.append(paged_attention(qr, kc, vc, tables, torch.full((1,), t + 1, dtype=torch.int32, device="cuda")))
    got = torch.cat(outs)
    kc2, vc2 = torch.zeros_like(kc), torch.zeros_like(vc)
    q, k, v = qkv.split((hq, hk, hk), 1)
    pos = torch.arange(300, device="cuda")
    slots = tables[0].long()[pos // page] * page + pos % page
    qr = rope_store_kvcache(q, k, v, pos, table, kc2, vc2, slots)
    assert torch.equal(kc, kc2) and torch.equal(vc, vc2)
    c = Case(BF16, hq, hk, d, page, [300], [300], seed=1)
    c.q, c.kc, c.vc, c.tables = qr, kc2, vc2, tables
    c.check(got)
    c.check(c.run())


def test_output_in_the_queries_place():
    """out may be the query tensor itself, cut along the cache or not."""
    for contexts in ([40, 3], [5000, 900]):
        c = Case(BF16, 32, 4, 128, 16, [5, 9], contexts, seed=40)
        want = c.run().clone()
        q = c.q
        assert c.run(out=q) is q and torch.equal(q, want)


def test_graph_pool_shared_by_two_graphs():
    """Two graphs captured into one memory pool and replayed one after the other, as an engine keeps one per batch size."""
    cases = [Case(BF16, 32, 4, 128, 256, [1] * n, [3000] * n, seed=41 + n) for n in (1, 4)]
    want = [c.run(query_start=None).clone() for c in cases]
    pool = torch.cuda.graph_pool_handle()
    graphs, outs = [], []
    for c in cases:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, pool=pool):
            outs.append(c.run(query_start=None))
        graphs.append(gr)
    for i in (0, 1, 1, 0, 1):
        graphs[i].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[i], want[i])


def test_strides_of_single_entries_do_not_matter():
    """One token, one kv head, one block: the stride of such a dimension may be any number."""
    c = Case(BF16, 4, 1, 64, 16, [1], [16], seed=50, poison=False)
    kc, vc = c.kc[c.tables[0, 0].long()][None].contiguous(), c.vc[c.tables[0, 0].long()][None].contiguous()
    q = c.q[:1].contiguous()
    table = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    want = paged_attention(q, kc, vc, table, c.lens)
    q2 = q.as_strided((1, 4, 64), (3, 64, 1))
    k2, v2 = kc.as_strided((1, 16, 1, 64), (5, 64, 7, 1)), vc.as_strided((1, 16, 1, 64), (1, 64, 9, 1))
    assert torch.equal(paged_attention(q2, k2, v2, table.as_strided((1, 1), (77, 55)), c.lens), want)
    before = kc.clone()
    store_kvcache(q[:, :1].as_strided((1, 1, 64), (1, 3, 1)), q[:, 1:2], k2, v2, torch.tensor([5], device="cuda"))
    assert torch.equal(kc[0, 5, 0], q[0, 0]) and torch.equal(vc[0, 5, 0], q[0, 1])
    kc[0, 5] = before[0, 5]
    assert torch.equal(kc, before)
