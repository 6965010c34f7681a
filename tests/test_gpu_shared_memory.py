"""B200: outputs that partly cover what the call reads are refused; views of one buffer that do not touch are not."""
import pytest
import torch

from on_device_sd_b200 import paged_attention, rope_store_kvcache, rotary_table, store_kvcache
from test_gpu_attention import BF16, F32, Case

pytestmark = pytest.mark.gpu


def test_attention_output_that_partly_covers_the_queries():
    c = Case(BF16, 8, 2, 64, 16, [3, 2], [700, 40], seed=80)
    buf = torch.zeros(9, 8, 64, dtype=BF16, device="cuda")
    q = buf[2:7]
    q.copy_(c.q)
    args = (c.kc, c.vc, c.tables, c.lens)
    kw = dict(query_start=c.qstart, max_query_len=3)
    want = paged_attention(q, *args, **kw)
    for out in (buf[1:6], buf[4:9], buf.view(-1)[2 * 512 + 64:][: 5 * 512].view(5, 8, 64), buf.view(-1, 4, 64).as_strided((5, 8, 64), (256, 64, 1), 1024)):
        with pytest.raises(ValueError, match="shares memory"):
            paged_attention(q, *args, out=out, **kw)
    with pytest.raises(ValueError, match="k_cache"):
        paged_attention(q, *args, out=c.kc.view(-1)[: 5 * 512].view(5, 8, 64), **kw)
    with pytest.raises(ValueError, match="v_cache"):
        paged_attention(q, *args, out=c.vc.view(-1)[512: 6 * 512].view(5, 8, 64), **kw)
    # beside the queries in the same rows, and the queries themselves
    wide = torch.zeros(5, 20, 64, dtype=BF16, device="cuda")
    wide[:, :8] = c.q
    assert torch.equal(paged_attention(wide[:, :8], *args, out=wide[:, 12:], **kw), want) and torch.equal(wide[:, :8], c.q)
    assert torch.equal(paged_attention(q, *args, out=buf[2:7], **kw), want)
    # one cache for keys and values is read twice, which harms nothing
    both = paged_attention(c.q, c.kc, c.kc, c.tables, c.lens, **kw)
    assert torch.equal(both, paged_attention(c.q, c.kc, c.kc.clone(), c.tables, c.lens, **kw))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_cache_write_into_its_own_inputs(dtype):
    T, hq, hk, d = 12, 8, 2, 64
    g = torch.Generator("cuda").manual_seed(81)
    qkv = torch.randn(T, hq + 2 * hk, d, generator=g, device="cuda").to(dtype)
    q, k, v = qkv.split((hq, hk, hk), 1)
    table, pos = rotary_table(d, T, device="cuda"), torch.arange(T, device="cuda")
    kc, vc = (torch.zeros(2, 8, hk, d, dtype=dtype, device="cuda") for _ in range(2))
    want = rope_store_kvcache(q, k, v, pos, table, kc, vc, pos)
    for out, name in ((qkv[:, 1: 1 + hq], "query"), (qkv[:, 4: 4 + hq], "query")):
        with pytest.raises(ValueError, match=name):
            rope_store_kvcache(q, k, v, pos, table, kc, vc, pos, out=out)
    other = torch.randn(T, hq, d, generator=g, device="cuda").to(dtype)
    with pytest.raises(ValueError, match="key"):
        rope_store_kvcache(q, other[:, :hk], v, pos, table, kc, vc, pos, out=other)
    with pytest.raises(ValueError, match="value"):
        rope_store_kvcache(q, k, other[:, hk: 2 * hk], pos, table, kc, vc, pos, out=other)
    with pytest.raises(ValueError, match="shares memory"):
        store_kvcache(k, v, kc, kc, pos)
    pool = torch.zeros(5, 8, hk, d, dtype=dtype, device="cuda")
    with pytest.raises(ValueError, match="shares memory"):
        store_kvcache(k, v, pool[:3], pool[2:], pos)
    # both caches in one allocation, one block of each after the other
    pair = torch.zeros(2, 2, 8, hk, d, dtype=dtype, device="cuda")
    got = rope_store_kvcache(q, k, v, pos, table, pair[:, 0], pair[:, 1], pos)
    assert torch.equal(got, want) and torch.equal(pair[:, 0], kc) and torch.equal(pair[:, 1], vc)
    assert torch.equal(rope_store_kvcache(q, k, v, pos, table, kc, vc, pos, out=q), want)
