"""B200: the step operators together, as a speculative engine uses them around the MoE block: draft steps of one token per
sequence, a verify step over the drafted spans, acceptance, and the next round over the same cache."""
import math
import subprocess
import sys

import pytest
import torch

from conftest import ROOT
from on_device_sd_b200 import MoEContext, paged_attention, rope_store_kvcache, rotary_table, verify_draft
from on_device_sd_b200.synth import make_layer
from test_gpu_verify_draft import rule

pytestmark = pytest.mark.gpu
L, H, E, K, I, HQ, HK, D, V, PAGE, B, GAMMA = 2, 64, 8, 2, 32, 4, 2, 32, 101, 4, 3, 3
EPS = 1e-6


class Model:
    """Two decoder layers in fp32: the library's norms, MoE block, cache write and attention; projections are torch's."""

    def __init__(self):
        g = torch.Generator("cuda").manual_seed(1)
        r = lambda *s, scale=1.0: scale * torch.randn(*s, generator=g, device="cuda")
        self.ctx = MoEContext(H, E, K, I, torch.float32, num_layers=L, max_tokens=64)
        for layer in range(L):
            m = make_layer(H, E, K, I, torch.float32, 1, seed=layer)
            self.ctx.set_gate(layer, m.gate_w.cuda() * 5)
            for e, p in m.experts.items():
                self.ctx.set_expert(layer, e, {k: (v * 8).cuda() for k, v in p.items()})
        self.emb, self.head = r(V, H), r(V, H, scale=0.4)
        self.draft_head = self.head + r(V, H, scale=0.05)
        self.wqkv, self.wo = r(L, (HQ + 2 * HK) * D, H, scale=H ** -0.5), r(L, H, HQ * D, scale=(HQ * D) ** -0.5)
        self.norms = 1 + r(L, 2, H, scale=0.1)
        self.qw, self.kw = 1 + r(L, D, scale=0.1), 1 + r(L, D, scale=0.1)
        self.table = rotary_table(D, 256, 1e4, "cuda")

    def run(self, tokens, attend):
        h = self.emb[tokens]
        for layer in range(L):
            x = self.ctx.rmsnorm(h, self.norms[layer, 0].contiguous(), EPS)
            q, k, v = (x @ self.wqkv[layer].T).view(-1, HQ + 2 * HK, D).split((HQ, HK, HK), 1)
            a = attend(layer, q, k, v)
            h = self.ctx.forward_fused_norm(layer, a.reshape(-1, HQ * D) @ self.wo[layer].T, self.norms[layer, 1].contiguous(), EPS, residual=h)
        return h

    def dense(self, tokens):
        """The same over a whole sequence, with norm, rotation and attention in 64 bits from the definitions."""
        pos = torch.arange(len(tokens), device="cuda")
        cos, sin = self.table[pos][:, None, : D // 2].double(), self.table[pos][:, None, D // 2:].double()

        def turn(x, w):
            x = x.double()
            x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w.double()
            a, b = x[..., : D // 2], x[..., D // 2:]
            return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)

        def attend(layer, q, k, v):
            q, k, v = turn(q, self.qw[layer]), turn(k, self.kw[layer]), v.double()
            k, v = k.repeat_interleave(HQ // HK, 1), v.repeat_interleave(HQ // HK, 1)
            s = torch.einsum("qhd,khd->hqk", q, k) / math.sqrt(D)
            s = s.masked_fill(pos[None, None, :] > pos[None, :, None], -math.inf)
            return torch.einsum("hqk,khd->qhd", s.softmax(-1), v).float()

        return self.run(tokens, attend)


class Cache:
    def __init__(self):
        g = torch.Generator("cuda").manual_seed(2)
        blocks = 3 * 16
        self.k = [torch.full((blocks, PAGE, HK, D), math.nan, device="cuda") for _ in range(L)]
        self.v = [t.clone() for t in self.k]
        self.tables = torch.randperm(blocks, generator=g, device="cuda").to(torch.int32).view(B, 16)

    def slots(self, seq, pos):
        return self.tables[seq, pos // PAGE].long() * PAGE + pos % PAGE

    def attend(self, model, seq, pos, lens, start=None, span=None):
        slots = self.slots(seq, pos)

        def f(layer, q, k, v):
            q = rope_store_kvcache(q, k, v, pos, model.table, self.k[layer], self.v[layer], slots, q_norm_weight=model.qw[layer],
                                   k_norm_weight=model.kw[layer], eps=EPS)
            return paged_attention(q, self.k[layer], self.v[layer], self.tables, lens, query_start=start, max_query_len=span)
        return f


def test_rounds_of_draft_verify_accept():
    model, cache = Model(), Cache()
    g = torch.Generator("cuda").manual_seed(3)
    seqs = [torch.randint(0, V, (n,), generator=g, device="cuda") for n in (5, 1, 9)]
    i32 = dict(dtype=torch.int32, device="cuda")
    # prompts: one ragged batch
    spans = [len(s) for s in seqs]
    starts = torch.tensor([0] + spans, **i32).cumsum(0).int()
    seq = torch.repeat_interleave(torch.arange(B, device="cuda"), torch.tensor(spans, device="cuda"))
    pos = torch.cat([torch.arange(n, device="cuda") for n in spans])
    h = model.run(torch.cat(seqs), cache.attend(model, seq, pos, torch.tensor(spans, **i32), starts, max(spans)))
    want = torch.cat([model.dense(s) for s in seqs])
    # fp32 against 64-bit attention through two layers: errors of 2^-24 on sums of at most 128 terms, a few hundred times that in all
    assert (h - want).abs().max() <= 1e-4 * want.abs().max()
    # every sequence's next token: the last row's most likely one
    last = [starts[b + 1].item() - 1 for b in range(B)]
    seqs = [torch.cat((s, (h[last[b]] @ model.head.T).argmax().view(1))) for b, s in enumerate(seqs)]
    taken = []
    for rounds in range(4):
        base = torch.tensor([len(s) for s in seqs], device="cuda")               # the last of these tokens is not in the cache yet
        tok = torch.stack([s[-1] for s in seqs])
        drafts, probs = [], []
        for j in range(GAMMA):
            p = base - 1 + j
            h = model.run(tok, cache.attend(model, torch.arange(B, device="cuda"), p, (p + 1).int()))
            dp = torch.softmax(h @ model.draft_head.T, -1)
            tok = torch.multinomial(dp, 1, generator=g).flatten()
            drafts.append(tok)
            probs.append(dp)
        counts = [GAMMA, rounds % (GAMMA + 1), GAMMA - rounds % 2]               # spans of different lengths, empty ones among them
        draft_start = torch.tensor([0] + counts, **i32).cumsum(0).int()
        dt = torch.cat([torch.stack(drafts)[:n, b] for b, n in enumerate(counts)])
        dp = torch.cat([torch.stack(probs)[:n, b] for b, n in enumerate(counts)])
        # verify: the last token and the drafts of each sequence; their keys overwrite those of the draft steps
        tokens = torch.cat([torch.cat((seqs[b][-1:], torch.stack(drafts)[: counts[b], b])) for b in range(B)])
        n1 = torch.tensor([n + 1 for n in counts], device="cuda")
        start = torch.cat((torch.zeros(1, device="cuda"), n1.cumsum(0))).int()
        seq = torch.repeat_interleave(torch.arange(B, device="cuda"), n1)
        pos = torch.cat([base[b] - 1 + torch.arange(counts[b] + 1, device="cuda") for b in range(B)])
        h = model.run(tokens, cache.attend(model, seq, pos, (base + n1 - 1).int(), start, GAMMA + 1))
        for b in range(B):
            full = model.dense(torch.cat((seqs[b], torch.stack(drafts)[: counts[b], b])))
            rows = slice(int(start[b]), int(start[b + 1]))
            assert (h[rows] - full[len(seqs[b]) - 1:]).abs().max() <= 1e-4 * full.abs().max()
        target = torch.softmax(h @ model.head.T, -1)
        u, w = torch.rand(len(dt), generator=g, device="cuda"), torch.rand(B, generator=g, device="cuda")
        out, acc = verify_draft(dt, target, dp, u, w, draft_start=draft_start, max_draft_len=GAMMA)
        ro, ra = rule(dt, target, dp, u, w, draft_start.tolist(), GAMMA)
        assert torch.equal(out.cpu(), ro) and torch.equal(acc.cpu(), ra)
        taken += acc.tolist()
        seqs = [torch.cat((s, out[b, : int(acc[b]) + 1])) for b, s in enumerate(seqs)]
    assert 0 < sum(taken) < 4 * B * GAMMA, "some drafts were taken and some refused"
    # what the cache holds after the rounds is what the tokens say: one more draft step
    base = torch.tensor([len(s) for s in seqs], device="cuda")
    h = model.run(torch.stack([s[-1] for s in seqs]), cache.attend(model, torch.arange(B, device="cuda"), base - 1, base.int()))
    for b in range(B):
        full = model.dense(seqs[b])
        assert (h[b] - full[-1]).abs().max() <= 1e-4 * full.abs().max()


def test_captured_draft_step_replays_as_the_sequence_grows():
    """One graph of a whole draft step (both layers, MoE included), replayed with new tokens, positions and lengths."""
    model, cache, eager = Model(), Cache(), Cache()
    tok, pos, lens = torch.zeros(B, dtype=torch.long, device="cuda"), torch.zeros(B, dtype=torch.long, device="cuda"), torch.ones(B, dtype=torch.int32, device="cuda")
    seq = torch.arange(B, device="cuda")
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        model.run(tok, cache.attend(model, seq, pos, lens))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = model.run(tok, cache.attend(model, seq, pos, lens))
    g = torch.Generator("cuda").manual_seed(4)
    for step in range(40):
        t = torch.randint(0, V, (B,), generator=g, device="cuda")
        tok.copy_(t)
        pos.fill_(step)
        lens.fill_(step + 1)
        graph.replay()
        want = model.run(t, eager.attend(model, seq, pos.clone(), lens.clone()))
        torch.cuda.synchronize()
        assert torch.equal(out, want)


FIRST_CALL = """
import sys, torch
sys.path.insert(0, sys.argv[1])
from on_device_sd_b200 import paged_attention, rope_store_kvcache, rotary_table, verify_draft
q = torch.randn(2, 8, 64, device="cuda").half(); k = torch.randn(2, 2, 64, device="cuda").half()
kc, vc = (torch.randn(40, 16, 2, 64, device="cuda").half() for _ in range(2))
tables = torch.arange(40, dtype=torch.int32, device="cuda").view(2, 20)
lens = torch.tensor([300, 7], dtype=torch.int32, device="cuda"); pos = torch.tensor([299, 6], device="cuda")
slots = tables.gather(1, (pos // 16)[:, None]).long().flatten() * 16 + pos % 16
table = rotary_table(64, 512, device="cuda")
p = torch.softmax(torch.randn(4, 1000, device="cuda"), -1); d = torch.softmax(torch.randn(2, 1000, device="cuda"), -1)
tok = torch.tensor([3, 5], device="cuda"); u = torch.rand(2, device="cuda"); w = torch.rand(2, device="cuda")
start = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
def step():
    x = rope_store_kvcache(q, k, k, pos, table, kc, vc, slots)
    return paged_attention(x, kc, vc, tables, lens), *verify_draft(tok, p, d, u, w, draft_start=start, max_draft_len=1)
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    outs = step()
for o in outs: o.fill_(9)
g.replay()
want = step()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(outs, want))
"""


def test_first_call_of_a_process_may_be_captured():
    r = subprocess.run([sys.executable, "-c", FIRST_CALL, str(ROOT)], capture_output=True, text=True, timeout=180)
    assert r.returncode == 0, r.stderr[-2000:]
