"""The attention side of a speculative decoding step, as cases to time: writing new keys and values into a paged
cache (head norm and rotary embedding included), attention of one or a few new tokens per sequence over that cache,
and the verification of drafted tokens.

`listed()` and `draw()` give cases, `prepare()` what a program has in hand before the call, `run()` one pass: the
operators in elementary torch operations, or the library's calls when `own` is set.  `exact()` evaluates the
definitions in 64 bits."""
import math
import random

import torch

own = False

_DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
_BYTES = {"float32": 4, "float16": 2, "bfloat16": 2}
_EPS = 1e-6


# -- cases ------------------------------------------------------------------------------------------
def _attention(name, batch, span, context, heads, kv_heads, head_dim, page, dtype, ragged, lse, spread):
    return {"name": name, "op": "attention", "batch": batch, "span": span, "context": context, "heads": heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "page": page, "dtype": dtype, "ragged": ragged, "lse": lse, "spread": spread}


def _store(name, tokens, heads, kv_heads, head_dim, page, dtype, norm, spread):
    return {"name": name, "op": "store", "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "page": page,
            "dtype": dtype, "norm": norm, "spread": spread}


def _verify(name, batch, drafts, vocab, dtype, sampled, ragged, spread):
    return {"name": name, "op": "verify", "batch": batch, "drafts": drafts, "vocab": vocab, "dtype": dtype, "sampled": sampled,
            "ragged": ragged, "spread": spread}


def listed():
    return [
        # one sequence's draft step just after a short prompt: nothing but latency
        _attention("attn_first_token", 1, 1, 33, 32, 4, 128, 256, "bfloat16", False, False, 1),
        # draft step of a batch in mid-generation, Qwen3-shaped heads, the engine's pages of 256 slots
        _attention("attn_draft_batch", 16, 1, 6000, 32, 4, 128, 256, "bfloat16", True, False, 2),
        # verify step: spans of up to 5 tokens (4 drafted and the one before), Mixtral-shaped heads, small pages
        _attention("attn_verify_batch", 32, 5, 2500, 32, 8, 128, 16, "float16", True, False, 3),
        # one long document: few rows, all parallelism along the cache
        _attention("attn_long_single", 1, 1, 131071, 32, 4, 128, 256, "bfloat16", False, True, 4),
        # full-precision toy model with small heads and pages that divide nothing
        _attention("attn_fp32_small", 7, 3, 1000, 8, 2, 64, 24, "float32", True, True, 5),
        # the largest verify batch: 64 sequences of up to 16384 tokens, spans of up to 5
        _attention("attn_verify_large", 64, 5, 16384, 32, 4, 128, 256, "bfloat16", True, False, 6),
        # the token of a single sequence's draft step
        _store("store_one_token", 1, 32, 4, 128, 256, "bfloat16", True, 7),
        # the tokens of a verify batch
        _store("store_verify_batch", 257, 32, 4, 128, 256, "bfloat16", True, 8),
        # a chunk of a prompt, heads without norms
        _store("store_prompt_chunk", 8191, 32, 8, 128, 16, "float16", False, 9),
        # one sequence with four drafted tokens
        _verify("verify_one", 1, 4, 32000, "float32", True, False, 10),
        # a verify batch over a large vocabulary, drafts sampled from a distribution
        _verify("verify_batch", 48, 5, 151936, "float32", True, True, 11),
        # the same with greedy drafts (no draft distribution) and 16-bit target probabilities
        _verify("verify_greedy_bf16", 64, 4, 128256, "bfloat16", False, True, 12),
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["attention", "attention", "store", "verify"])
    spread = rng.randrange(1 << 30)
    heads, kv_heads, head_dim = rng.choice([(32, 4, 128), (32, 8, 128), (16, 2, 64), (8, 8, 128), (8, 1, 256), (4, 2, 32), (12, 2, 128)])
    page = rng.choice([1, 16, 24, 64, 128, 256])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    if kind == "attention":
        batch = _log_int(rng, 1, 128)
        span = rng.choice([1, 1, 1, 2, 3, 5, 8])
        context = _log_int(rng, span, 100000)
        row = kv_heads * head_dim * _BYTES[dtype] * 2
        context = max(span, min(context, (1 << 29) // (row * batch)))
        return _attention("", batch, span, context, heads, kv_heads, head_dim, page, dtype, rng.random() < 0.7, rng.random() < 0.5, spread)
    if kind == "store":
        return _store("", _log_int(rng, 1, 4000), heads, kv_heads, head_dim, page, dtype, rng.random() < 0.5, spread)
    return _verify("", _log_int(rng, 1, 48), rng.choice([1, 2, 3, 4, 5]), _log_int(rng, 500, 151936), dtype, rng.random() < 0.6,
                   rng.random() < 0.6, spread)


def _lengths(case):
    """(new tokens, tokens in the cache with them) of every sequence of an attention case."""
    rng = random.Random(case["spread"])
    spans, contexts = [], []
    for _ in range(case["batch"]):
        n = rng.randint(1, case["span"]) if case["ragged"] else case["span"]
        c = int(case["context"] * rng.uniform(0.05, 1.0)) if case["ragged"] else case["context"]
        spans.append(n)
        contexts.append(max(n, c))
    return spans, contexts


def _draft_counts(case):
    rng = random.Random(case["spread"])
    return [rng.randint(0, case["drafts"]) if case["ragged"] else case["drafts"] for _ in range(case["batch"])]


def work(case):
    e = _BYTES[case["dtype"]] if "dtype" in case else 4
    if case["op"] == "attention":
        spans, contexts = _lengths(case)
        d, h, hk = case["head_dim"], case["heads"], case["kv_heads"]
        pairs = sum(n * (c - n) + n * (n + 1) // 2 for n, c in zip(spans, contexts))
        pages = sum((c + case["page"] - 1) // case["page"] for c in contexts)
        moved = 2 * sum(contexts) * hk * d * e + 2 * sum(spans) * h * d * e + 4 * (pages + 2 * case["batch"])
        if case["lse"]:
            moved += 4 * sum(spans) * h
        return {"bytes": moved, "flops": 4 * pairs * h * d}
    if case["op"] == "store":
        t, d, h, hk = case["tokens"], case["head_dim"], case["heads"], case["kv_heads"]
        moved = 2 * t * (h + 2 * hk) * d * e + t * (d * 4 + 16)
        return {"bytes": moved, "flops": t * (h + hk) * d * (3 + (4 if case["norm"] else 0))}
    # verification ends in one draw per sequence from a row of the target's probabilities, less the draft's row where a
    # sampled draft was refused; which one it is depends on the data, so the larger is stated where a draft exists
    counts = _draft_counts(case)
    rows = sum(2 if n and case["sampled"] else 1 for n in counts)
    n = sum(counts)
    return {"bytes": rows * case["vocab"] * e + n * (8 + 4 + 2 * e) + len(counts) * (8 + (case["drafts"] + 1) * 8),
            "flops": 3 * rows * case["vocab"]}


# -- inputs -----------------------------------------------------------------------------------------
def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g, device="cuda", dtype=dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 1000003 + case["spread"])
    dt = _DTYPES[case["dtype"]]
    return {"attention": _prepare_attention, "store": _prepare_store, "verify": _prepare_verify}[case["op"]](case, g, dt)


def _prepare_attention(case, g, dt):
    spans, contexts = _lengths(case)
    h, hk, d, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    used = [(c + page - 1) // page for c in contexts]
    blocks = sum(used) + 3
    # queries and keys after head norms have unit scale; pages lie in the order in which a pool handed them out
    k = _randn(g, blocks, page, hk, d, dtype=dt)
    v = _randn(g, blocks, page, hk, d, dtype=dt)
    q = _randn(g, sum(spans), h, d, dtype=dt)
    order = torch.randperm(blocks, generator=g, device="cuda").to(torch.int32)
    tables = torch.zeros(len(spans), max(used), dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(used):
        tables[i, :n] = order[at: at + n]
        at += n
    starts = [0]
    for n in spans:
        starts.append(starts[-1] + n)
    return {"op": "attention", "q": q, "k": k, "v": v, "tables": tables, "spans": spans, "contexts": contexts, "starts": starts,
            "context_lens": torch.tensor(contexts, dtype=torch.int32, device="cuda"),
            "query_start": torch.tensor(starts, dtype=torch.int32, device="cuda"), "span": case["span"], "lse": case["lse"]}


def _angles(d, positions, base=1e6):
    inv = base ** (-torch.arange(0, d, 2, dtype=torch.float64, device="cuda") / d)
    a = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * inv
    return torch.cat((a.cos(), a.sin()), dim=-1).float()


def _prepare_store(case, g, dt):
    t, h, hk, d, page = case["tokens"], case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    blocks = (t + page - 1) // page + 2
    limit = 40960
    # the projection's output row holds queries, keys and values side by side
    qkv = _randn(g, t, (h + 2 * hk) * d, dtype=dt)
    q, k, v = (x.view(t, -1, d) for x in qkv.split((h * d, hk * d, hk * d), dim=-1))
    slots = torch.randperm(blocks * page, generator=g, device="cuda")[:t]
    if t > 8:
        slots[t // 2] = -1        # a padded token of a captured batch
    weights = [1.0 + 0.1 * _randn(g, d) for _ in range(2)] if case["norm"] else [None, None]
    return {"op": "store", "q": q, "k": k, "v": v, "slots": slots, "cos_sin": _angles(d, limit),
            "positions": torch.randint(0, limit, (t,), generator=g, device="cuda"),
            "q_weight": None if weights[0] is None else weights[0].to(dt), "k_weight": None if weights[1] is None else weights[1].to(dt),
            "k_cache": _randn(g, blocks, page, hk, d, dtype=dt), "v_cache": _randn(g, blocks, page, hk, d, dtype=dt)}


def _prepare_verify(case, g, dt):
    counts, vocab = _draft_counts(case), case["vocab"]
    total, batch = sum(counts), len(counts)
    target_logits = _randn(g, total + batch, vocab) * 2.5
    starts = [0]
    for n in counts:
        starts.append(starts[-1] + n)
    rows = torch.tensor([s + i + j for i, (s, n) in enumerate(zip(starts, counts)) for j in range(n)], dtype=torch.int64, device="cuda")
    # the draft model is close to the target; greedy drafts are its most likely token
    draft_logits = target_logits[rows] + _randn(g, total, vocab) * 0.7
    draft = torch.softmax(draft_logits, dim=-1)
    if case["sampled"]:
        noise = torch.rand(total, vocab, generator=g, device="cuda").clamp_min(1e-9)
        tokens = (draft_logits - torch.log(-torch.log(noise))).argmax(dim=-1) if total else rows
    else:
        tokens = draft_logits.argmax(dim=-1) if total else rows
    return {"op": "verify", "tokens": tokens, "target": torch.softmax(target_logits, dim=-1).to(dt),
            "draft": draft.to(dt) if case["sampled"] else None, "counts": counts, "drafts": case["drafts"],
            "accept": torch.rand(total, generator=g, device="cuda"), "sample": torch.rand(batch, generator=g, device="cuda"),
            "starts": torch.tensor(starts, dtype=torch.int32, device="cuda")}


# -- one pass ---------------------------------------------------------------------------------------
def run(state):
    if own:
        return {"attention": _own_attention, "store": _own_store, "verify": _own_verify}[state["op"]](state)
    return {"attention": _plain_attention, "store": _plain_store, "verify": _plain_verify}[state["op"]](state)


def _own_attention(s):
    from on_device_sd_b200 import paged_attention
    return paged_attention(s["q"], s["k"], s["v"], s["tables"], s["context_lens"], query_start=s["query_start"] if s["span"] > 1 else None,
                           max_query_len=s["span"], return_lse=s["lse"])


def _own_store(s):
    from on_device_sd_b200 import rope_store_kvcache
    out = rope_store_kvcache(s["q"], s["k"], s["v"], s["positions"], s["cos_sin"], s["k_cache"], s["v_cache"], s["slots"],
                             q_norm_weight=s["q_weight"], k_norm_weight=s["k_weight"], eps=_EPS)
    return out, s["k_cache"], s["v_cache"]


def _own_verify(s):
    from on_device_sd_b200 import verify_draft
    return verify_draft(s["tokens"], s["target"], s["draft"], s["accept"], s["sample"], draft_start=s["starts"], max_draft_len=s["drafts"])


def _plain_attention(s):
    q, page = s["q"], s["k"].shape[1]
    t, h, d = q.shape
    hk = s["k"].shape[2]
    out = torch.empty_like(q)
    lse = torch.empty(t, h, dtype=torch.float32, device=q.device)
    for i, (n, c, at) in enumerate(zip(s["spans"], s["contexts"], s["starts"])):
        ids = s["tables"][i, : (c + page - 1) // page].long()
        k = s["k"][ids].view(-1, hk, d)[:c].float()
        v = s["v"][ids].view(-1, hk, d)[:c].float()
        x = q[at: at + n].float().view(n, hk, h // hk, d)
        scores = torch.matmul(x.permute(1, 2, 0, 3).reshape(hk, -1, d), k.permute(1, 2, 0)) / math.sqrt(d)      # [kv head, (group, token), key]
        visible = torch.arange(c, device=q.device) <= (c - n + torch.arange(n, device=q.device))[:, None]
        scores = scores.view(hk, h // hk, n, c).masked_fill(~visible, -math.inf)
        top = scores.amax(dim=-1, keepdim=True)
        p = torch.exp(scores - top)
        norm = p.sum(dim=-1, keepdim=True)
        y = torch.matmul((p / norm).view(hk, -1, c), v.permute(1, 0, 2)).view(hk, h // hk, n, d)
        out[at: at + n] = y.permute(2, 0, 1, 3).reshape(n, h, d).to(q.dtype)
        lse[at: at + n] = (top + torch.log(norm)).squeeze(-1).permute(2, 0, 1).reshape(n, h)
    return (out, lse) if s["lse"] else out


def _rotate(x, weight, angles, work_dtype):
    x = x.to(work_dtype)
    if weight is not None:
        x = x / torch.sqrt((x * x).mean(dim=-1, keepdim=True) + _EPS) * weight.to(work_dtype)
    half = x.shape[-1] // 2
    cos, sin = angles[:, None, :half].to(work_dtype), angles[:, None, half:].to(work_dtype)
    a, b = x[..., :half], x[..., half:]
    return torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)


def _plain_store(s):
    dt = s["q"].dtype
    angles = s["cos_sin"][s["positions"]]
    q = _rotate(s["q"], s["q_weight"], angles, torch.float32).to(dt)
    k = _rotate(s["k"], s["k_weight"], angles, torch.float32).to(dt)
    keep = s["slots"] >= 0
    slots = s["slots"][keep]
    hk, d = k.shape[1:]
    s["k_cache"].view(-1, hk, d)[slots] = k[keep]
    s["v_cache"].view(-1, hk, d)[slots] = s["v"][keep]
    return q, s["k_cache"], s["v_cache"]


def _plain_verify(s):
    tokens, target, draft, starts, width = s["tokens"], s["target"], s["draft"], s["starts"].long(), s["drafts"]
    dev = tokens.device
    first, counts = starts[:-1], starts[1:] - starts[:-1]
    batch = counts.numel()
    step = torch.arange(width, device=dev)
    real = step[None] < counts[:, None]
    at = torch.where(real, first[:, None] + step[None], 0)
    if tokens.numel():
        x = tokens[at]
        row = at + torch.arange(batch, device=dev)[:, None]
        p = target[row, x].double()
        q = draft[at, x].double() if draft is not None else torch.ones_like(p)
        good = real & (p > s["accept"][at].double() * q)
    else:
        x, good = torch.zeros_like(at), real
    accepted = good.long().cumprod(dim=1).sum(dim=1)
    # the draw after the accepted prefix; sums over a vocabulary in 64 bits, or neighbouring tokens would change places
    rest = target[first + torch.arange(batch, device=dev) + accepted].double()
    stopped = accepted < counts
    if tokens.numel():
        where = torch.where(stopped, first + accepted, 0)
        if draft is not None:
            less = (rest - draft[where].double()).clamp_min(0.0)
        else:
            less = rest.scatter(1, tokens[where][:, None], 0.0)
        rest = torch.where(stopped[:, None] & (less.sum(dim=1, keepdim=True) > 0), less, rest)
    run_sum = rest.cumsum(dim=1)
    goal = s["sample"].double()[:, None] * run_sum[:, -1:]
    last = rest.shape[1] - 1 - (rest > 0).flip(1).long().argmax(dim=1)
    hit = run_sum > goal
    token = torch.where(hit.any(dim=1), hit.long().argmax(dim=1), last)
    out = torch.full((batch, width + 1), -1, dtype=torch.int64, device=dev)
    out[:, :width] = torch.where(step[None] < accepted[:, None], x, -1)
    out.scatter_(1, accepted[:, None], token[:, None])
    return out, accepted.int()


# -- the definitions in 64 bits ---------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"attention": _exact_attention, "store": _exact_store, "verify": _exact_verify}[case["op"]](s)


def _exact_attention(s):
    q, k, v = s["q"], s["k"], s["v"]
    h, hk, d, page = q.shape[1], k.shape[2], q.shape[2], k.shape[1]
    out = torch.empty(q.shape, dtype=torch.float64, device=q.device)
    lse = torch.empty(q.shape[:2], dtype=torch.float64, device=q.device)
    for b, c in enumerate(s["contexts"]):
        key = torch.arange(c, device=q.device)
        block = s["tables"][b].long()[key // page]
        for j in range(hk):
            kj, vj = k[block, key % page, j].double(), v[block, key % page, j].double()
            heads = slice(j * (h // hk), (j + 1) * (h // hk))
            for i in range(s["spans"][b]):
                row = s["starts"][b] + i
                n = c - s["spans"][b] + i + 1
                z = q[row, heads].double() @ kj[:n].T / math.sqrt(d)
                total = torch.logsumexp(z, dim=-1)
                out[row, heads] = torch.exp(z - total[:, None]) @ vj[:n]
                lse[row, heads] = total
    return (out, lse) if s["lse"] else out


def _exact_store(s):
    d = s["q"].shape[-1]
    table = s["cos_sin"].double()[s["positions"]]
    turn = torch.complex(table[:, : d // 2], table[:, d // 2:])[:, None]

    def turned(x, w):
        x = x.double()
        if w is not None:
            x = x * torch.rsqrt(x.square().sum(dim=-1, keepdim=True) / d + _EPS) * w.double()
        z = torch.complex(x[..., : d // 2], x[..., d // 2:]) * turn
        return torch.cat((z.real, z.imag), dim=-1)

    q, k = turned(s["q"], s["q_weight"]), turned(s["k"], s["k_weight"])
    k_cache, v_cache = s["k_cache"].double(), s["v_cache"].double()
    page = k_cache.shape[1]
    used = torch.nonzero(s["slots"] >= 0).flatten()
    slot = s["slots"][used]
    k_cache[slot // page, slot % page] = k[used]
    v_cache[slot // page, slot % page] = s["v"][used].double()
    return q, k_cache, v_cache


def _exact_verify(s):
    starts = s["starts"].tolist()
    tokens, accept, sample = s["tokens"].tolist(), s["accept"].tolist(), s["sample"].tolist()
    out = torch.full((len(sample), s["drafts"] + 1), -1, dtype=torch.int64)
    taken = []
    for b, u in enumerate(sample):
        n, base = starts[b + 1] - starts[b], starts[b]
        j = 0
        while j < n:
            x = tokens[base + j]
            p = float(s["target"][base + b + j, x])
            q = float(s["draft"][base + j, x]) if s["draft"] is not None else 1.0
            if not p > accept[base + j] * q:
                break
            out[b, j] = x
            j += 1
        rest = s["target"][base + b + j].double()
        if j < n:
            less = torch.zeros_like(rest)
            if s["draft"] is not None:
                less = (rest - s["draft"][base + j].double()).clamp(min=0)
            else:
                less.copy_(rest)
                less[tokens[base + j]] = 0
            if float(less.sum()) > 0:
                rest = less
        sums = torch.cumsum(rest, dim=0)
        past = torch.nonzero(sums > u * sums[-1])
        token = past[0] if past.numel() else torch.nonzero(rest > 0)[-1]
        out[b, j] = int(token)
        taken.append(j)
    return out.to(s["tokens"].device), torch.tensor(taken, dtype=torch.int32, device=s["tokens"].device)
