"""CPU: what the cache write, the paged attention and the draft verification refuse, before any launch."""
import ctypes

import pytest
import torch

from on_device_sd_b200 import _lib, paged_attention, rope_store_kvcache, rotary_table, store_kvcache, verify_draft

P = 4096   # any 16-byte aligned address: refused calls never look behind it


def store_args(**kw):
    a = _lib.StoreKvArgs()
    for n in ("query", "key", "value", "query_out", "k_cache", "v_cache", "positions", "slots", "cos_sin"):
        setattr(a, n, P)
    for n in ("q_token_stride", "q_head_stride", "k_token_stride", "k_head_stride", "v_token_stride", "v_head_stride", "o_token_stride",
              "o_head_stride", "cache_block_stride", "cache_slot_stride", "cache_head_stride"):
        setattr(a, n, 1024)
    a.num_tokens, a.num_heads, a.num_kv_heads, a.head_dim, a.num_blocks, a.block_size, a.max_position, a.dtype = 4, 8, 2, 64, 3, 16, 100, _lib.BF16
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def attn_args(**kw):
    a = _lib.PagedAttentionArgs()
    for n in ("query", "k_cache", "v_cache", "block_tables", "context_lens", "out"):
        setattr(a, n, P)
    for n in ("q_token_stride", "q_head_stride", "o_token_stride", "o_head_stride", "cache_block_stride", "cache_slot_stride", "cache_head_stride"):
        setattr(a, n, 1024)
    a.num_tokens = a.num_seqs = 4
    a.num_heads, a.num_kv_heads, a.head_dim, a.num_blocks, a.block_size, a.max_blocks_per_seq, a.max_query_len = 8, 2, 64, 3, 16, 2, 1
    a.dtype, a.scale = _lib.BF16, 0.125
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def verify_args(**kw):
    a = _lib.VerifyDraftArgs()
    for n in ("draft_tokens", "target_probs", "draft_probs", "accept_uniform", "sample_uniform", "draft_start", "tokens_out", "accepted_out"):
        setattr(a, n, P)
    a.target_stride = a.draft_stride = 1000
    a.num_seqs, a.vocab_size, a.max_draft_len, a.num_draft_tokens, a.num_target_rows, a.dtype = 2, 1000, 4, 8, 10, _lib.F32
    for k, v in kw.items():
        setattr(a, k, v)
    return a


ARG, UNSUP = _lib.E_ARG, _lib.E_UNSUPPORTED


@pytest.mark.parametrize("change, code, word", [
    (dict(dtype=7), ARG, b"dtype"), (dict(head_dim=80), UNSUP, b"head_dim"), (dict(num_heads=7), ARG, b"multiple"),
    (dict(num_kv_heads=0), ARG, b"head counts"), (dict(num_tokens=-1), ARG, b"negative"), (dict(block_size=0), ARG, b"negative"),
    (dict(key=None), ARG, b"null"), (dict(slots=None), ARG, b"null"), (dict(query_out=None), ARG, b"query_out"),
    (dict(positions=None), ARG, b"positions"), (dict(max_position=0), ARG, b"positions"), (dict(value=P + 2), ARG, b"aligned"),
    (dict(k_norm_weight=P + 8), ARG, b"aligned"), (dict(k_token_stride=1028), ARG, b"strides"), (dict(cache_head_stride=4), ARG, b"strides"),
])
def test_store_refuses(change, code, word):
    lib = _lib.load()
    assert lib.b200moe_store_kv(ctypes.byref(store_args(**change)), None) == code
    assert word in lib.b200moe_last_error(None)


@pytest.mark.parametrize("change, code, word", [
    (dict(dtype=-1), ARG, b"dtype"), (dict(head_dim=96), UNSUP, b"head_dim"), (dict(num_kv_heads=3), ARG, b"multiple"),
    (dict(num_tokens=5), ARG, b"one token per sequence"), (dict(num_seqs=-1), ARG, b"negative"), (dict(block_size=0), ARG, b"negative"),
    (dict(max_query_len=-2), ARG, b"negative"), (dict(context_lens=None), ARG, b"null"), (dict(block_tables=None), ARG, b"null"),
    (dict(out=None), ARG, b"null"), (dict(query=P + 4), ARG, b"aligned"), (dict(workspace=P + 4), ARG, b"aligned"),
    (dict(q_head_stride=1001), ARG, b"strides"), (dict(scale=0.0), ARG, b"scale"), (dict(scale=-1.0), ARG, b"scale"),
    (dict(scale=float("nan")), ARG, b"scale"), (dict(scale=float("inf")), ARG, b"scale"),
    (dict(block_size=1 << 20, max_blocks_per_seq=1 << 12), UNSUP, b"slots"),
])
def test_attention_refuses(change, code, word):
    lib = _lib.load()
    assert lib.b200moe_paged_attention(ctypes.byref(attn_args(**change)), None) == code
    assert word in lib.b200moe_last_error(None)


@pytest.mark.parametrize("change, code, word", [
    (dict(dtype=3), ARG, b"dtype"), (dict(vocab_size=0), ARG, b"vocabulary"), (dict(num_seqs=-1), ARG, b"negative"),
    (dict(max_draft_len=-1), ARG, b"negative"), (dict(vocab_size=(1 << 30) + 1), UNSUP, b"vocabulary"), (dict(num_seqs=1 << 25), UNSUP, b"2^24"),
    (dict(target_probs=None), ARG, b"null"), (dict(draft_tokens=None), ARG, b"null"), (dict(accept_uniform=None), ARG, b"null"),
    (dict(tokens_out=None), ARG, b"null"), (dict(draft_start=None), ARG, b"null"),
])
def test_verify_refuses(change, code, word):
    lib = _lib.load()
    assert lib.b200moe_verify_draft(ctypes.byref(verify_args(**change)), None) == code
    assert word in lib.b200moe_last_error(None)


def test_null_arguments_and_empty_calls():
    lib = _lib.load()
    for f in (lib.b200moe_store_kv, lib.b200moe_paged_attention, lib.b200moe_verify_draft):
        assert f(None, None) == _lib.E_ARG
    assert lib.b200moe_store_kv(ctypes.byref(store_args(num_tokens=0)), None) == _lib.OK
    assert lib.b200moe_paged_attention(ctypes.byref(attn_args(num_tokens=0, num_seqs=0)), None) == _lib.OK
    assert lib.b200moe_verify_draft(ctypes.byref(verify_args(num_seqs=0)), None) == _lib.OK
    n = ctypes.c_int64(-1)
    ws = lib.b200moe_paged_attention_workspace
    assert ws(_lib.BF16, 1, 32, 4, 128, 1, 4, 16, None) == _lib.E_ARG
    assert ws(_lib.BF16, 1, 32, 5, 128, 1, 4, 16, ctypes.byref(n)) == _lib.E_ARG
    assert ws(_lib.BF16, 1, 32, 4, 128, -1, 4, 16, ctypes.byref(n)) == _lib.E_ARG
    assert ws(_lib.BF16, -1, 32, 4, 128, 1, 4, 16, ctypes.byref(n)) == _lib.E_ARG
    assert ws(_lib.BF16, 1, 32, 4, 128, 1, 4, 0, ctypes.byref(n)) == _lib.E_ARG
    assert ws(_lib.BF16, 1, 32, 4, 100, 1, 4, 16, ctypes.byref(n)) == _lib.E_UNSUPPORTED


def test_argument_structs_have_the_headers_layout(tmp_path):
    """Sizes and the offsets of the last fields, from the C compiler."""
    import shutil
    import subprocess
    from conftest import ROOT
    gcc = shutil.which("gcc")
    if gcc is None:
        pytest.skip("no gcc")
    fields = [("b200moe_store_kv_args", _lib.StoreKvArgs), ("b200moe_paged_attention_args", _lib.PagedAttentionArgs),
              ("b200moe_verify_draft_args", _lib.VerifyDraftArgs)]
    lines = ['#include <stddef.h>', '#include <stdio.h>', '#include "b200moe.h"', "int main(void){"]
    for name, cls in fields:
        lines.append(f'printf("%zu\\n", sizeof({name}));')
        for f, _ in cls._fields_:
            lines.append(f'printf("%zu\\n", offsetof({name}, {f}));')
    src = tmp_path / "layout.c"
    src.write_text("\n".join(lines + ["return 0;}"]))
    exe = tmp_path / "layout"
    subprocess.run([gcc, "-std=c99", "-I", str(ROOT / "include"), str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    want = []
    for _, cls in fields:
        want.append(ctypes.sizeof(cls))
        want += [getattr(cls, f).offset for f, _ in cls._fields_]
    assert got == want


def test_status_bits_match_the_header():
    import re
    from conftest import ROOT
    text = (ROOT / "include" / "b200moe.h").read_text()
    for n in ("BAD_EXPERT_ID", "BAD_OFFSETS", "WAIT_EXPIRED", "BAD_SLOT", "BAD_POSITION", "BAD_PAGE", "BAD_LENGTH", "BAD_TOKEN", "BAD_PROBS"):
        m = re.search(rf"#define\s+B200MOE_DEV_{n}\s+(\d+)", text)
        assert m and int(m.group(1)) == getattr(_lib, f"DEV_{n}")


def test_cpu_tensors_are_refused():
    q, k = torch.zeros(2, 4, 32), torch.zeros(2, 2, 32)
    cache, i32 = torch.zeros(2, 16, 2, 32), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="no CPU path"):
        paged_attention(q, cache, cache, torch.zeros(2, 1, dtype=torch.int32), i32)
    with pytest.raises(ValueError, match="no CPU path"):
        store_kvcache(k, k, cache, cache, i32)
    with pytest.raises(ValueError, match="no CPU path"):
        rope_store_kvcache(q, k, k, i32, rotary_table(32, 8), cache, cache, i32)
    with pytest.raises(ValueError, match="no CPU path"):
        verify_draft(torch.zeros(2, dtype=torch.int64), torch.zeros(3, 8), None, torch.zeros(2), torch.zeros(1),
                     draft_start=torch.tensor([0, 2], dtype=torch.int32), max_draft_len=2)
    with pytest.raises(TypeError, match="unsupported dtype"):
        paged_attention(q.double(), cache.double(), cache.double(), torch.zeros(2, 1, dtype=torch.int32), i32)


def test_rotary_table_is_the_formula_in_64_bits():
    import math
    t = rotary_table(64, 5000, 1e4)
    assert t.shape == (5000, 64) and t.dtype == torch.float32
    for pos, i in ((0, 0), (1, 0), (4999, 0), (4999, 31), (777, 13)):
        a = pos * 1e4 ** (-2 * i / 64)
        # one rounding to fp32, and the last digits of two 64-bit evaluations
        assert abs(t[pos, i].item() - math.cos(a)) <= 2.0 ** -24 + 1e-11
        assert abs(t[pos, 32 + i].item() - math.sin(a)) <= 2.0 ** -24 + 1e-11
