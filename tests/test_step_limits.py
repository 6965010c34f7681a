"""CPU: sizes whose products would pass the integers of the kernels are refused before any launch."""
import ctypes

import pytest

from on_device_sd_b200 import _lib
from test_step_refusals import attn_args, store_args

BIG = dict(block_size=1 << 15, max_blocks_per_seq=1 << 15)        # 2^30 slots, the most a table may span


@pytest.mark.parametrize("change, word", [
    (dict(num_tokens=1 << 27, num_seqs=1 << 27, num_heads=8, num_kv_heads=8, **BIG), b"work"),
    (dict(num_tokens=1 << 27, num_seqs=1 << 27, num_heads=8, num_kv_heads=2, **BIG), b"work"),
    (dict(num_tokens=1 << 28, num_seqs=1 << 28, num_heads=8, num_kv_heads=2), b"tokens x heads"),
])
def test_attention_work(change, word):
    lib = _lib.load()
    assert lib.b200moe_paged_attention(ctypes.byref(attn_args(**change)), None) == _lib.E_UNSUPPORTED
    assert word in lib.b200moe_last_error(None)


@pytest.mark.parametrize("change", [
    dict(num_tokens=1 << 17, num_seqs=1 << 17, num_heads=8, num_kv_heads=8, **BIG),       # 2^17 sequences of 2^30 slots
    dict(num_tokens=4096, num_seqs=4096, num_heads=128, num_kv_heads=8, block_size=256, max_blocks_per_seq=4096),
])
def test_large_calls_pass_the_checks(change):
    """Without a device the next thing that is missing is the device."""
    import torch
    if torch.cuda.is_available():
        pytest.skip("the arguments point nowhere")
    lib = _lib.load()
    assert lib.b200moe_paged_attention(ctypes.byref(attn_args(**change)), None) == _lib.E_CUDA


def test_store_heads():
    lib = _lib.load()
    assert lib.b200moe_store_kv(ctypes.byref(store_args(num_tokens=1 << 29)), None) == _lib.E_UNSUPPORTED
    assert b"tokens x heads" in lib.b200moe_last_error(None)
