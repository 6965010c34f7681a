"""B200: verification against target rows that are too few or more than needed, and batches around every launch form."""
import pytest
import torch

from on_device_sd_b200 import _lib, verify_draft
from test_gpu_verify_draft import BF16, F16, F32, check, make, run

pytestmark = pytest.mark.gpu


def test_fewer_target_rows_than_sequences_are_refused():
    c = make([1, 0, 2], 300, F32, True, seed=90)
    with pytest.raises(ValueError, match="target_probs"):
        run(dict(c, target=c["target"][:2]), 2)


def test_a_missing_row_is_reported_and_only_its_sequence_goes_without():
    c = make([2, 3, 1], 300, F32, True, seed=91)
    good, n = run(c, 3)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out, m = run(dict(c, target=c["target"][:-1]), 3, status=status)
    assert status.item() == _lib.DEV_BAD_LENGTH and torch.equal(out[:2], good[:2]) and torch.equal(m[:2], n[:2])
    assert (out[2] == -1).all() and m[2] == 0


@pytest.mark.parametrize("sampled", [True, False])
def test_padded_drafts_need_no_target_rows(sampled):
    """A captured step has room for the longest spans; what lies behind draft_start's end is not looked at."""
    c = make([2, 0, 3], 1000, F32, sampled, seed=92)
    good, n = run(c, 3)
    pad = dict(c, tokens=torch.cat((c["tokens"], torch.full((4,), -7, device="cuda"))), accept=torch.cat((c["accept"], torch.full((4,), float("nan"), device="cuda"))),
               draft=None if c["draft"] is None else torch.cat((c["draft"], torch.full((4, 1000), float("nan"), device="cuda"))))
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out, m = run(pad, 3, status=status)
    assert status.item() == 0 and torch.equal(out, good) and torch.equal(m, n)


@pytest.mark.parametrize("dtype, vocab", [(F32, 5000), (BF16, 4099), (F16, 8192)])
@pytest.mark.parametrize("batch", [74, 75, 100, 148, 149, 296, 297])
def test_batches_around_the_launch_forms(dtype, vocab, batch):
    g = torch.Generator().manual_seed(batch)
    check(make(torch.randint(0, 5, (batch,), generator=g).tolist(), vocab, dtype, batch % 2 == 0, seed=batch), 4)
