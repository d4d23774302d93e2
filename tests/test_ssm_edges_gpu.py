"""Short convolution and selective scan at the edges of what their
documentation allows: every launch shape of the step, values that are not
numbers, offsets out of order, states that grow, the longest token axis."""

import pytest
import torch

import ssm_ref
import wkvm_b200 as wk
from wkvm_b200 import _lib, ops

pytestmark = pytest.mark.gpu

BF, FH, F32 = torch.bfloat16, torch.float16, torch.float32
NAMES = ("x", "dt", "A", "B", "C")


@pytest.mark.parametrize("T", [2 ** 26 + 7, 2 ** 31 - 1])
def test_scan_longest_token_axis(cuda, T):
    """One channel of as many tokens as an int32 counts, the inputs repeated by
    a stride of 0: the state settles where x delta / (1 - e^-delta) has it."""
    one = torch.ones(1, 1, 1, device=cuda, dtype=BF)
    row = torch.ones(1, 1, 8, device=cuda, dtype=BF).expand(1, T, 8)
    o, ht = wk.selective_scan(one.expand(1, T, 1), (0.5 * one).expand(1, T, 1), -torch.ones(1, 8, device=cuda), row, row,
                              dt_softplus=False, output_final_state=True)
    h = 0.5 / (1 - torch.tensor(-0.5, dtype=torch.float64).exp().item())
    # 1 / (1 - e^-1/2) < 3 roundings of 2^-22 settle; the output's own half step
    assert (ht.double() - h).abs().max().item() <= 3 * 2.0 ** -22 * h
    rest = o[0, 60:, 0]  # e^-30 of the empty start
    assert rest.min() == rest.max() and abs(rest[0].item() - 8 * h) <= (2.0 ** -8 + 2.0 ** -19) * 8 * h
    assert abs(o[0, 0, 0].item() - 4) <= 2.0 ** -8 * 4
