"""GPU tests of sizes that the library's 32-bit counts do not hold: refused before anything is allocated for them (the operands are one element,
expanded)."""
import pytest
import torch

from jaxrwkv_b200 import _lib
from jaxrwkv_b200.gated_recurrence import gated_recurrence, gated_recurrence_step
from jaxrwkv_b200.group_norm import group_norm_act

pytestmark = pytest.mark.gpu


def test_counts_beyond_32_bits():
    one, state = torch.zeros(1, device="cuda", dtype=torch.bfloat16), torch.zeros(1, device="cuda")
    many = (1 << 32) + 1                    # 1 in 32 bits
    bad = [lambda: gated_recurrence(one.expand(many, 1, 1), one.expand(many, 1, 1), state.expand(many, 1)),
           lambda: gated_recurrence(one.expand(1, many, 1), one.expand(1, many, 1), state.expand(1, 1)),
           lambda: gated_recurrence(one.expand(1, 1, many), one.expand(1, 1, many), state.expand(1, many)),
           lambda: gated_recurrence_step(one.expand(many, 1), one.expand(many, 1), state.expand(many, 1)),
           lambda: gated_recurrence_step(one.expand(1, many), one.expand(1, many), state.expand(1, many)),
           lambda: group_norm_act(one.expand(1, many), None, None, many)]
    held = torch.cuda.memory_allocated()
    for call in bad:
        with pytest.raises(_lib.B200WKVError, match="32 bits"):
            call()
    assert torch.cuda.memory_allocated() == held


def test_a_step_without_channels():
    with pytest.raises(_lib.B200WKVError, match="channels"):
        gated_recurrence_step(*(torch.zeros((), device="cuda") for _ in range(3)))
