"""CPU tests of how flags are aligned with a call's leading axes under vmap."""
import pytest
import torch

from jaxrwkv_b200.rwkv7 import _vmap_flags


@pytest.mark.parametrize("n", [2, 3])
@pytest.mark.parametrize("dim", [0, 1])
def test_flags_of_instances_go_to_their_own(n, dim):
    B1, B2, T = 2, 3, 4
    per = torch.arange(n * T).reshape(n, T)                                  # one row of flags an instance
    _, starts = _vmap_flags(None, per if dim == 0 else per.t(), (None, dim), 2)
    got = starts.expand(n, B1, B2, T)
    for i in range(n):
        assert torch.equal(got[i], per[i].expand(B1, B2, T))
    length, _ = _vmap_flags(torch.arange(n), None, (0, None), 2)
    assert torch.equal(length.expand(n, B1, B2), torch.arange(n)[:, None, None].expand(n, B1, B2))
    part, _ = _vmap_flags(torch.arange(n * B2).reshape(n, B2), None, (0, None), 2)
    assert torch.equal(part.expand(n, B1, B2)[:, 1], torch.arange(n * B2).reshape(n, B2))


def test_flags_that_are_shared_stay_as_they_are():
    starts = torch.zeros(4)
    assert _vmap_flags(7, starts, (None, None), 2) == [7, starts]
    full = torch.zeros(3, 2, 4)
    assert _vmap_flags(None, full, (None, 0), 1)[1].shape == (3, 2, 4)
