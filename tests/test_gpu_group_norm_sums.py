"""GPU tests of the group norm's parameter gradients over many rows: what one thread adds up row after row."""
import pytest
import torch

from jaxrwkv_b200.group_norm import group_norm_act

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


# teams of lanes with one piece and two, of any size, added up within a thread block, single channels, whole thread blocks
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,G,D", [(32768, 32, 64), (32768, 9, 64), (90000, 2, 16), (32768, 12, 80), (32768, 4, 333), (32768, 4, 512), (32768, 1, 2048)])
def test_small_terms_behind_large_ones(rows, G, D, dtype):
    """db is the sum of gy where there is neither gate nor activation: 1024 ones, and behind them terms that vanish in a running 32-bit
    sum of 1.  Allowed are 16 rows a running sum (15 roundings), its own rounding and the result's, each of U times the
    terms' magnitudes.  dw is the same sum with signs, its terms off by x's normalisation too (a reciprocal root of 2 ulp, a product)."""
    small, C = 0.75 * U, G * D
    gy = torch.full((rows, C), small, device="cuda", dtype=dtype)
    gy[:1024] = 1.0
    x = torch.ones(rows, C, device="cuda", dtype=dtype)
    x[:, 1::2] = -1.0                       # of mean 0 and variance 1 where D is even
    weight, bias = torch.ones(C, device="cuda").requires_grad_(True), torch.zeros(C, device="cuda").requires_grad_(True)
    dw, db = torch.autograd.grad(group_norm_act(x, weight, bias, G, activation="none", eps=0.0), (weight, bias), gy)
    total = 1024 + (rows - 1024) * small
    assert ((db.double() - total).abs() <= 17 * U * total).all(), (db.double() / total - 1).abs().max() / U
    if D % 2 == 0:
        assert ((dw.double() - total * x[0].double()).abs() <= (17 + 4 + 1) * U * total).all()


def test_infinite_terms():
    """A sum that is infinite stays so, whichever row of many makes it that, and one that has no value has none."""
    rows, C = 40000, 128
    for at in (0, 300, 20000, 39999):
        gy = torch.ones(rows, C, device="cuda")
        gy[at, 3], gy[at, 4], gy[at, 5] = float("inf"), float("-inf"), float("nan")
        gy[:, 6] = 3e38
        bias = torch.zeros(C, device="cuda").requires_grad_(True)
        db, = torch.autograd.grad(group_norm_act(torch.zeros(rows, C, device="cuda"), None, bias, 32, activation="none"), bias, gy)
        assert db[3] == float("inf") and db[4] == float("-inf") and db[5].isnan() and db[6] == float("inf")
        rest = [c for c in range(C) if c not in (3, 4, 5, 6)]
        assert (db[rest] == rows).all()
