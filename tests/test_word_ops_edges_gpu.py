"""scan2cap_amd.word_ops where results are known exactly or where one value decides a row.  U = 2^-24, half a
step of float32."""
import pytest
import torch

from tests import words_common  # noqa: F401  (first: the binding)
from scan2cap_amd import word_ops

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.mark.parametrize("T", [1.0, 2.0])
@pytest.mark.parametrize("rows,V", [(1, 3500), (3, 50001), (2, 65537), (300, 200003), (2100, 3500)])
def test_gradients_of_uniform_rows_carry_one_rounding(rows, V, T):
    """All logits equal: every 2^d is 1 and their sum V exactly, so that p = 1 / V carries the division's
    rounding alone, for upstream gradients and temperatures that are powers of two.  A probability formed as
    2^(d - log2 V) is up to 10 roundings off at these V."""
    x = torch.full((rows, V), 1.25, device="cuda", requires_grad=True)
    t = torch.full((rows,), 7, device="cuda")
    dx, = torch.autograd.grad([word_ops.token_scores(x, t, temperature=T).logp], [x], [torch.ones(rows, device="cuda")])
    want = torch.full((V,), -1.0 / V / T, dtype=torch.float64, device="cuda")
    want[7] += 1 / T
    assert bool(((dx.double() - want).abs() <= 2 * U * want.abs()).all())
    ids = torch.tensor([5, V - 1, 0, -1], device="cuda").expand(rows, 4)
    loss = word_ops.distill_loss(x, ids, torch.full((rows, 4), -2.0, device="cuda"), temperature=T)
    dx, = torch.autograd.grad([loss], [x], [torch.ones(rows, device="cuda")])
    want = torch.full((V,), 1.0 / V / T, dtype=torch.float64, device="cuda")
    want[ids[0, :3]] -= 1 / (3 * T)
    # the slots: a rounding of 1 / 3, one of the sum
    assert bool(((dx.double() - want).abs() <= 3 * U * want.abs()).all())
