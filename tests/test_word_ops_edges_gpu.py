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


@pytest.mark.parametrize("rows,V", [(20, 70), (8, 140000), (300, 3500), (2100, 1000)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_bad_teacher_slot_makes_the_whole_row_nan(rows, V, dtype):
    """NaN or +inf among a row's used slots, or a used word outside the vocabulary, however small its weight: loss and
    every element of the gradient NaN; the same in empty slots and masked rows: no trace, and none in other rows."""
    g = torch.Generator(device="cuda").manual_seed(rows)
    x = torch.randn(rows, V, generator=g, device="cuda").to(dtype)
    ids = torch.randint(0, V, (rows, 5), generator=g, device="cuda")
    w = torch.randn(rows, 5, generator=g, device="cuda")
    good_ids, good_w = ids.clone(), w.clone()
    w[0, 2] = float("nan")
    w[1, 4] = float("inf")
    w[2] = float("inf")
    ids[3, 1] = V
    ids[4, 1], w[4, 1] = V + 5, -1000.0                       # 2^-1443 of the weight
    ids[5, 0], w[5, 0] = -1, float("nan")
    good_ids[5, 0] = -1
    ids[6, 3], w[6, 3] = 2 ** 40, float("-inf")
    good_ids[6, 3] = -1
    w[7, 0] = float("nan")
    mask = torch.ones(rows, dtype=torch.bool, device="cuda")
    mask[7] = False
    out = []
    for i, t in ((ids, w), (good_ids, good_w)):
        leaf = x.clone().requires_grad_()
        loss = word_ops.distill_loss(leaf, i, t, temperature=1.5, mask=mask)
        dx, = torch.autograd.grad([loss], [leaf], [torch.ones_like(loss)])
        out.append((loss.detach(), dx))
    (loss, dx), (want, want_dx) = out
    assert bool(loss[:5].isnan().all()) and bool(dx[:5].isnan().all())
    assert torch.equal(loss[5:], want[5:]) and torch.equal(dx[5:], want_dx[5:])
    assert bool(want.isfinite().all()) and loss[7].item() == 0 and bool((dx[7] == 0).all())


def _negated_view(t):
    """A real tensor of t's values whose memory holds their negatives."""
    v = torch.complex(torch.zeros_like(t), -t).conj().imag
    assert v.is_neg() and torch.equal(v, t)
    return v


def test_lazily_negated_tensors():
    """The imaginary part of a conjugated tensor (its sign is applied when it is read) in every place."""
    g = torch.Generator(device="cuda").manual_seed(4)
    n = lambda *s: torch.randn(*s, generator=g, device="cuda")                  # noqa: E731
    x, w, table = n(6, 90), n(6, 3), n(90, 8)
    t = torch.randint(0, 90, (6,), generator=g, device="cuda")
    ids = torch.randint(0, 90, (6, 3), generator=g, device="cuda")
    up, up_y = n(6), n(6, 8)
    got, want = [], []
    for out, f in ((want, lambda v: v), (got, _negated_view)):
        for train in (False, True):
            a = f(x).detach().requires_grad_(train)
            # (columns beside each other: every second float, as an imaginary part lies, is refused for a table)
            b = (table if f(x) is x else torch._neg_view(-table)).detach().requires_grad_(train)
            y = [word_ops.token_scores(a, t, top_k=4).logp, word_ops.distill_loss(a, ids, f(w)),
                 word_ops.embed_tokens(t, b, scale=2.0)]
            out += y
            if train:
                for o, leaf, u in zip(y, (a, a, b), (up, up, up_y)):
                    out += torch.autograd.grad([o], [leaf], [f(u)])
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    with pytest.raises(ValueError, match="adjacent"):
        word_ops.embed_tokens(t, _negated_view(table))
