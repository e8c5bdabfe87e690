"""The caption losses around the word operators where a call goes wrong easily."""
import pytest
import torch

from tests import words_common  # noqa: F401  (first: the binding)
from tests.test_word_paths import DEVICES, _losses
from scan2cap_amd import loss_helper as lh


@pytest.mark.parametrize("device", DEVICES)
def test_a_teacher_in_the_students_dict_is_refused(device):
    dd, teacher = _losses(device)
    own = dict(dd)
    for wrong in (own, dict(lang_cap=own["lang_cap"])):
        with pytest.raises(ValueError, match="dict of its own"):
            lh.attach_teacher(own, wrong, top_k=4)
    assert "teacher_top_ids" not in own
    # a teacher that ran first, for a student that has not run yet
    early = {k: v for k, v in dd.items() if k != "lang_cap"}
    lh.attach_teacher(early, teacher, top_k=4)
    late = lh.attach_teacher(dict(dd), teacher, top_k=4)
    assert torch.equal(early["teacher_top_ids"], late["teacher_top_ids"])

INF, NAN = float("inf"), float("nan")


@pytest.mark.parametrize("device", DEVICES)
def test_rows_that_take_no_part_leave_no_trace(device):
    """Padding and bad boxes may hold NaN, slots may be empty by their logit, a student's row may be all -inf: the
    losses and gradients of the others are those of a batch without them."""
    dd, teacher = _losses(device)
    lh.attach_teacher(dd, teacher, top_k=6)
    ids, w, x = dd["teacher_top_ids"], dd["teacher_top_logits"], dd["lang_cap"]
    V = x.shape[-1]

    def both(x):
        leaf = x.clone().requires_grad_()
        d = dict(dd, lang_cap=leaf)
        kd = lh.compute_cap_distill_loss(d, temperature=2.0)
        total, words = lh.caption_log_likelihood(d)
        g1, = torch.autograd.grad(kd, leaf, retain_graph=True)
        g2, = torch.autograd.grad(total.sum(), leaf)
        return kd.detach(), words.detach(), g1, g2
    w[0, 2] = -INF                                    # no used slot
    w[0, 3, 2:] = -INF
    ids[0, 3, 4] = V + 3                              # in an empty slot
    want = both(x)
    assert all(bool(t.isfinite().all()) for t in want) and bool((want[2][0, 2] == 0).all())
    y = x.clone()
    y[1, 4:] = NAN                                    # padding
    got = both(y)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    y[2] = NAN                                        # a bad box: not distilled, but its words are scored
    got = both(y)
    assert torch.equal(got[0], want[0]) and torch.equal(got[2], want[2])
    # a row in which nothing can be said
    y = x.clone()
    y[0, 1] = -INF
    kd, words, g1, g2 = both(y)
    assert kd.item() == INF and words[0, 1].item() == -INF
    assert bool((g1[0, 1] == 0).all()) and bool((g2[0, 1] == 0).all())
    g1[0, 1], g2[0, 1] = want[2][0, 1], want[3][0, 1]
    assert torch.equal(g1, want[2]) and torch.equal(g2, want[3])


@pytest.mark.parametrize("device", DEVICES)
def test_a_teachers_nan_is_not_swallowed(device):
    dd, teacher = _losses(device)
    lh.attach_teacher(dd, teacher, top_k=6)
    dd["teacher_top_logits"][0, 0, 1] = NAN
    leaf = dd["lang_cap"].clone().requires_grad_()
    kd = lh.compute_cap_distill_loss(dict(dd, lang_cap=leaf))
    g, = torch.autograd.grad(kd, leaf)
    assert bool(kd.isnan()) and bool(g[0, 0].isnan().all()) and bool(g[0, 1:].isfinite().all())


@pytest.mark.parametrize("device", DEVICES)
def test_a_teacher_that_can_say_nothing_teaches_nothing(device):
    dd, teacher = _losses(device)
    teacher["lang_cap"][0, 0] = -INF
    lh.attach_teacher(dd, teacher, top_k=6)
    leaf = dd["lang_cap"].clone().requires_grad_()
    kd = lh.compute_cap_distill_loss(dict(dd, lang_cap=leaf))
    g, = torch.autograd.grad(kd, leaf)
    assert bool(kd.isfinite()) and bool((g[0, 0] == 0).all()) and bool(g.isfinite().all())
