"""The word operators where the framework calls them: word embeddings from `lang_ids`, a trainable embedding
table, caption distillation and caption likelihoods, on the CPU (the plain formulas) and the GPU (the kernels),
against float64."""
import numpy as np
import pytest
import torch

from tests import golden_common as gc
from tests import plain_caption_common as pc
from tests import words_common  # noqa: F401  (first: the binding)

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
U = 2.0 ** -24


def _batch(device, seed=3):
    vocabulary, embeddings = gc.vocab_and_embeddings(pc.V)
    dd = {k: torch.from_numpy(v) for k, v in pc.make_inputs(embeddings, vocabulary, seed).items()}
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(4, pc.V, (pc.B, pc.T + 1), generator=g)
    ids[1, pc.T - 2:] = 0
    table = torch.from_numpy(np.stack([embeddings[vocabulary["idx2word"][str(i)]] for i in range(pc.V)])).float()
    dd.update(lang_ids=ids, lang_feat=table[ids] * (ids != 0).unsqueeze(-1), _num_words=pc.T,
              bbox_mask=torch.ones(pc.B, pc.K))
    return {k: v.to(device) if torch.is_tensor(v) else v for k, v in dd.items()}, vocabulary, embeddings


def _module(kind, device, vocabulary, embeddings):
    from scan2cap_amd.models import caption_module as cm
    torch.manual_seed(5)
    cls = cm.TopDownSceneCaptionModule if kind == "topdown" else cm.SceneCaptionModule
    return cls(vocabulary, embeddings, 300, 128, 512, pc.K).to(device).train()


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("kind", ["plain", "topdown"])
def test_word_embeddings_from_ids_are_the_callers(kind, device):
    dd, vocabulary, embeddings = _batch(device)
    mod = _module(kind, device, vocabulary, embeddings)
    without = {k: v for k, v in dd.items() if k != "lang_feat"}
    assert torch.equal(mod(dict(dd))["lang_cap"], mod(without)["lang_cap"])
    mod.eval()
    with torch.no_grad():
        a, b = (mod(dict(d), use_tf=False, is_eval=True, max_len=5)["lang_cap"] for d in (dd, without))
    assert torch.equal(a, b)


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("kind", ["plain", "topdown"])
def test_learned_word_embeddings_take_the_gradient(kind, device):
    """d loss / d table = the sum of d loss / d lang_feat over each word's places, none at padding."""
    dd, vocabulary, embeddings = _batch(device)
    mod = _module(kind, device, vocabulary, embeddings)
    feat = dd["lang_feat"].clone()[:, :pc.T - 1].requires_grad_()
    w = torch.randn(pc.B, pc.T - 1, pc.V, generator=torch.Generator().manual_seed(1)).to(device)
    (mod(dict(dd, lang_feat=feat))["lang_cap"] * w).sum().backward()
    assert "_emb_table" not in mod.state_dict()
    mod.learn_word_embeddings()
    mod.learn_word_embeddings()
    assert "_emb_table" in mod.state_dict() and isinstance(mod._emb_table, torch.nn.Parameter)
    without = {k: v for k, v in dd.items() if k != "lang_feat"}
    (mod(without)["lang_cap"] * w).sum().backward()
    ids = dd["lang_ids"][:, :pc.T - 1]
    want = torch.zeros(pc.V, 300, dtype=torch.float64, device=device)
    live = (ids != 0).unsqueeze(-1)
    want.index_add_(0, ids.reshape(-1), (feat.grad.double() * live).reshape(-1, 300))
    size = torch.zeros_like(want).index_add_(0, ids.reshape(-1), feat.grad.double().abs().reshape(-1, 300))
    # at most 18 places to a word: one rounding an addition, and on the GPU the recurrent kernels' two runs may
    # differ where they accumulate (1e-6 of the largest entry)
    tol = 20 * U * size + 1e-6 * float(want.abs().max())
    assert bool(((mod._emb_table.grad.double() - want).abs() <= tol).all())
    assert bool((mod._emb_table.grad[0] == 0).all())


def _losses(device, seed=7):
    g = torch.Generator().manual_seed(seed)
    B, T, V = 3, 8, 50
    ids = torch.randint(1, V, (B, T), generator=g)
    ids[1, 5:] = 0
    dd = dict(lang_cap=torch.randn(B, T - 1, V, generator=g) * 2, lang_ids=ids, lang_len=torch.tensor([8, 5, 8]),
              good_bbox_masks=torch.tensor([True, True, False]))
    teacher = dict(lang_cap=torch.randn(B, T - 1, V, generator=g) * 2)
    return [{k: v.to(device) for k, v in d.items()} for d in (dd, teacher)]


@pytest.mark.parametrize("device", DEVICES)
def test_caption_distillation(device):
    from scan2cap_amd import loss_helper as lh
    dd, teacher = _losses(device)
    dd["lang_cap"].requires_grad_()
    lh.attach_teacher(dd, teacher, top_k=6)
    assert dd["teacher_top_ids"].shape == (3, 7, 6) and not dd["teacher_top_logits"].requires_grad
    loss = lh.compute_cap_distill_loss(dd, temperature=2.0)
    g, = torch.autograd.grad(loss, dd["lang_cap"])
    x = dd["lang_cap"].detach().double().requires_grad_()
    top, at = torch.sort(teacher["lang_cap"].double(), dim=-1, descending=True, stable=True)
    assert torch.equal(at[..., :6], dd["teacher_top_ids"])
    q = torch.softmax(top[..., :6] / 2, -1)
    kl = (q * (q.log() - torch.log_softmax(x / 2, -1).gather(-1, at[..., :6]))).sum(-1)
    rows = (dd["lang_ids"][:, 1:] != 0) & dd["good_bbox_masks"].unsqueeze(1)
    want = 4 * (kl * rows).sum() / rows.sum()
    gw, = torch.autograd.grad(want, x)
    # sums of a few float32 terms of size 1 .. 10
    assert abs(float(loss.detach()) - float(want.detach())) <= 1e-5 * float(want.detach())
    assert float((g.double() - gw).abs().max()) <= 1e-5 * float(gw.abs().max())
    assert bool((g[2] == 0).all()) and bool((g[1, 4:] == 0).all())
    # empty slots
    dd["teacher_top_ids"][0, 0, 3:] = -1
    dd["teacher_top_ids"][0, 1] = -1
    q0 = torch.softmax(top[0, 0, :3] / 2, -1)
    kl0 = (q0 * (q0.log() - torch.log_softmax(x[0, 0] / 2, -1)[at[0, 0, :3]])).sum()
    want = want + 4 * (kl0 - kl[0, 0] - kl[0, 1]) / rows.sum()
    got = lh.compute_cap_distill_loss(dd, temperature=2.0)
    assert abs(float(got.detach()) - float(want.detach())) <= 1e-5 * float(want.detach())


@pytest.mark.parametrize("device", DEVICES)
def test_caption_log_likelihood(device):
    from scan2cap_amd import loss_helper as lh
    dd, _ = _losses(device)
    total, words = lh.caption_log_likelihood(dd, temperature=0.8)
    t = dd["lang_ids"][:, 1:]
    want = torch.log_softmax(dd["lang_cap"].double() / 0.8, -1).gather(-1, t.unsqueeze(-1)).squeeze(-1) * (t != 0)
    assert float((words.double() - want).abs().max()) <= U * 400
    assert float((total.double() - want.sum(-1)).abs().max()) <= U * 400 * 7
    with pytest.raises(ValueError, match="stale"):
        lh.caption_log_likelihood(dict(dd, _num_words=5))
    with pytest.raises(ValueError, match="stale"):
        lh.compute_cap_distill_loss(dict(dd, _num_words=1))


@pytest.mark.parametrize("device", DEVICES)
def test_distillation_joins_the_scene_loss(device, monkeypatch):
    """`distill` adds its share to the total and to the part that flows through the captioner, and 0 leaves
    everything as it was."""
    from scan2cap_amd import loss_helper as lh
    dd, teacher = _losses(device)
    lh.attach_teacher(dd, teacher, top_k=6)
    zero = torch.zeros((), device=device)
    det = dict(vote_loss=zero + 1, objectness_loss=zero + 2, box=zero, sem=zero + 3)
    B, K = 3, 4
    dd["objectness_scores"] = torch.zeros(B, K, 2, device=device)
    monkeypatch.setattr(lh.loss_fused, "available", lambda d: False)
    monkeypatch.setattr(lh, "compute_vote_loss", lambda d: det["vote_loss"])
    lab = torch.ones(B, K, dtype=torch.int64, device=device)
    monkeypatch.setattr(lh, "compute_objectness_loss", lambda d: (det["objectness_loss"], lab, lab.float(), lab))
    monkeypatch.setattr(lh, "compute_box_and_sem_cls_loss", lambda d, c: (zero,) * 5 + (det["sem"],))
    plain = lh.get_scene_cap_loss(dict(dd), device, None, None)
    assert "distill_loss" not in plain
    both = lh.get_scene_cap_loss(dict(dd), device, None, None, distill=0.5, distill_temperature=3.0)
    kd = lh.compute_cap_distill_loss(dd, 3.0)
    assert torch.equal(both["distill_loss"], kd)
    assert float(both["loss"]) == pytest.approx(float(plain["loss"]) + 0.5 * float(kd), rel=1e-6)
    assert float(both["_loss_det"] + both["_loss_rest"]) == pytest.approx(float(both["loss"]), rel=1e-6)
