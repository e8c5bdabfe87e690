"""A captioner whose word embeddings are learned, on the CPU and the GPU."""
import pytest
import torch

from tests import plain_caption_common as pc
from tests import words_common  # noqa: F401  (first: the binding)
from tests.test_word_paths import DEVICES, _batch, _module

KINDS = ["plain", "topdown"]


def _table_gradient(mod, dd, w):
    mod.zero_grad(set_to_none=True)
    (mod(dict(dd))["lang_cap"] * w).sum().backward()
    return mod._emb_table.grad


@pytest.mark.parametrize("device", DEVICES)
@pytest.mark.parametrize("kind", KINDS)
def test_learned_words_are_looked_up_beside_lang_feat(kind, device):
    """A batch that brings `lang_feat` too trains the table and decodes as one that does not."""
    dd, vocabulary, embeddings = _batch(device)
    mod = _module(kind, device, vocabulary, embeddings)
    mod.learn_word_embeddings()
    with torch.no_grad():
        mod._emb_table.mul_(1.5)
    without = {k: v for k, v in dd.items() if k != "lang_feat"}
    w = torch.randn(pc.B, pc.T - 1, pc.V, generator=torch.Generator().manual_seed(1)).to(device)
    want = _table_gradient(mod, without, w)
    assert float(want.abs().max()) > 0
    got = _table_gradient(mod, dd, w)
    # on the GPU the recurrent kernels' two runs may differ where they accumulate (1e-6 of the largest entry)
    assert float((got - want).abs().max()) <= 1e-6 * float(want.abs().max())
    mod.eval()
    with torch.no_grad():
        a, b = (mod(dict(d), use_tf=False, is_eval=True, max_len=5)["lang_cap"] for d in (dd, without))
    assert torch.equal(a, b)


@pytest.mark.parametrize("kind", KINDS)
def test_words_need_ids_or_features(kind):
    dd, vocabulary, embeddings = _batch("cpu")
    mod = _module(kind, "cpu", vocabulary, embeddings)
    feat_only = {k: v for k, v in dd.items() if k != "lang_ids"}
    mod(dict(feat_only))
    with pytest.raises(ValueError, match="no lang_ids"):
        mod({k: v for k, v in feat_only.items() if k != "lang_feat"})
    mod.learn_word_embeddings()
    with pytest.raises(ValueError, match="learned word embeddings"):
        mod(dict(feat_only))


def _annotations(device, dd, feat):
    from scan2cap_amd.scene_builder import AnnotationTable
    n = pc.B
    return AnnotationTable(device, dd["lang_feat"].cpu().numpy() if feat else None, dd["lang_ids"].cpu().numpy(),
                           dd["lang_len"].cpu().numpy(), [4] * n, [0] * n, [2] * n, [0] * n)


@pytest.mark.parametrize("device", DEVICES)
def test_annotations_without_features_feed_the_captioner(device):
    dd, vocabulary, embeddings = _batch(device)
    mod = _module("topdown", device, vocabulary, embeddings)
    picks = [1, 0]
    with_feat, without = (_annotations(device, dd, feat).gather(picks) for feat in (True, False))
    assert set(with_feat) - set(without) == {"lang_feat"}
    for k in without:
        assert torch.equal(with_feat[k], without[k])
    rest = {k: v for k, v in dd.items() if not k.startswith("lang_")}
    a, b = (mod(dict(rest, **batch))["lang_cap"] for batch in (with_feat, without))
    assert torch.equal(a, b)


def test_a_feeder_leaves_no_stale_features():
    from scan2cap_amd.scene_builder import BatchFeeder
    dd, _, _ = _batch("cpu")
    anns = _annotations("cpu", dd, False)
    with pytest.raises(ValueError, match="stale"):
        BatchFeeder(None, anns, [{"lang_ids": dd["lang_ids"]}, dict(dd)], stream=object())
    BatchFeeder(None, anns, [{"lang_ids": dd["lang_ids"]}], stream=object())
    BatchFeeder(None, _annotations("cpu", dd, True), [dict(dd)], stream=object())
