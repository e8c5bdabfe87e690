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


def _captioner(kind, vocabulary, embeddings):
    return _module(kind, "cpu", vocabulary, embeddings)


@pytest.mark.parametrize("kind", KINDS)
def test_learning_keeps_the_tables_storage(kind):
    """What holds the table's memory (a captured step) goes on reading the table."""
    _, vocabulary, embeddings = _batch("cpu")
    mod = _captioner(kind, vocabulary, embeddings)
    at, names = mod._emb_table.data_ptr(), [n for n, _ in mod.named_parameters()]
    assert mod.learn_word_embeddings() is mod
    assert mod._emb_table.data_ptr() == at and mod._emb_table.requires_grad
    assert sorted(n for n, _ in mod.named_parameters()) == sorted(names + ["_emb_table"])
    assert not dict(mod.named_buffers())


@pytest.mark.parametrize("kind", KINDS)
def test_state_dicts_load_with_and_without_learned_words(kind):
    _, vocabulary, embeddings = _batch("cpu")
    fresh, learned = (_captioner(kind, vocabulary, embeddings) for _ in range(2))
    learned.learn_word_embeddings()
    with torch.no_grad():
        for p in learned.parameters():
            p.add_(0.25)
    plain_state = {k: v.clone() for k, v in fresh.state_dict().items()}
    first_table = fresh._emb_table.clone()
    # learned -> fresh: learned from then on
    fresh.load_state_dict(learned.state_dict())
    assert isinstance(fresh._emb_table, torch.nn.Parameter)
    assert torch.equal(fresh._emb_table, first_table + 0.25)
    for k, v in learned.state_dict().items():
        assert torch.equal(fresh.state_dict()[k], v), k
    # not learned -> learned: the table stays, everything else is loaded
    learned.load_state_dict(plain_state)
    assert torch.equal(learned._emb_table, first_table + 0.25)
    for k, v in plain_state.items():
        assert torch.equal(learned.state_dict()[k], v), k
    # other keys are still required, and a table of another size is an error
    with pytest.raises(RuntimeError, match="classifier.bias"):
        learned.load_state_dict({k: v for k, v in plain_state.items() if k != "classifier.bias"})
    with pytest.raises(RuntimeError, match="_emb_table"):
        _captioner(kind, vocabulary, embeddings).load_state_dict(dict(plain_state, _emb_table=torch.zeros(3, 300)))


@pytest.mark.parametrize("kind", KINDS)
def test_checkpoints_with_learned_words(kind, tmp_path):
    """save_checkpoint / load_checkpoint between models that both learned the table, and the refusal, with nothing
    changed, where one did not."""
    from scan2cap_amd import checkpoint as ck
    _, vocabulary, embeddings = _batch("cpu")

    def made(learn):
        mod = _captioner(kind, vocabulary, embeddings)
        if learn:
            mod.learn_word_embeddings()
        opt = torch.optim.Adam(mod.parameters(), lr=1e-3)
        for p in mod.parameters():
            p.grad = torch.full_like(p, 0.5)
        return mod, opt
    for learn in (True, False):
        root = str(tmp_path / str(learn))
        mod, opt = made(learn)
        opt.step()
        ck.save_checkpoint(root, 3, mod, opt, {"best": 1.0})
        again, opt2 = made(learn)
        assert ck.load_checkpoint(root, again, opt2)[0] == 3
        for k, v in mod.state_dict().items():
            assert torch.equal(again.state_dict()[k], v), k
        assert len(opt2.state_dict()["state"]) == len(opt.state_dict()["state"])
        other, opt3 = made(not learn)
        before = {k: v.clone() for k, v in other.state_dict().items()}
        with pytest.raises(ValueError, match="learn_word_embeddings"):
            ck.load_checkpoint(root, other, opt3)
        assert other.state_dict().keys() == before.keys() and not opt3.state_dict()["state"]
        for k, v in before.items():
            assert torch.equal(other.state_dict()[k], v), k
