"""Operators around the captioner's word logits, forward and backward, on the hand-written kernels of
csrc/s2c_vocab.hip and csrc/s2c_embed.hip (C ABI: include/s2c_words.h; torch binding:
csrc/s2c_words_torch.cpp):

    token_scores   log probabilities of given words, entropy, the best alternatives
    distill_loss   KL divergence from a teacher's top logits to the softmax over the whole vocabulary
    embed_tokens   embedding lookup with scaling, and the table's gradient summed by sorted words

Logits and tables may be float32, bfloat16 or float16; statistics, sums and losses are float32, gradients
come in their input's type, rounded once.  Work is enqueued on the current stream of the tensors' device,
nothing synchronises, scratch memory is allocated per call.  Arguments that the kernels do not take are
refused with ValueError (shapes, types, ranges) or RuntimeError (CPU tensors: there is no fallback).
Values that live on the device cannot be refused without a synchronisation: a word index outside the
vocabulary is never used as an address and turns its row's results into NaN.

Everything may be captured into a graph and replayed.  A backward pass is captured while no eager graph of
the same leaves is alive (drop its outputs first): torch would synchronise the leaves' own stream inside
the capture, which it does not survive.  Second derivatives and forward-mode tangents are refused.
"""
import collections
import importlib.machinery
import importlib.util
import os

import torch

from . import _C
from . import build as _build

MAX_TOP = 64             # S2C_WORDS_MAX_TOP
MAX_SLOTS = 256          # S2C_WORDS_MAX_SLOTS
MAX_DIM = 1 << 24        # S2C_WORDS_MAX_DIM

TokenScores = collections.namedtuple("TokenScores", "logp entropy top_logp top_ids")


def _load():
    if not os.path.exists(_build.EXT_PATH):
        raise _C.S2CError("s2c_words_ext.so not found at %s -- run `python -m scan2cap_amd.build` (there is no "
                          "fallback for the word operators)" % _build.EXT_PATH)
    loader = importlib.machinery.ExtensionFileLoader("s2c_words_ext", _build.EXT_PATH)
    module = importlib.util.module_from_spec(importlib.util.spec_from_loader("s2c_words_ext", loader))
    loader.exec_module(module)
    return module


_ext = _load()


def _refuse(numbers, **tensors):
    """After a TypeError of the binding: say which argument is no tensor, or what the other arguments are."""
    for name, t in tensors.items():
        if not torch.is_tensor(t):
            raise ValueError("%s must be a tensor, not %s" % (name, type(t).__name__)) from None
    raise ValueError("numbers of a wrong type or out of range: %r" % (numbers,)) from None


def _given(**tensors):
    return {name: t for name, t in tensors.items() if t is not None}


def token_scores(logits, tokens=None, top_k=0, temperature=1.0, ignore_index=None):
    """Scores of words under p = softmax(logits / temperature), in one pass over the logits.

    logits (..., V): any leading axes.  tokens (...): the words to score, int64 or int32, or None.
    -> TokenScores(logp, entropy, top_logp, top_ids):
      logp (...) float32        log p[tokens]                                    (None without tokens)
      entropy (...) float32     -sum p log p
      top_logp (..., top_k)     log p of the top_k <= 64 largest logits, descending    (None if top_k is 0)
      top_ids (..., top_k)      their indices (int64); equal logits in ascending index order
    All but top_ids are differentiable with respect to the logits.

    Rows whose token equals `ignore_index` (padding) are not read: logp = entropy = top_logp = 0, top_ids
    = -1 (an empty slot of `distill_loss`), zero gradient.  Logits of -inf are words that cannot be said;
    a row of nothing else has logp -inf, entropy 0 and zero gradient.  A token outside [0, V) makes logp
    and the row's gradient NaN, as a logit of NaN or +inf does to everything in its row."""
    try:
        return TokenScores._make(_ext.token_scores(logits, tokens, top_k, temperature, ignore_index))
    except TypeError:
        _refuse(dict(top_k=top_k, temperature=temperature, ignore_index=ignore_index), logits=logits,
                **_given(tokens=tokens))


def distill_loss(logits, teacher_ids, teacher_logits, temperature=1.0, mask=None):
    """KL(q || p) of every row, float32 (...): q = the teacher's softmax over its K <= 256 slots
    (teacher_ids, teacher_logits) (..., K) at `temperature`, p = softmax(logits / temperature) over all V
    words.  Differentiable with respect to `logits`; the teacher is a constant.  (Hinton's factor
    temperature^2 is the caller's.)

    Log probabilities serve as teacher logits as well (`token_scores(...).top_ids / .top_logp` of the
    teacher).  A slot with a negative id or a logit of -inf is empty; an id may occur twice.  Rows with
    mask (..., bool) False are not read; they and rows without a used slot have loss 0 and zero gradient.
    A used slot with an id >= V (whatever its weight) or a logit of NaN or +inf makes the row's loss and whole
    gradient NaN; a row of logits that are all -inf has loss +inf and zero gradient."""
    try:
        return _ext.distill_loss(logits, teacher_ids, teacher_logits, temperature, mask)
    except TypeError:
        _refuse(dict(temperature=temperature), logits=logits, teacher_ids=teacher_ids, teacher_logits=teacher_logits,
                **_given(mask=mask))


def embed_tokens(tokens, table, scale=1.0, padding_idx=None):
    """scale * table[tokens]: tokens (...) int64 or int32, table (V, D) with adjacent columns (rows may be
    strided) -> (..., D) of the table's type.  Tokens equal to `padding_idx` (any integer but int64's lowest,
    in the table or not) give zeros and no gradient; a token outside [0, V) gives a row of NaN and no
    gradient.  The table's gradient is dense, summed in float32 over each word's places in their order (the
    same bits every time)."""
    try:
        return _ext.embed_tokens(tokens, table, scale, padding_idx)
    except TypeError:
        _refuse(dict(scale=scale, padding_idx=padding_idx), tokens=tokens, table=table)
