"""scan2cap_amd.word_ops on the CPU: what it refuses, at the Python entry points and at the C ABI (whose
checks run on the host before any launch)."""
import ctypes
import os
import re

import pytest
import torch

from tests import words_common  # noqa: F401  (first: the binding)
from scan2cap_amd import _C, word_ops

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_I, _LL, _F, _P = ctypes.c_int, ctypes.c_longlong, ctypes.c_float, ctypes.c_void_p


class _Logits(ctypes.Structure):
    _fields_ = [("rows", _I), ("V", _I), ("dtype", _I), ("n1", _I), ("n2", _I), ("inv_t", _F),
                ("s0", _LL), ("s1", _LL), ("s2", _LL), ("x", _P)]


class _ScoresArgs(ctypes.Structure):
    _fields_ = [("lg", _Logits), ("k", _I), ("has_ignore", _I), ("ignore", _LL), ("token", _P),
                ("logp", _P), ("entropy", _P), ("top_logp", _P), ("top_ids", _P), ("stats", _P),
                ("ws", _P)]


class _DistillArgs(ctypes.Structure):
    _fields_ = [("lg", _Logits), ("K", _I), ("teacher_dtype", _I), ("ids", _P), ("teacher", _P),
                ("mask", _P), ("loss", _P), ("stats", _P), ("ws", _P)]


def _lib():
    lib = _C.load()
    for name, types in (("s2c_token_scores_fwd", [_P, _P]), ("s2c_token_scores_bwd", [_P] * 6),
                        ("s2c_distill_fwd", [_P, _P]), ("s2c_distill_bwd", [_P] * 4),
                        ("s2c_embed_fwd", [_LL, _I, _I, _I, _LL, _P, _P, _F, _LL, _P, _P]),
                        ("s2c_embed_grad", [_LL, _I, _I, _I, _LL, _P, _P, _F, _LL, _P, _P, _P])):
        getattr(lib, name).argtypes, getattr(lib, name).restype = types, _I
    return lib


def _x(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype)


def _i(*shape, dtype=torch.int64):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("call", [
    lambda: word_ops.token_scores(_x(2, 5, dtype=torch.float64), _i(2)),
    lambda: word_ops.token_scores(_i(2, 5), _i(2)),
    lambda: word_ops.token_scores(torch.tensor(1.0), _i(1)),
    lambda: word_ops.token_scores(_x(2, 0), _i(2)),
    lambda: word_ops.token_scores([[0.0]], _i(1)),
    lambda: word_ops.token_scores(_x(2, 5), _x(2)),
    lambda: word_ops.token_scores(_x(2, 5), _i(3)),
    lambda: word_ops.token_scores(_x(2, 5), _i(1)),
    lambda: word_ops.token_scores(_x(2, 5), _i(2, dtype=torch.bool)),
    lambda: word_ops.token_scores(_x(2, 5), _i(2), top_k=6),
    lambda: word_ops.token_scores(_x(2, 500), _i(2), top_k=65),
    lambda: word_ops.token_scores(_x(2, 5), _i(2), top_k=-1),
    lambda: word_ops.token_scores(_x(2, 5), _i(2), temperature=0.0),
    lambda: word_ops.token_scores(_x(2, 5), _i(2), temperature=-1.0),
    lambda: word_ops.token_scores(_x(2, 5), _i(2), temperature=float("nan")),
    lambda: word_ops.token_scores(_x(2, 5), _i(2), temperature=float("inf")),
    lambda: word_ops.token_scores(_x(2, 5), _i(2), temperature=1e-40),
    lambda: word_ops.token_scores(_x(2, 5), ignore_index=0),
    lambda: word_ops.distill_loss(_x(2, 5), _i(2), _x(2)),
    lambda: word_ops.distill_loss(_x(2, 5), _i(2, 3), _x(2, 4)),
    lambda: word_ops.distill_loss(_x(2, 5), _i(3, 3), _x(3, 3)),
    lambda: word_ops.distill_loss(_x(2, 5), _i(2, 0), _x(2, 0)),
    lambda: word_ops.distill_loss(_x(2, 500), _i(2, 257), _x(2, 257)),
    lambda: word_ops.distill_loss(_x(2, 5), _x(2, 3), _x(2, 3)),
    lambda: word_ops.distill_loss(_x(2, 5), _i(2, 3), _i(2, 3)),
    lambda: word_ops.distill_loss(_x(2, 5), _i(2, 3), _x(2, 3).requires_grad_()),
    lambda: word_ops.distill_loss(_x(2, 5), _i(2, 3), _x(2, 3), mask=_i(2)),
    lambda: word_ops.distill_loss(_x(2, 5), _i(2, 3), _x(2, 3), mask=_i(3, dtype=torch.bool)),
    lambda: word_ops.distill_loss(_x(2, 5), _i(2, 3), _x(2, 3), temperature=0),
    lambda: word_ops.embed_tokens(_i(3), _x(4, 5, dtype=torch.float64)),
    lambda: word_ops.embed_tokens(_i(3), _x(4)),
    lambda: word_ops.embed_tokens(_i(3), _x(0, 4)),
    lambda: word_ops.embed_tokens(_x(3), _x(4, 5)),
    lambda: word_ops.embed_tokens(_i(3), _x(5, 4).t()),
    lambda: word_ops.embed_tokens(_i(3), _x(4, 5), scale=float("inf")),
    lambda: word_ops.embed_tokens([1], _x(4, 5)),
])
def test_refused_arguments(call):
    with pytest.raises(ValueError):
        call()


@pytest.mark.parametrize("call", [
    lambda: word_ops.token_scores(_x(2, 5), _i(2)),
    lambda: word_ops.distill_loss(_x(2, 5), _i(2, 3), _x(2, 3)),
    lambda: word_ops.embed_tokens(_i(3), _x(4, 5)),
])
def test_cpu_tensors_are_refused(call):
    with pytest.raises(RuntimeError, match="CPU not supported"):
        call()


def test_limits_are_the_headers():
    txt = open(os.path.join(ROOT, "include", "s2c_words.h")).read()
    get = lambda n: eval(re.search(r"#define %s +(.+?) */\*" % n, txt).group(1))   # noqa: E731,S307
    assert get("S2C_WORDS_MAX_TOP") == word_ops.MAX_TOP
    assert get("S2C_WORDS_MAX_SLOTS") == word_ops.MAX_SLOTS
    assert get("S2C_WORDS_MAX_DIM") == word_ops.MAX_DIM


def test_argument_structs_follow_the_header():
    txt = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "s2c_words.h")).read(), flags=re.S)
    structs = dict((n, b) for b, n in re.findall(r"typedef struct \{(.*?)\} (\w+);", txt, flags=re.S))
    for name, cls in (("s2c_logits", _Logits), ("s2c_token_scores_args", _ScoresArgs),
                      ("s2c_distill_args", _DistillArgs)):
        fields = []
        for decl in structs[name].split(";"):
            if decl.strip():
                fields += [re.sub(r"\W", "", v.split()[-1]) for v in decl.split(",")]
        assert fields == [f[0] for f in cls._fields_], name
    lib = _C.load()
    lib.s2c_words_args_sizeof.argtypes = [ctypes.c_int]
    lib.s2c_words_args_sizeof.restype = ctypes.c_longlong
    for i, cls in enumerate((_Logits, _ScoresArgs, _DistillArgs)):
        assert lib.s2c_words_args_sizeof(i) == ctypes.sizeof(cls)


EINVAL = -1
P = 1 << 20          # an address that no check may follow


def _lg(**kw):
    d = dict(rows=2, V=8, dtype=0, n1=1, n2=2, inv_t=1.0, s0=0, s1=0, s2=8, x=P)
    d.update(kw)
    return _Logits(**d)


@pytest.mark.parametrize("lg", [dict(rows=-1), dict(V=0), dict(V=-3), dict(dtype=3), dict(dtype=-1), dict(n1=0),
                                dict(n2=0), dict(inv_t=0.0), dict(inv_t=-1.0), dict(inv_t=float("nan")),
                                dict(inv_t=float("inf")), dict(x=None), dict(x=P + 2), dict(x=P + 1, dtype=1)])
def test_c_entries_refuse_bad_logits(lg):
    lib = _lib()
    s = _ScoresArgs(_lg(**lg), 0, 0, 0, P, P, P, None, None, P, P)
    d = _DistillArgs(_lg(**lg), 3, 0, P, P, None, P, P, P)
    assert lib.s2c_token_scores_fwd(ctypes.addressof(s), None) == EINVAL
    assert lib.s2c_token_scores_bwd(ctypes.addressof(s), P, P, None, P, None) == EINVAL
    assert lib.s2c_distill_fwd(ctypes.addressof(d), None) == EINVAL
    assert lib.s2c_distill_bwd(ctypes.addressof(d), P, P, None) == EINVAL


def test_c_entries_refuse_bad_arguments():
    lib = _lib()
    scores = lambda **kw: _ScoresArgs(**dict(dict(      # noqa: E731
        lg=_lg(), k=2, has_ignore=0, ignore=0, token=P, logp=P, entropy=P, top_logp=P, top_ids=P, stats=P,
        ws=P), **kw))
    for kw in (dict(k=-1), dict(k=9), dict(k=65, lg=_lg(V=100, s2=100)), dict(logp=None), dict(entropy=None),
               dict(top_logp=None), dict(top_ids=None)):
        a = scores(**kw)
        assert lib.s2c_token_scores_fwd(ctypes.addressof(a), None) == EINVAL, kw
    a = scores()
    assert lib.s2c_token_scores_fwd(None, None) == EINVAL
    assert lib.s2c_token_scores_bwd(ctypes.addressof(a), P, P, P, None, None) == EINVAL
    assert lib.s2c_token_scores_bwd(ctypes.addressof(a), P, P, P, P + 2, None) == EINVAL
    for stats in (None, P + 8):
        a = scores(stats=stats)
        assert lib.s2c_token_scores_bwd(ctypes.addressof(a), P, P, P, P, None) == EINVAL
    assert lib.s2c_token_scores_fwd(ctypes.addressof(a), None) == EINVAL
    # many words of few rows: joined through a workspace
    for ws in (None, P + 4):
        a = scores(lg=_lg(V=1 << 18, s2=1 << 18), ws=ws)
        assert lib.s2c_token_scores_fwd(ctypes.addressof(a), None) == EINVAL
    distill = lambda **kw: _DistillArgs(**dict(dict(    # noqa: E731
        lg=_lg(), K=3, teacher_dtype=0, ids=P, teacher=P, mask=None, loss=P, stats=P, ws=P), **kw))
    for kw in (dict(K=0), dict(K=257), dict(teacher_dtype=5), dict(ids=None), dict(teacher=None),
               dict(loss=None)):
        d = distill(**kw)
        assert lib.s2c_distill_fwd(ctypes.addressof(d), None) == EINVAL, kw
    d = distill()
    assert lib.s2c_distill_bwd(ctypes.addressof(d), None, P, None) == EINVAL
    assert lib.s2c_distill_bwd(ctypes.addressof(d), P, None, None) == EINVAL
    for stats in (None, P + 4):
        d = distill(stats=stats)
        assert lib.s2c_distill_bwd(ctypes.addressof(d), P, P, None) == EINVAL
    assert lib.s2c_distill_fwd(ctypes.addressof(d), None) == EINVAL
    d = distill(lg=_lg(V=1 << 18, s2=1 << 18), ws=None)
    assert lib.s2c_distill_fwd(ctypes.addressof(d), None) == EINVAL
    fwd = lambda N=2, V=3, D=4, dt=0, ld=4, tok=P, tab=P, out=P: lib.s2c_embed_fwd(       # noqa: E731
        N, V, D, dt, ld, tok, tab, 1.0, -1, out, None)
    for kw in (dict(N=-1), dict(V=0), dict(D=0), dict(D=(1 << 24) + 1), dict(dt=3), dict(ld=-1), dict(tok=None),
               dict(tab=None), dict(out=None), dict(tab=P + 2), dict(out=P + 1, dt=1)):
        assert fwd(**kw) == EINVAL, kw
    grad = lambda N=2, V=3, D=4, dt=0, ld=4, tok=P, g=P, out=P: lib.s2c_embed_grad(        # noqa: E731
        N, V, D, dt, ld, tok, g, 1.0, -1, out, P, None)
    for kw in (dict(N=-1), dict(V=0), dict(D=0), dict(D=(1 << 24) + 1), dict(dt=3), dict(ld=-1), dict(tok=None),
               dict(g=None), dict(out=None), dict(g=P + 2), dict(out=P + 1, dt=2)):
        assert grad(**kw) == EINVAL, kw
    # many tokens: sorted in a workspace
    assert lib.s2c_embed_grad(5000, 300, 4, 0, 4, P, P, 1.0, -1, P, None, None) == EINVAL
    assert lib.s2c_embed_grad(5000, 300, 4, 0, 4, P, P, 1.0, -1, P, P + 8, None) == EINVAL
    assert lib.s2c_embed_grad(1 << 31, 300, 4, 0, 4, P, P, 1.0, -1, P, P, None) == EINVAL
    # nothing to do is no error and no launch
    z = scores(lg=_lg(rows=0, x=None))
    assert lib.s2c_token_scores_fwd(ctypes.addressof(z), None) == 0
    assert fwd(N=0) == 0
