"""Operators around the captioner's word logits, forward and backward, on the hand-written kernels of
csrc/s2c_vocab.hip and csrc/s2c_embed.hip (C ABI: include/s2c_words.h):

    token_scores   log probabilities of given words, entropy, the best alternatives
    distill_loss   KL divergence from a teacher's top logits to the softmax over the whole vocabulary
    embed_tokens   embedding lookup with scaling, and the table's gradient summed by sorted words

Logits and tables may be float32, bfloat16 or float16; statistics, sums and losses are float32, gradients
come in their input's type, rounded once.  Work is enqueued on the current stream of the tensors' device,
nothing synchronises, scratch memory is allocated per call.  Arguments that the kernels do not take are
refused with ValueError (shapes, types, ranges) or RuntimeError (CPU tensors: there is no fallback).
Values that live on the device cannot be refused without a synchronisation: a word index outside the
vocabulary is never used as an address and turns its row's results into NaN.
"""
import collections
import ctypes
import math

import torch
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from . import _C

_I, _LL, _F, _P = ctypes.c_int, ctypes.c_longlong, ctypes.c_float, ctypes.c_void_p

MAX_TOP = 64             # S2C_WORDS_MAX_TOP
MAX_SLOTS = 256          # S2C_WORDS_MAX_SLOTS
MAX_DIM = 1 << 24        # S2C_WORDS_MAX_DIM
_NONE = -(1 << 63)       # no padding word
_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


class _Logits(ctypes.Structure):
    """include/s2c_words.h: s2c_logits"""
    _fields_ = [("rows", _I), ("V", _I), ("dtype", _I), ("n1", _I), ("n2", _I), ("inv_t", _F),
                ("s0", _LL), ("s1", _LL), ("s2", _LL), ("x", _P)]


class _ScoresArgs(ctypes.Structure):
    """include/s2c_words.h: s2c_token_scores_args"""
    _fields_ = [("lg", _Logits), ("k", _I), ("has_ignore", _I), ("ignore", _LL), ("token", _P),
                ("logp", _P), ("entropy", _P), ("top_logp", _P), ("top_ids", _P), ("stats", _P),
                ("ws", _P)]


class _DistillArgs(ctypes.Structure):
    """include/s2c_words.h: s2c_distill_args"""
    _fields_ = [("lg", _Logits), ("K", _I), ("teacher_dtype", _I), ("ids", _P), ("teacher", _P),
                ("mask", _P), ("loss", _P), ("stats", _P), ("ws", _P)]


_C.register("s2c_token_scores_fwd", [_P, _P])
_C.register("s2c_token_scores_bwd", [_P, _P, _P, _P, _P, _P])
_C.register("s2c_distill_fwd", [_P, _P])
_C.register("s2c_distill_bwd", [_P, _P, _P, _P])
_C.register("s2c_embed_fwd", [_LL, _I, _I, _I, _LL, _P, _P, _F, _LL, _P, _P])
_C.register("s2c_embed_grad", [_LL, _I, _I, _I, _LL, _P, _P, _F, _LL, _P, _P, _P])

TokenScores = collections.namedtuple("TokenScores", "logp entropy top_logp top_ids")


def _check(cond, msg, *args):
    if not cond:
        raise ValueError(msg % tuple(str(a) if isinstance(a, tuple) else a for a in args))


def _check_gpu(**tensors):
    first = None
    for name, t in tensors.items():
        if t is None:
            continue
        if not t.is_cuda:
            raise RuntimeError("%s must be a GPU tensor: CPU not supported" % name)
        first = first or (name, t)
        if t.device != first[1].device:
            raise RuntimeError("%s is on %s, %s on %s" % (name, t.device, first[0], first[1].device))


def _check_float(name, t):
    _check(torch.is_tensor(t), "%s must be a tensor", name)
    _check(t.dtype in _DTYPES, "%s must be float32, bfloat16 or float16, not %s", name, t.dtype)


def _check_ids(name, t, shape=None):
    _check(torch.is_tensor(t), "%s must be a tensor", name)
    _check(t.dtype in (torch.int64, torch.int32), "%s must be int64 or int32, not %s", name, t.dtype)
    _check(shape is None or tuple(t.shape) == tuple(shape), "%s has shape %s, %s is needed", name,
           tuple(t.shape), shape)


def _ids(t):
    return t.to(torch.int64).contiguous()


def _ptr(t):
    return None if t is None else t.data_ptr()


_SIZES = {"s2c_token_scores_workspace_bytes": [_I] * 4, "s2c_distill_workspace_bytes": [_I] * 3,
          "s2c_embed_grad_workspace_bytes": [_LL, _I, _I]}
_size_fns = {}


def _workspace(name, device, *args):
    f = _size_fns.get(name)
    if f is None:
        f = getattr(_C.load(), name)
        f.argtypes, f.restype = _SIZES[name], _LL
        _size_fns[name] = f
    n = f(*args)
    return torch.empty(n, dtype=torch.uint8, device=device) if n else None


def _run(name, device, *args, alg_bytes=0):
    """One entry point on the device's current stream.  A training batch's launch takes 5 - 10 us, as long
    as the Python around it: the device is switched only where it is another one, and the stream's handle
    is asked for directly."""
    if _C.TIMER.enabled:
        _C.TIMER.alg_bytes = int(alg_bytes)
    if device.index == torch._C._cuda_getDevice():
        _C.call(name, *args, torch._C._cuda_getCurrentRawStream(device.index))
    else:
        with torch.cuda.device(device):
            _C.call(name, *args, torch._C._cuda_getCurrentRawStream(device.index))


def _f32(g):
    if g is None or (g.dtype is torch.float32 and g.is_contiguous()):
        return g
    return g.to(torch.float32).contiguous()


def _merge_axes(shape, strides):
    """The axes as few (size, stride) pairs that step alike."""
    out = []
    for n, s in zip(shape, strides):
        if n == 1:
            continue
        if out and out[-1][1] == n * s:
            out[-1] = (out[-1][0] * n, s)
        else:
            out.append((n, s))
    return out


def _logits(x, temperature):
    """x (..., V) as the kernels read it: (tensor, s2c_logits).  Up to three leading axes of any strides
    are read in place (a decoder's word-major logits permuted to (B, K, T, V)); more, or words that are
    not adjacent, are copied first."""
    V = x.shape[-1]
    rows = x.numel() // V
    if x.is_contiguous():
        return x, _Logits(rows, V, _DTYPES[x.dtype], 1, max(rows, 1), 1.0 / temperature, 0, 0, V, x.data_ptr())
    if V > 1 and x.stride(-1) != 1:
        x = x.contiguous()
    axes = _merge_axes(x.shape[:-1], x.stride()[:-1])
    if len(axes) > 3:
        x = x.contiguous()
        axes = _merge_axes(x.shape[:-1], x.stride()[:-1])
    axes = [(1, 0)] * (3 - len(axes)) + axes
    return x, _Logits(rows, V, _DTYPES[x.dtype], axes[1][0], axes[2][0], 1.0 / temperature,
                      axes[0][1], axes[1][1], axes[2][1], x.data_ptr())


def _first_order(fn, ctx, grads):
    """The gradients are not differentiable again; the guard that says so is put around them only where a
    graph of the backward pass is asked for (create_graph)."""
    if torch.is_grad_enabled():
        return once_differentiable(fn._backward)(ctx, *grads)
    return fn._backward(ctx, *grads)


def _check_logits(x, temperature):
    _check_float("logits", x)
    _check(x.dim() >= 1 and x.shape[-1] >= 1, "logits need a vocabulary axis, not shape %s", tuple(x.shape))
    _check(x.numel() // x.shape[-1] < 2 ** 31 and x.shape[-1] < 2 ** 31,
           "logits: more than 2^31 rows or words")
    t = float(temperature)
    _check(math.isfinite(t) and 1e-30 <= t <= 1e30, "temperature must be positive and finite, not %r",
           temperature)
    return t


class _TokenScores(Function):
    @staticmethod
    def forward(ctx, logits, tokens, top_k, temperature, ignore_index):
        x, lg = _logits(logits, temperature)
        shape, dev = logits.shape[:-1], logits.device
        f32 = dict(dtype=torch.float32, device=dev)
        logp = torch.empty(shape, **f32) if tokens is not None else None
        entropy = torch.empty(shape, **f32)
        top_logp = torch.empty(shape + (top_k,), **f32) if top_k else None
        top_ids = torch.empty(shape + (top_k,), dtype=torch.int64, device=dev) if top_k else None
        stats = torch.empty((lg.rows, 4), **f32)
        args = _ScoresArgs(lg, top_k, int(ignore_index is not None), ignore_index or 0, _ptr(tokens),
                           _ptr(logp), entropy.data_ptr(), _ptr(top_logp), _ptr(top_ids), stats.data_ptr(),
                           None)
        if lg.rows:
            ws = _workspace("s2c_token_scores_workspace_bytes", dev, lg.rows, lg.V, lg.dtype, top_k)
            args.ws = _ptr(ws)
            _run("s2c_token_scores_fwd", dev, ctypes.addressof(args),
                 alg_bytes=x.numel() * x.element_size() + lg.rows * (16 + 12 * top_k))
        ctx.set_materialize_grads(False)
        if top_ids is not None:
            ctx.mark_non_differentiable(top_ids)
        if ctx.needs_input_grad[0]:
            ctx.save_for_backward(x, tokens, top_ids, stats)      # what `args` points to
            ctx.args, ctx.shape = args, logits.shape
        return logp, entropy, top_logp, top_ids

    @staticmethod
    def _backward(ctx, g_logp, g_entropy, g_top, _g_ids):
        x = ctx.saved_tensors[0]
        dx = torch.empty(ctx.shape, dtype=x.dtype, device=x.device)
        if ctx.args.lg.rows:
            if g_logp is None and g_entropy is None and g_top is None:
                return None, None, None, None, None
            gl, ge, gt = _f32(g_logp), _f32(g_entropy), _f32(g_top)
            _run("s2c_token_scores_bwd", x.device, ctypes.addressof(ctx.args), _ptr(gl), _ptr(ge), _ptr(gt),
                 dx.data_ptr(), alg_bytes=2 * x.numel() * x.element_size())
        return dx, None, None, None, None

    @staticmethod
    def backward(ctx, *grads):
        return _first_order(_TokenScores, ctx, grads)


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
    t = _check_logits(logits, temperature)
    top_k = int(top_k)
    _check(0 <= top_k <= min(MAX_TOP, logits.shape[-1]), "top_k must be in [0, min(%d, V)], not %d", MAX_TOP,
           top_k)
    if tokens is not None:
        _check_ids("tokens", tokens, tuple(logits.shape[:-1]))
    else:
        _check(ignore_index is None, "ignore_index needs tokens")
    _check_gpu(logits=logits, tokens=tokens)
    tokens = None if tokens is None else _ids(tokens)
    return TokenScores(*_TokenScores.apply(logits, tokens, top_k, t,
                                           None if ignore_index is None else int(ignore_index)))


class _Distill(Function):
    @staticmethod
    def forward(ctx, logits, ids, teacher, mask, temperature):
        x, lg = _logits(logits, temperature)
        dev = logits.device
        loss = torch.empty(logits.shape[:-1], dtype=torch.float32, device=dev)
        stats = torch.empty((lg.rows, 4), dtype=torch.float32, device=dev)
        args = _DistillArgs(lg, ids.shape[-1], _DTYPES[teacher.dtype], ids.data_ptr(), teacher.data_ptr(),
                            _ptr(mask), loss.data_ptr(), stats.data_ptr(), None)
        if lg.rows:
            ws = _workspace("s2c_distill_workspace_bytes", dev, lg.rows, lg.V, lg.dtype)
            args.ws = _ptr(ws)
            _run("s2c_distill_fwd", dev, ctypes.addressof(args),
                 alg_bytes=x.numel() * x.element_size() + ids.numel() * (8 + teacher.element_size()))
        ctx.set_materialize_grads(False)
        if ctx.needs_input_grad[0]:
            ctx.save_for_backward(x, ids, teacher, stats)         # what `args` points to
            ctx.args, ctx.shape = args, logits.shape
        return loss

    @staticmethod
    def _backward(ctx, g_loss):
        if g_loss is None:
            return None, None, None, None, None
        x = ctx.saved_tensors[0]
        dx = torch.empty(ctx.shape, dtype=x.dtype, device=x.device)
        if ctx.args.lg.rows:
            g = _f32(g_loss)
            _run("s2c_distill_bwd", x.device, ctypes.addressof(ctx.args), g.data_ptr(), dx.data_ptr(),
                 alg_bytes=2 * x.numel() * x.element_size())
        return dx, None, None, None, None

    @staticmethod
    def backward(ctx, *grads):
        return _first_order(_Distill, ctx, grads)


def distill_loss(logits, teacher_ids, teacher_logits, temperature=1.0, mask=None):
    """KL(q || p) of every row, float32 (...): q = the teacher's softmax over its K <= 256 slots
    (teacher_ids, teacher_logits) (..., K) at `temperature`, p = softmax(logits / temperature) over all V
    words.  Differentiable with respect to `logits`; the teacher is a constant.  (Hinton's factor
    temperature^2 is the caller's.)

    Log probabilities serve as teacher logits as well (`token_scores(...).top_ids / .top_logp` of the
    teacher).  A slot with a negative id or a logit of -inf is empty; an id may occur twice.  Rows with
    mask (..., bool) False are not read; they and rows without a used slot have loss 0 and zero gradient.
    A used id >= V makes the row's loss and gradient NaN; a row of logits that are all -inf has loss +inf
    and zero gradient."""
    t = _check_logits(logits, temperature)
    _check(torch.is_tensor(teacher_ids) and teacher_ids.dim() == logits.dim(),
           "teacher_ids needs the logits' leading axes and a slot axis")
    K = teacher_ids.shape[-1]
    _check(1 <= K <= MAX_SLOTS, "1 to %d teacher slots a row, not %d", MAX_SLOTS, K)
    shape = tuple(logits.shape[:-1])
    _check_ids("teacher_ids", teacher_ids, shape + (K,))
    _check_float("teacher_logits", teacher_logits)
    _check(tuple(teacher_logits.shape) == shape + (K,), "teacher_logits has shape %s, %s is needed",
           tuple(teacher_logits.shape), shape + (K,))
    _check(not (teacher_logits.requires_grad and torch.is_grad_enabled()),
           "teacher_logits requires a gradient, which distill_loss does not form: detach it")
    if mask is not None:
        _check(torch.is_tensor(mask) and mask.dtype == torch.bool and tuple(mask.shape) == shape,
               "mask must be a bool tensor of shape %s", shape)
        mask = mask.contiguous()
    _check_gpu(logits=logits, teacher_ids=teacher_ids, teacher_logits=teacher_logits, mask=mask)
    ids = _ids(teacher_ids)
    return _Distill.apply(logits, ids, teacher_logits.contiguous(), mask, t)


class _EmbedTokens(Function):
    @staticmethod
    def forward(ctx, tokens, table, scale, padding):
        (V, D), N, dev = table.shape, tokens.numel(), table.device
        out = torch.empty(tokens.shape + (D,), dtype=table.dtype, device=dev)
        if N and D:
            _run("s2c_embed_fwd", dev, N, V, D, _DTYPES[table.dtype], table.stride(0), tokens.data_ptr(),
                 table.data_ptr(), scale, padding, out.data_ptr(),
                 alg_bytes=2 * out.numel() * out.element_size())
        ctx.set_materialize_grads(False)
        if ctx.needs_input_grad[1]:
            ctx.save_for_backward(tokens)
            ctx.opts = (N, V, D, table.dtype, scale, padding)
        return out

    @staticmethod
    def _backward(ctx, g):
        if g is None:
            return None, None, None, None
        tokens, = ctx.saved_tensors
        N, V, D, dtype, scale, padding = ctx.opts
        dev = g.device
        d_table = torch.empty((V, D), dtype=dtype, device=dev)
        if D:
            ld = D
            if not g.is_contiguous():
                axes = _merge_axes(g.shape[:-1], g.stride()[:-1])
                if len(axes) > 1 or (D > 1 and g.stride(-1) != 1):
                    g = g.contiguous()
                elif axes:
                    ld = axes[0][1]
            ws = _workspace("s2c_embed_grad_workspace_bytes", dev, N, V, D)
            _run("s2c_embed_grad", dev, N, V, D, _DTYPES[dtype], ld, tokens.data_ptr(), g.data_ptr(), scale,
                 padding, d_table.data_ptr(), _ptr(ws), alg_bytes=(N * D + V * D) * g.element_size())
        return None, d_table, None, None

    @staticmethod
    def backward(ctx, *grads):
        return _first_order(_EmbedTokens, ctx, grads)


def embed_tokens(tokens, table, scale=1.0, padding_idx=None):
    """scale * table[tokens]: tokens (...) int64 or int32, table (V, D) with adjacent columns (rows may be
    strided) -> (..., D) of the table's type.  Tokens equal to `padding_idx` (any integer) give zeros and
    no gradient; a token outside [0, V) gives a row of NaN and no gradient.  The table's gradient is
    dense, summed in float32 over each word's places in their order (the same bits every time)."""
    _check_float("table", table)
    _check(table.dim() == 2 and 1 <= table.shape[0] < 2 ** 31 and table.shape[1] <= MAX_DIM,
           "table must be (V, D) with 1 <= V and D <= 2^24, not %s", tuple(table.shape))
    _check(table.shape[1] <= 1 or table.stride(1) == 1, "the table's columns must be adjacent")
    s = float(scale)
    _check(math.isfinite(s) and abs(s) <= 3e38, "scale must be finite, not %r", scale)
    _check_ids("tokens", tokens)
    _check(tokens.numel() < 2 ** 31, "tokens: more than 2^31")
    _check_gpu(table=table, tokens=tokens)
    tokens = _ids(tokens)
    return _EmbedTokens.apply(tokens, table, s, _NONE if padding_idx is None else int(padding_idx))
