"""The word operators of the captioner -- what is timed and what is compared.

`scan2cap_amd.word_ops` offers three operators around the word logits:

    token_scores   log probabilities of given words, entropy, the best alternatives (+ gradient)
    distill_loss   KL divergence from a teacher's top logits to the full vocabulary (+ gradient)
    embed_tokens   embedding lookup with scaling, and the table's gradient

Every case is one pass through one of them.  `run` computes it from elementary torch operations in
32 bits (`own` false) or through the framework's entry point (`own` true).
"""
import math

import torch

own = False

_DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_SIZE = {"f32": 4, "bf16": 2, "f16": 2}
PAD = 0                     # the vocabulary's padding word


# ---- the cases -----------------------------------------------------------------------------------
def _scores(name, rows, vocab, dtype, train, top_k, temperature=1.0, boxes=0, pad=0.0):
    """boxes > 0: the logits lie word-major, (rows / boxes, boxes, vocab), as a decoder that writes one
    word of every box at a time leaves them, and are scored as (boxes, words, vocab)."""
    return dict(name=name, op="scores", rows=rows, vocab=vocab, dtype=dtype, train=train, top_k=top_k,
                temperature=temperature, boxes=boxes, pad=pad)


def _distill(name, rows, vocab, dtype, train, slots, temperature=1.0, ragged=False, pad=0.0):
    return dict(name=name, op="distill", rows=rows, vocab=vocab, dtype=dtype, train=train, slots=slots,
                temperature=temperature, ragged=ragged, pad=pad)


def _embed(name, tokens, vocab, dim, dtype, train, scale=1.0, pad=0.0):
    return dict(name=name, op="embed", tokens=tokens, vocab=vocab, dim=dim, dtype=dtype, train=train,
                scale=scale, pad=pad)


def listed():
    return [
        # one word of one sequence over a large vocabulary: the latency of a single decoding step
        _scores("scores_one_word", 1, 32768, "bf16", False, 5),
        # one decoding step of a batch of sequences with twenty alternatives each
        _scores("scores_step", 64, 131072, "bf16", False, 20, temperature=0.7),
        # every word of every box of an evaluation batch (8 scenes, 256 boxes, 29 words), as the greedy
        # decoder leaves the logits
        _scores("scores_eval", 8 * 256 * 29, 3500, "f32", False, 5, boxes=8 * 256),
        # the captioner's training batch (8 captions of up to 31 words) under a policy gradient with an
        # entropy term
        _scores("scores_train", 8 * 31, 3500, "f32", True, 0, pad=0.3),
        # the same step with a large vocabulary of odd size, in 16 bits
        _scores("scores_train_wide", 4096, 50001, "bf16", True, 8, temperature=1.3, pad=0.1),
        # distillation in the captioner's training batch
        _distill("distill_train", 8 * 31, 3500, "f32", True, 16, temperature=2.0, pad=0.3),
        # ... over a large vocabulary
        _distill("distill_train_wide", 4096, 65536, "bf16", True, 64, temperature=2.0),
        # ... with an odd vocabulary, slots left empty and rows without any
        _distill("distill_ragged", 1000, 10007, "f16", True, 33, ragged=True),
        # the next word of every box of an evaluation batch
        _embed("embed_step", 8 * 256, 3500, 300, "f32", False),
        # a training batch's captions, with the gradient of the table
        _embed("embed_train", 8 * 32, 3500, 300, "f32", True, pad=0.3),
        # a long batch over a large table
        _embed("embed_train_wide", 131072, 50001, 1024, "bf16", True, scale=32.0),
        # an odd row width
        _embed("embed_odd", 8191, 10007, 515, "f16", True, scale=0.5, pad=0.1),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["scores", "distill", "embed"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    train = rng.random() < 0.6
    pad = rng.choice([0.0, 0.1, 0.3])
    if op == "embed":
        dim = _log_int(rng, 16, 4096)
        vocab = _log_int(rng, 64, min(131072, (1 << 25) // dim))
        tokens = _log_int(rng, 1, min(131072, (1 << 26) // dim))
        c = _embed("", tokens, vocab, dim, dtype, train, rng.choice([1.0, 0.5, math.sqrt(dim)]), pad)
    else:
        vocab = _log_int(rng, 64, 262144)
        rows = _log_int(rng, 1, min(32768, (1 << 27) // vocab))
        temperature = rng.choice([1.0, 1.0, 0.7, 2.0])
        if op == "scores":
            boxes = 0
            if rng.random() < 0.3 and rows >= 4:
                words = rng.randint(2, min(31, rows))
                boxes = rows // words
                rows = boxes * words
            c = _scores("", rows, vocab, dtype, train, rng.choice([0, 1, 5, 20, 32]), temperature, boxes,
                        pad)
        else:
            c = _distill("", rows, vocab, dtype, train, _log_int(rng, 1, min(128, vocab // 2)),
                         temperature, rng.random() < 0.5, pad)
    del c["name"]
    return c


# ---- inputs ----------------------------------------------------------------------------------------
def _logits(gen, rows, vocab, dtype):
    """Rows of word logits: a frequency-shaped bias plus each row's own spread; a few words of the
    vocabulary are never said (-inf)."""
    dev = "cuda"
    x = torch.randn(rows, vocab, generator=gen, device=dev) * 2.0
    x -= 0.5 * torch.log1p(torch.arange(vocab, device=dev, dtype=torch.float32))
    never = torch.rand(vocab, generator=gen, device=dev) < 0.02
    never[2:4] = False
    x[:, never] = float("-inf")
    said = torch.nonzero(~never).view(-1)
    said = said[said != PAD]
    words = said[torch.randint(0, said.numel(), (rows,), generator=gen, device=dev)]
    # a trained model favours the word that is said
    x[torch.arange(rows, device=dev), words] += 4.0
    return x.to(_DT[dtype]), words


def _padded(gen, words, pad):
    if pad > 0:
        gone = torch.rand(words.shape, generator=gen, device="cuda") < pad
        words = torch.where(gone, torch.full_like(words, PAD), words)
    return words


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dev = "cuda"
    st = dict(case)
    if case["op"] == "scores":
        x, words = _logits(gen, case["rows"], case["vocab"], case["dtype"])
        words = _padded(gen, words, case["pad"])
        shape = (case["rows"],)
        if case["boxes"]:
            n = case["boxes"]
            x = x.view(case["rows"] // n, n, case["vocab"]).transpose(0, 1)
            words = words.view(case["rows"] // n, n).t().contiguous()
            shape = tuple(words.shape)
        st.update(x=x, words=words)
        if case["train"]:
            st["g_logp"] = torch.randn(shape, generator=gen, device=dev)
            st["g_entropy"] = torch.randn(shape, generator=gen, device=dev) * 0.1
    elif case["op"] == "distill":
        R, V, K = case["rows"], case["vocab"], case["slots"]
        x, words = _logits(gen, R, V, case["dtype"])
        # the teacher sees what the student sees, with noise of its own
        t = x.float() + torch.randn(R, V, generator=gen, device=dev) * 0.5
        top, ids = torch.topk(t, K, dim=-1)
        del t
        if case["ragged"]:
            n = torch.randint(0, K + 1, (R, 1), generator=gen, device=dev)
            ids = torch.where(torch.arange(K, device=dev) < n, ids, torch.full_like(ids, -1))
        mask = None
        if case["pad"] > 0:
            mask = torch.rand(R, generator=gen, device=dev) >= case["pad"]
        st.update(x=x, ids=ids.contiguous(), teacher=top.to(_DT[case["dtype"]]).contiguous(), mask=mask)
        if case["train"]:
            st["g_loss"] = torch.rand(R, generator=gen, device=dev) + 0.5
    else:
        N, V, D = case["tokens"], case["vocab"], case["dim"]
        # words follow a 1 / rank law
        u = torch.rand(N, generator=gen, device=dev, dtype=torch.float64)
        ids = (torch.exp(u * math.log(V + 1.0)) - 1.0).long().clamp_(0, V - 1)
        ids = torch.where(ids == PAD, torch.randint(1, V, (N,), generator=gen, device=dev), ids)
        st["ids"] = _padded(gen, ids, case["pad"])
        st["table"] = (torch.randn(V, D, generator=gen, device=dev) * 0.3).to(_DT[case["dtype"]])
        if case["train"]:
            st["g_out"] = torch.randn(N, D, generator=gen, device=dev).to(_DT[case["dtype"]])
    return st


# ---- plain forms -----------------------------------------------------------------------------------
def _plain_scores(s):
    x, words, k, t = s["x"], s["words"], s["top_k"], s["temperature"]
    z = x.float() / t
    d = z - z.amax(dim=-1, keepdim=True)
    e = torch.exp(d)
    total = e.sum(dim=-1, keepdim=True)
    logq = d - torch.log(total)
    p = e / total
    live = words != PAD
    zero = torch.zeros((), device=x.device)
    logp = torch.where(live, torch.gather(logq, -1, words.unsqueeze(-1)).squeeze(-1), zero)
    h = -torch.where(p > 0, p * logq, zero).sum(dim=-1)
    entropy = torch.where(live, h, zero)
    out = [logp, entropy]
    if k:
        ids = torch.sort(x.float(), dim=-1, descending=True, stable=True)[1][..., :k]
        top = torch.gather(logq, -1, ids)
        out.append(torch.where(live.unsqueeze(-1), top, zero))
        out.append(torch.where(live.unsqueeze(-1), ids, torch.full_like(ids, -1)))
    if s["train"]:
        gl = torch.where(live, s["g_logp"], zero).unsqueeze(-1)
        ge = torch.where(live, s["g_entropy"], zero).unsqueeze(-1)
        g = -p * (gl + ge * torch.where(p > 0, logq + h.unsqueeze(-1), zero))
        g = g + gl * (torch.arange(x.shape[-1], device=x.device) == words.unsqueeze(-1))
        out.append((g / t).to(x.dtype))
    return out


def _plain_distill(s):
    x, ids, t = s["x"], s["ids"], s["temperature"]
    zero = torch.zeros((), device=x.device)
    z = x.float() / t
    d = z - z.amax(dim=-1, keepdim=True)
    e = torch.exp(d)
    total = e.sum(dim=-1, keepdim=True)
    logp = d - torch.log(total)
    used = ids >= 0
    w = s["teacher"].float() / t
    peak = torch.where(used, w, torch.full_like(w, -3e38)).amax(dim=-1, keepdim=True)
    ew = torch.where(used, torch.exp(torch.where(used, w - peak, zero)), zero)
    sum_w = ew.sum(dim=-1, keepdim=True)
    q = ew / torch.where(sum_w > 0, sum_w, torch.ones_like(sum_w))
    logq = torch.where(used, w - peak - torch.log(torch.where(sum_w > 0, sum_w, torch.ones_like(sum_w))),
                       zero)
    safe = ids.clamp(min=0)
    terms = torch.where(q > 0, q * (logq - torch.gather(logp, -1, safe)), zero)
    live = used.any(dim=-1)
    if s["mask"] is not None:
        live = live & s["mask"]
    out = [torch.where(live, terms.sum(dim=-1), zero)]
    if s["train"]:
        g = torch.where(live, s["g_loss"], zero).unsqueeze(-1)
        dz = g * (e / total)
        dz.scatter_add_(-1, safe, -g * q)
        out.append((dz / t).to(x.dtype))
    return out


def _plain_embed(s):
    ids, table = s["ids"], s["table"]
    live = (ids != PAD).unsqueeze(-1)
    out = [(table.float()[ids] * s["scale"] * live).to(table.dtype)]
    if s["train"]:
        g = torch.zeros(table.shape, device=table.device)
        g.index_add_(0, ids, s["g_out"].float() * live)
        out.append((g * s["scale"]).to(table.dtype))
    return out


# ---- one pass ----------------------------------------------------------------------------------------
def run(s):
    if not own:
        with torch.no_grad():
            return {"scores": _plain_scores, "distill": _plain_distill, "embed": _plain_embed}[s["op"]](s)
    from scan2cap_amd import word_ops
    if s["op"] == "scores":
        x = s["x"].detach().requires_grad_(s["train"])
        r = word_ops.token_scores(x, s["words"], top_k=s["top_k"], temperature=s["temperature"],
                                  ignore_index=PAD)
        out = [r.logp, r.entropy] + ([r.top_logp, r.top_ids] if s["top_k"] else [])
        if s["train"]:
            out += torch.autograd.grad([r.logp, r.entropy], [x], [s["g_logp"], s["g_entropy"]])
    elif s["op"] == "distill":
        x = s["x"].detach().requires_grad_(s["train"])
        loss = word_ops.distill_loss(x, s["ids"], s["teacher"], temperature=s["temperature"],
                                     mask=s["mask"])
        out = [loss]
        if s["train"]:
            out += torch.autograd.grad([loss], [x], [s["g_loss"]])
    else:
        table = s["table"].detach().requires_grad_(s["train"])
        y = word_ops.embed_tokens(s["ids"], table, scale=s["scale"], padding_idx=PAD)
        out = [y]
        if s["train"]:
            out += torch.autograd.grad([y], [table], [s["g_out"]])
    return [o.detach() for o in out]


# ---- what a pass cannot do without -------------------------------------------------------------------
def _distinct(vocab, tokens):
    """Expected number of distinct words among `tokens` draws of the 1 / rank law."""
    v = torch.arange(vocab, dtype=torch.float64)
    p = (torch.log(v + 2.0) - torch.log(v + 1.0)) / math.log(vocab + 1.0)
    return float((1.0 - torch.exp(tokens * torch.log1p(-p))).sum())


def work(case):
    b = _SIZE[case["dtype"]]
    if case["op"] == "embed":
        N, V, D = case["tokens"], case["vocab"], case["dim"]
        live = 1.0 - case["pad"]          # padding words read no row and leave no gradient
        size = 8 * N + b * D * (min(N, _distinct(V, N)) + N)
        flops = N * D
        if case["train"]:
            size += b * D * (N * live + V)
            flops += N * D + V * D
        return {"bytes": int(size), "flops": int(flops)}
    R, V = case["rows"], case["vocab"]
    live = 1.0 - case["pad"]              # rows of padding words take no part
    size, flops = b * R * V * live, 6.0 * R * V * live
    if case["op"] == "scores":
        size += R * (8 + 4 + 4 + 12 * case["top_k"])
        extra = 8
    else:
        size += R * (case["slots"] * (8 + b) + 4)
        extra = 4
    if case["train"]:
        size += b * R * V + R * extra
        flops += 6.0 * R * V * live
    return {"bytes": int(size), "flops": int(flops)}


# ---- the definition in 64 bits ------------------------------------------------------------------------
def _by_rows(rows, vocab):
    step = max(1, (1 << 26) // vocab)
    return [(i, min(rows, i + step)) for i in range(0, rows, step)]


def _exact_scores(s):
    V, k, t = s["vocab"], s["top_k"], s["temperature"]
    x, words = s["x"].reshape(-1, V), s["words"].reshape(-1)
    g = [s[n].reshape(-1) for n in ("g_logp", "g_entropy")] if s["train"] else None
    parts = []
    for a, b in _by_rows(x.shape[0], V):
        z = x[a:b].double().requires_grad_(s["train"])
        live = words[a:b] != PAD
        with torch.enable_grad():
            lp = torch.log_softmax(z / t, dim=-1)
            said = lp[torch.arange(b - a, device=x.device), words[a:b]]
            finite = lp.masked_fill(torch.isinf(lp), 0.0)
            h = -(torch.exp(lp) * finite).sum(-1)
        row = [torch.where(live, said.detach(), 0.0), torch.where(live, h.detach(), 0.0)]
        if k:
            # lowest index first among equal values: order by (value, -index), one word at a time
            v = x[a:b].double().clone()
            ids = torch.empty((b - a, k), dtype=torch.int64, device=x.device)
            index = torch.arange(V, device=x.device)
            for j in range(k):
                best = v.max(dim=-1, keepdim=True)[0]
                ids[:, j] = torch.where(v == best, index, V).min(dim=-1)[0]
                v.scatter_(1, ids[:, j:j + 1], float("-inf"))
            row.append(torch.where(live[:, None], lp.detach().gather(1, ids), 0.0))
            row.append(torch.where(live[:, None], ids, -1))
        if g is not None:
            up = [torch.where(live, gi[a:b].double(), 0.0) for gi in g]
            # a word that is never said takes no gradient; log_softmax's backward forms it as 0 already,
            # the entropy's through `finite` likewise
            row.append(torch.autograd.grad([said, h], [z], up)[0])
        parts.append(row)
    out = [torch.cat(c) for c in zip(*parts)]
    shape = tuple(s["words"].shape)
    return [o.reshape(shape + tuple(o.shape[1:])) for o in out]


def _exact_distill(s):
    V, t = s["vocab"], s["temperature"]
    parts = []
    for a, b in _by_rows(s["rows"], V):
        z = s["x"][a:b].double().requires_grad_(s["train"])
        ids = s["ids"][a:b]
        q = torch.softmax((s["teacher"][a:b].double() / t).masked_fill(ids < 0, float("-inf")), dim=-1)
        q = torch.nan_to_num(q, nan=0.0)                      # rows without any slot
        if s["mask"] is not None:
            q = q * s["mask"][a:b, None]
        with torch.enable_grad():
            lp = torch.log_softmax(z / t, dim=-1).gather(1, ids.clamp(min=0))
            loss = (torch.special.xlogy(q, q) - torch.where(q > 0, q * lp, 0.0)).sum(-1)
        row = [loss.detach()]
        if s["train"]:
            row += torch.autograd.grad([loss], [z], [s["g_loss"][a:b].double()])
        parts.append(row)
    return [torch.cat(c) for c in zip(*parts)]


def _exact_embed(s):
    ids, table = s["ids"], s["table"].double()
    table[PAD] = 0.0
    out = [torch.index_select(table, 0, ids) * s["scale"]]
    if s["train"]:
        # sums over each word's places, in the order of the words
        order = torch.argsort(ids)
        run_end = torch.cumsum(torch.bincount(ids, minlength=s["vocab"]), 0)
        parts = []
        for c in range(0, s["dim"], 128):
            acc = torch.cumsum(s["g_out"][order, c:c + 128].double(), 0)
            acc = torch.cat([torch.zeros_like(acc[:1]), acc])[run_end]
            parts.append(torch.diff(acc, dim=0, prepend=torch.zeros_like(acc[:1])))
        g = torch.cat(parts, 1) * s["scale"]
        g[PAD] = 0.0
        out.append(g)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"scores": _exact_scores, "distill": _exact_distill, "embed": _exact_embed}[case["op"]](s)
