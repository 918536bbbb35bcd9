"""Measured cases of the operators on the logits behind a model's head: training by a teacher's most likely tokens, and what a
serving program does to logits before it looks at their log probabilities.

* ``distill``       divergence of a student's rows from a teacher's ``K`` most likely tokens and the rest, with the log
                    probabilities of the batch's own targets, and what the gradient needs of each row (``stats``).
* ``distill_grad``  the gradient with respect to the logits (of a vocabulary shard), from gradients of both.
* ``adjust``        penalties for tokens of the row's history, biases of single tokens, a grammar's bit mask, temperature.
* ``adjust_grad``   the gradient with respect to the logits before that.

``beta``: 0 the divergence of the student from the teacher, 1 of the teacher from the student, between them of both from
their mixture.  ``rest``: the tokens that are not listed are one more alternative; without it the teacher is renormed over its list.
Logits: a wide normal distribution with heavy tails; the listed tokens' are near the teacher's, as those of a student that has learned
some.  One list in sixteen ends early, one target in eight is none.  History: small numbers are frequent, P(t) goes by
1 / (t + 1); between a quarter and all of its places count, a part of them are the prompt.  ``allowed``: the share of the
vocabulary that a grammar leaves.  ``given``: what the call has besides mask and scale: "p" penalties, "b" biases.
"""
import math

import torch

own = False     # False: plain forms.  True: the calls that a user makes of the framework

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}
BIASES = 48     # tokens with a bias of their own in each row
LEAST_REST = 2.0 ** -22     # what float32 log probabilities tell from a list that holds everything: a smaller rest is none, or this for beta 1


def _distill(name, N, V, K, type, beta=0.0, rest=True, targets=True, scale=1.0, masked=0.0, index="i64"):
    return dict(name=name, kind="distill", N=N, V=V, K=K, type=type, beta=beta, rest=rest, targets=targets, scale=scale,
                masked=masked, index=index)


def _distill_grad(name, N, V, K, type, beta=0.0, rest=True, targets=True, scale=1.0, masked=0.0, index="i64", shards=1, shard=0):
    return dict(_distill(name, N, V, K, type, beta, rest, targets, scale, masked, index), kind="distill_grad", shards=shards,
                shard=shard)


def _adjust(name, N, V, H, type, out, given, allowed=None, scaled=True, into=False, index="i64", kind="adjust"):
    return dict(name=name, kind=kind, N=N, V=V, H=H, type=type, out=out, given=given, allowed=allowed, scaled=scaled, into=into,
                index=index)


def listed():
    return [
        # a short batch with a few alternatives from a stored file, odd vocabulary, everything in float32
        _distill("distill_short", 333, 32003, 8, "f32", targets=False, index="i32"),
        # a training batch of 8192 tokens with 20 alternatives and the batch's own targets
        _distill("distill_train", 8192, 128256, 20, "bf16"),
        # the student's own text, scored by both: mixture of the two, 64 alternatives, a temperature
        _distill("distill_mixture", 2048, 50257, 64, "f16", beta=0.5, targets=False, scale=0.5),
        # the gradient of the training batch
        _distill_grad("distill_grad_train", 8192, 128256, 20, "bf16"),
        # the gradient of an eighth of the vocabulary, 128 renormed alternatives
        _distill_grad("distill_grad_shard", 4096, 19008, 128, "bf16", rest=False, targets=False, shards=8, shard=3),
        # the gradient towards a teacher's peaks on a short batch, odd vocabulary
        _distill_grad("distill_grad_short", 517, 32003, 50, "f16", beta=1.0, scale=0.8),
        # one decoding step of 16 requests: penalties, biases, a grammar, temperatures; float32 for the choice
        _adjust("adjust_decode", 16, 128256, 2048, "bf16", "f32", "pb", allowed=0.5),
        # one decoding step of 64 requests under a strict grammar, in the logits' place
        _adjust("adjust_grammar", 64, 151936, 0, "bf16", "bf16", "", allowed=0.01, scaled=False, into=True),
        # one decoding step of 128 requests with long histories, odd vocabulary
        _adjust("adjust_long", 128, 50257, 16384, "f32", "f32", "p", index="i32"),
        # scores of 1024 places of drafted texts
        _adjust("adjust_drafts", 1024, 128256, 1024, "bf16", "bf16", "pb", allowed=0.5),
        # the gradient of a policy's batch that was drawn under a grammar with penalties
        _adjust("adjust_grad_policy", 2048, 128256, 1024, "bf16", "bf16", "p", allowed=0.5, kind="adjust_grad"),
        # ... of one short text, odd vocabulary, float32
        _adjust("adjust_grad_short", 77, 32003, 500, "f32", "f32", "p", index="i32", kind="adjust_grad"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    most = 4.2e9    # bytes of the largest listed case
    while True:
        kind = rng.choice(["distill", "distill", "distill_grad", "distill_grad", "adjust", "adjust", "adjust", "adjust_grad"])
        type, index = rng.choice(["bf16", "bf16", "f16", "f32"]), rng.choice(["i64", "i32"])
        V = rng.choice([_log(rng, 500, 262144), 128 * _log(rng, 8, 2048)])
        if kind in ("distill", "distill_grad"):
            beta = rng.choice([0.0, 0.0, 0.5, 0.1, 1.0])
            c = dict(kind=kind, N=_log(rng, 1, 32768), V=V, K=rng.choice([_log(rng, 1, 256), 20, 64]), type=type, beta=beta,
                     rest=beta == 1.0 or rng.random() < 0.6, targets=rng.random() < 0.5, scale=rng.choice([1.0, 1.0, 0.5, 1.25]),
                     masked=rng.choice([0.0, 0.0, 0.5, 0.99]), index=index)
            if kind == "distill_grad":
                c["shards"] = rng.choice([1, 1, 2, 8])
                c["shard"] = rng.randrange(c["shards"])
        else:
            c = dict(kind=kind, N=_log(rng, 1, 8192), V=V, H=_log(rng, 1, 32768), type=type, out=rng.choice([type, type, "f32"]),
                     given=rng.choice(["p", "p", "pb", "b", ""]), allowed=rng.choice([None, 0.5, 0.9, 0.01]),
                     scaled=rng.random() < 0.6, into=False, index=index)
            if kind == "adjust_grad":
                c["given"] = c["given"].replace("b", "")
            if not c["given"] and c["allowed"] is None:
                c["given"] = "p"
            if kind == "adjust" and not c["given"] and not c["scaled"]:
                c["into"], c["out"] = True, type
            if "p" not in c["given"]:
                c["H"] = 0
        if 4 * c.get("K", 1) <= V and work(c)["bytes"] <= most and c["N"] * c["V"] * c.get("shards", 1) <= 2 ** 30.5:
            return c


# ---- what a pass has to read and write -----------------------------------------------------------------
def work(c):
    n, e = c["N"] * c["V"], SIZE[c["type"]]
    index = 8 if c["index"] == "i64" else 4
    if c["kind"] == "distill":
        rows = c["K"] * (index + 8) + 28 + (index + 4 if c["targets"] else 0)
        return dict(bytes=n * e + c["N"] * rows, flops=4 * n)
    if c["kind"] == "distill_grad":
        rows = c["K"] * (index + 4) + 24 + (index + 4 if c["targets"] else 0)
        return dict(bytes=2 * n * e + c["N"] * rows, flops=4 * n)
    held = 0.625 * c["N"] * c["H"]      # places that count, on average
    bits = n / 8 if c["allowed"] is not None else 0
    if c["into"]:
        return dict(bytes=bits + n * (1 - c["allowed"]) * e, flops=n)
    if c["kind"] == "adjust_grad":
        return dict(bytes=n * (SIZE[c["out"]] + e) + bits + held * index, flops=2 * n)
    biases = c["N"] * BIASES * (index + 4) if "b" in c["given"] else 0
    return dict(bytes=n * (e + SIZE[c["out"]]) + bits + held * index + biases, flops=2 * n)


# ---- inputs --------------------------------------------------------------------------------------------
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _uniform(g, *shape):
    return torch.rand(*shape, generator=g, device="cuda")


def _tokens(g, shape, V, index):
    t = (torch.exp(_uniform(g, *shape).double() * math.log(V + 1.0)) - 1.0).floor().clamp_(0, V - 1)
    return t.to(torch.int64 if index == "i64" else torch.int32)


def _normal(g, rows, columns, type, size=1.0, tails=0.0):
    x = torch.empty(rows, columns, dtype=TYPES[type], device="cuda")
    step = max(1, (1 << 28) // max(1, columns))
    for at in range(0, rows, step):
        u = torch.randn(min(step, rows - at), columns, generator=g, device="cuda")
        x[at:at + step] = size * (u + tails * u ** 3 if tails else u)
    return x


def _distinct(g, N, V, K, index):
    """K different tokens in each row, in no order: one from each of K equal pieces of the vocabulary."""
    width = V // K
    t = torch.arange(K, device="cuda") * width + (_uniform(g, N, K) * width).long().clamp_(max=width - 1)
    return t.to(torch.int64 if index == "i64" else torch.int32)


def _prepare_distill(c, g):
    N, K, shards = c["N"], c["K"], c.get("shards", 1)
    V = c["V"] * shards
    x = _normal(g, N, V, c["type"], 1.8, 0.08)
    if c["masked"]:
        x.masked_fill_(_uniform(g, V) < c["masked"], float("-inf"))
    # the teacher's: between half and nearly all of the probability on its list, the largest first
    own_mass = torch.log(0.5 + 0.499 * _uniform(g, N, 1))
    q, order = (torch.log_softmax(2.0 * torch.randn(N, K, generator=g, device="cuda"), 1) + own_mass).sort(1, descending=True)
    t = _distinct(g, N, V, K, c["index"]).gather(1, order)
    level = math.log(V * (1.0 - 0.9 * c["masked"])) + 0.5 * (1.8 * c["scale"]) ** 2
    near = (level + 1.0 + q + 0.7 * torch.randn(N, K, generator=g, device="cuda")) / c["scale"]
    x.scatter_(1, t.long(), near.to(x.dtype))
    if K >= 4:
        t[5::16, K - K // 4:] = -1
        q[5::16, K - K // 4:] = float("-inf")
    c["vocab"], c["tokens"], c["teacher"] = V, t, q
    c["target"] = None
    if c["targets"]:
        c["target"] = _tokens(g, (N,), V, c["index"])
        c["target"][::3] = t[::3, 0]
        c["target"][::8] = -100
    c["logits"] = x
    if c["kind"] == "distill_grad":
        # what the forward pass left, and the gradients that reach it
        c["stats"] = _in_pieces(lambda rows: _left(c, rows)["stats"], c)
        size = 16.0 if c["type"] == "f16" else 1.0 / N     # a program that trains in f16 scales its loss
        c["d_loss"] = (0.5 + _uniform(g, N)) * size
        c["d_logp"] = -(0.5 + _uniform(g, N)) * 0.3 * size if c["targets"] else None
        c["first"] = c["shard"] * c["V"]
        if shards > 1:
            c["logits"] = x[:, c["first"]:c["first"] + c["V"]].contiguous()
    return c


def _bits(g, N, V, share):
    """A row's mask as words of 32 bits, token t in bit t % 32 of word t // 32."""
    words = (V + 31) // 32
    got = torch.empty(N, words, dtype=torch.int32, device="cuda")
    step = max(1, (1 << 27) // (words * 32))
    place = torch.arange(32, device="cuda")
    for at in range(0, N, step):
        n = min(step, N - at)
        bits = (_uniform(g, n, words, 32) < share).long() << place
        got[at:at + n] = bits.sum(2).to(torch.int32)    # (bit 31 is the sign: the low 32 bits are kept)
    return got


def prepare(case, seed):
    c, g = dict(case), _generator(seed)
    if c["kind"].startswith("distill"):
        return _prepare_distill(c, g)
    N, V, H = c["N"], c["V"], c["H"]
    c["logits"] = _normal(g, N, V, c["type"], 1.8, 0.08)
    for name in ("history", "lengths", "prompts", "repetition", "frequency", "presence", "bias_tokens", "bias", "words", "scale"):
        c[name] = None
    if "p" in c["given"]:
        c["history"] = _tokens(g, (N, H), V, c["index"])
        c["lengths"] = (H * (0.25 + 0.75 * _uniform(g, N))).ceil().to(torch.int32)
        c["prompts"] = (c["lengths"] * _uniform(g, N)).to(torch.int32)
        c["repetition"] = 1.0 + 0.3 * _uniform(g, N)
        c["frequency"], c["presence"] = _uniform(g, N), _uniform(g, N)
    if "b" in c["given"]:
        c["bias_tokens"] = _distinct(g, N, V, min(BIASES, V), c["index"])
        c["bias"] = 4.0 * torch.randn(N, c["bias_tokens"].shape[1], generator=g, device="cuda")
    if c["allowed"] is not None:
        c["words"] = _bits(g, N, V, c["allowed"])
    if c["scaled"]:
        c["scale"] = 0.5 + 1.5 * _uniform(g, N)
    if c["kind"] == "adjust_grad":
        c["grad"] = _normal(g, N, V, c["out"], 1e-2)
    return c


# ---- plain forms ---------------------------------------------------------------------------------------
def _in_pieces(f, c):
    """f of some rows at a time, put together (inputs' own statistics; a pass takes all rows at once)."""
    step = max(1, (1 << 28) // c["vocab"])
    return torch.cat([f(slice(at, at + step)) for at in range(0, c["N"], step)])


def _level(x):
    """A largest logit to subtract: 0 where there is none above -inf."""
    return torch.where(torch.isneginf(x), 0.0, x)


def _left(c, rows=slice(None)):
    x, t = c["logits"][rows].float(), c["tokens"][rows].long()
    N, V, scale, beta = x.shape[0], x.shape[1], c["scale"], c["beta"]
    lq = c["teacher"][rows].double()
    used = (t >= 0) & (t < V) & (lq > -math.inf)
    at = torch.where(used, t, 0)
    is_listed = torch.zeros(N, V + 1, dtype=torch.bool, device=x.device).scatter_(1, torch.where(used, t, V), True)[:, :V]
    rest = x.masked_fill(is_listed, -math.inf)
    others = rest.amax(1, keepdim=True)
    of_rest = torch.exp((rest - _level(others)) * scale).sum(1)
    x_k = torch.where(used, x.gather(1, at), -math.inf)
    largest = torch.maximum(others, x_k.amax(1, keepdim=True))
    d_k, d_out = (x_k - largest).double() * scale, (others - largest)[:, 0].double() * scale
    s_out = of_rest.double() * torch.exp(d_out)
    s = s_out + torch.exp(d_k).sum(1)
    log_s, log_s_out = torch.log(s), torch.log(of_rest)
    lp = torch.where(used, d_k - log_s[:, None], -math.inf)
    p, p_out = torch.exp(lp), s_out / s
    q = torch.exp(torch.where(used, lq, -math.inf))
    mass = q.sum(1, keepdim=True)
    if c["rest"]:
        r = 1.0 - mass[:, 0]
        r = torch.where((s_out > 0) & ((r >= LEAST_REST) | (beta == 1.0)), r.clamp(min=LEAST_REST), 0.0)
    else:
        q, r = q / mass.clamp(min=1e-300), torch.zeros_like(s)
    lq, lr, l_out = torch.log(q), torch.log(r), d_out + log_s_out.double() - log_s
    total = q.sum(1) + r
    if beta == 0.0:
        loss = torch.where(used, q * (lq - lp), 0.0).sum(1) + torch.where(r > 0, r * (lr - l_out), 0.0)
        pull, c_out = p * total[:, None] - q, total * p_out - r
    elif beta == 1.0:
        a, a_out = torch.where(used, lp - lq, 0.0), torch.where(s_out > 0, l_out - lr, 0.0)
        loss = (p * a).sum(1) + p_out * a_out
        pull, c_out = p * (a - loss[:, None]), p_out * (a_out - loss)
    else:
        m, m_out = beta * q + (1 - beta) * p, beta * r + (1 - beta) * p_out
        a = torch.where(p > 0, lp - torch.log(m), 0.0)
        a_out = torch.where(s_out > 0, l_out - torch.log(m_out), 0.0)
        to = torch.where(q > 0, q * (lq - torch.log(m)), 0.0).sum(1) + torch.where(r > 0, r * (lr - torch.log(m_out)), 0.0)
        mean = (p * a).sum(1) + p_out * a_out
        loss = beta * to + (1 - beta) * mean
        pull, c_out = (1 - beta) * p * (a - mean[:, None]), (1 - beta) * p_out * (a_out - mean)
    pull = torch.where(used, pull, 0.0)
    got = {"loss": loss.float(), "lse": (largest[:, 0].double() * scale + log_s).float(),
           "stats": torch.cat([largest, log_s[:, None].float(), others, log_s_out[:, None], c_out[:, None].float(), pull.float()], 1)}
    if c["target"] is not None:
        w = c["target"][rows].long()
        here = (w >= 0) & (w < V)
        got["logp"] = torch.where(here, (x.gather(1, torch.where(here, w, 0)[:, None]) - largest)[:, 0] * scale - log_s, 0.0).float()
    return got


def _distill_grad_plain(c):
    x, scale, stats = c["logits"].float(), c["scale"], c["stats"]
    V = x.shape[1]
    share = torch.exp((x - _level(stats[:, 2:3])) * scale - _level(stats[:, 3:4]))      # of what is not listed
    t = c["tokens"].long() - c["first"]
    here = (t >= 0) & (t < V) & (c["tokens"] >= 0)
    g = torch.cat([c["d_loss"][:, None] * stats[:, 4:5] * share, torch.zeros_like(x[:, :1])], 1)
    g.scatter_(1, torch.where(here, t, V), c["d_loss"][:, None] * stats[:, 5:])     # (the last column takes what is elsewhere)
    if c["target"] is not None:
        held = (c["target"] >= 0) & (c["target"] < c["vocab"])
        d = torch.where(held, c["d_logp"], 0.0)
        w = c["target"].long() - c["first"]
        g[:, :V] -= torch.exp((x - stats[:, 0:1]) * scale - stats[:, 1:2]).mul_(d[:, None])
        g.scatter_add_(1, torch.where(held & (w >= 0) & (w < V), w, V)[:, None], d[:, None])
    return (g[:, :V] * scale).to(c["logits"].dtype)


def _ruled_out(c):
    words = c["words"]
    bits = (words[:, :, None] >> torch.arange(32, dtype=torch.int32, device=words.device)) & 1
    return (bits == 0).reshape(words.shape[0], -1)[:, :c["V"]]


def _history(c):
    """How often each token is in a row's history behind the prompt, and whether it is there at all."""
    N, V, t = c["N"], c["V"], c["history"].long()
    place = torch.arange(t.shape[1], device=t.device)
    counts = place < c["lengths"][:, None]
    n = torch.zeros(N, V, device=t.device).scatter_add_(1, t, (counts & (place >= c["prompts"][:, None])).float())
    return n, torch.zeros(N, V, device=t.device).scatter_add_(1, t, counts.float()) > 0


def _adjust_plain(c):
    if c["into"]:
        return c["logits"].masked_fill_(_ruled_out(c), float("-inf"))
    y = c["logits"].float()
    if c["history"] is not None:
        n, there = _history(c)
        rep = c["repetition"][:, None]
        y = torch.where(there, torch.where(y > 0, y / rep, y * rep), y)
        y = y - c["frequency"][:, None] * n - c["presence"][:, None] * (n > 0)
    if c["bias"] is not None:
        y = y.scatter_add(1, c["bias_tokens"].long(), c["bias"])
    if c["scale"] is not None:
        y = y * c["scale"][:, None]
    if c["words"] is not None:
        y = torch.where(_ruled_out(c), -math.inf, y)
    return y.to(TYPES[c["out"]])


def _adjust_grad_plain(c):
    g = c["grad"].float()
    if c["scale"] is not None:
        g = g * c["scale"][:, None]
    if c["history"] is not None:
        there, rep = _history(c)[1], c["repetition"][:, None]
        g = torch.where(there, torch.where(c["logits"].float() > 0, g / rep, g * rep), g)
    if c["words"] is not None:
        g = torch.where(_ruled_out(c), 0.0, g)
    return g.to(c["logits"].dtype)


# ---- a pass --------------------------------------------------------------------------------------------
def _framework():
    import os
    import sys
    package = os.path.join(os.getcwd(), "hetu-galvatron_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    from galvatron_dp import operators
    return operators


_ops = None


def run(c):
    if own:
        return _run_own(c)
    kind = c["kind"]
    if kind == "distill":
        return _left(c)
    if kind == "distill_grad":
        return _distill_grad_plain(c)
    return _adjust_plain(c) if kind == "adjust" else _adjust_grad_plain(c)


def _run_own(c):
    global _ops
    ops = _ops = _ops or _framework()
    kind = c["kind"]
    if kind == "distill":
        r = ops.distillation(c["logits"], c["tokens"], c["teacher"], scale=c["scale"], beta=c["beta"], rest=c["rest"],
                             targets=c["target"], stats=True)
        got = {"loss": r.loss, "lse": r.lse, "stats": r.stats}
        if c["target"] is not None:
            got["logp"] = r.logp
        return got
    if kind == "distill_grad":
        return ops.distillation_grad(c["logits"], c["tokens"], c["stats"], c["d_loss"], scale=c["scale"], targets=c["target"],
                                     grad_logp=c["d_logp"], first=c["first"], vocab=c["vocab"])
    if kind == "adjust":
        return ops.adjust_logits(c["logits"], c["history"], lengths=c["lengths"], prompts=c["prompts"], repetition=c["repetition"],
                                 frequency=c["frequency"], presence=c["presence"], bias_tokens=c["bias_tokens"], bias=c["bias"],
                                 scale=c["scale"], allowed=c["words"], into=c["logits"] if c["into"] else None,
                                 dtype=TYPES[c["out"]])
    return ops.adjust_logits_grad(c["logits"], c["grad"], c["history"], lengths=c["lengths"], repetition=c["repetition"],
                                  scale=c["scale"], allowed=c["words"])


# ---- the definitions in 64 bits ------------------------------------------------------------------------
def exact(case, seed):
    c = prepare(case, seed)
    f = {"distill": _exact_distill, "distill_grad": _exact_distill_grad, "adjust": _exact_adjust, "adjust_grad": _exact_adjust}[c["kind"]]
    step = max(1, (1 << 26) // c["V"])
    parts = [f(c, slice(at, at + step)) for at in range(0, c["N"], step)]
    if isinstance(parts[0], dict):
        return {k: torch.cat([p[k] for p in parts]) for k in parts[0]}
    return torch.cat(parts)


def _exact_distill(c, rows):
    """Divergences of the two distributions over the list's tokens and the rest; their gradients by differentiating these."""
    ell = torch.log_softmax(c["logits"][rows].double() * c["scale"], 1)
    largest = c["logits"][rows].double().amax(1)
    t, lq = c["tokens"][rows].long(), c["teacher"][rows].double()
    out = {k: [] for k in ("loss", "lse", "stats")}
    n, V = ell.shape
    gone = (t < 0) | (t >= V) | torch.isneginf(lq)
    row = torch.arange(n, device=ell.device)[:, None].expand_as(t)
    others = ell.clone()
    others[row[~gone], t[~gone]] = -math.inf
    u = torch.cat([ell.gather(1, t.clamp(0, V - 1)).masked_fill(gone, -1e300), torch.logsumexp(others, 1)[:, None]], 1)
    of_others = others.amax(1, keepdim=True)
    of_others = torch.cat([c["logits"][rows].double().masked_fill(torch.isneginf(others), -math.inf).amax(1, keepdim=True), u[:, -1:] - of_others], 1)
    del others
    no_rest = torch.isneginf(u[:, -1:])
    u = u.masked_fill(torch.cat([torch.zeros_like(gone), no_rest], 1), -1e300).requires_grad_(True)
    lp = torch.log_softmax(u, 1)
    lq = lq.masked_fill(gone, -math.inf)
    if c["rest"]:
        left = 1.0 - lq.exp().sum(1, keepdim=True)
        none = no_rest if c["beta"] == 1.0 else no_rest | (left < LEAST_REST)
        left = left.clamp(min=LEAST_REST).log().masked_fill(none, -math.inf)
        lq = torch.cat([lq, left], 1)
    else:
        lq = torch.cat([lq - torch.logsumexp(lq, 1, keepdim=True), torch.full_like(lq[:, :1], -math.inf)], 1)
    there = ~torch.cat([gone, no_rest], 1)
    held = there & ~torch.isneginf(lq)
    lq = torch.where(held, lq, 0.0)
    q, p = torch.where(held, lq.exp(), 0.0), torch.where(there, lp.exp(), 0.0)
    beta = c["beta"]
    if beta == 0.0:
        loss = (q * (lq - torch.where(held, lp, 0.0))).sum(1)
    elif beta == 1.0:
        loss = (p * (torch.where(there, lp, 0.0) - lq)).sum(1)
    else:
        lm = torch.log(torch.where(there, beta * q + (1 - beta) * p, 1.0))
        loss = beta * (q * (lq - lm)).sum(1) + (1 - beta) * (p * (torch.where(there, lp, 0.0) - lm)).sum(1)
    d, = torch.autograd.grad(loss.sum(), u)
    with torch.no_grad():
        lse = torch.logsumexp(c["logits"][rows].double() * c["scale"], 1)
        stats = torch.cat([largest[:, None], (lse - largest * c["scale"])[:, None], of_others, torch.where(no_rest, 0.0, d[:, -1:]),
                           torch.where(gone, 0.0, d[:, :-1])], 1)
        out = {"loss": loss.detach(), "lse": lse, "stats": stats}
        if c["target"] is not None:
            w = c["target"][rows].long()
            out["logp"] = torch.where((w >= 0) & (w < V), ell.gather(1, w.clamp(0, V - 1)[:, None])[:, 0], 0.0)
    return out


def _exact_distill_grad(c, rows):
    x, s = c["logits"][rows].double(), c["stats"][rows].double()
    n, V = x.shape
    d = c["d_loss"][rows].double()[:, None]
    out = torch.exp(c["scale"] * (x - s[:, 2:3].clamp(min=-1e300)) - s[:, 3:4].clamp(min=-1e300)) * (s[:, 4:5] * d)
    out.masked_fill_(torch.isneginf(x), 0.0)
    row = torch.arange(n, device=x.device)
    t = c["tokens"][rows].long()
    local = t - c["first"]
    inside = (t >= 0) & (local >= 0) & (local < V)
    out[row[:, None].expand_as(t)[inside], local[inside]] = (s[:, 5:] * d)[inside]
    if c["target"] is not None:
        w = c["target"][rows].long()
        g = c["d_logp"][rows].double() * ((w >= 0) & (w < c["vocab"]))
        out -= g[:, None] * torch.exp(c["scale"] * (x - s[:, :1]) - s[:, 1:2])
        w = w - c["first"]
        inside = (w >= 0) & (w < V)
        out[row[inside], w[inside]] += g[inside]
    return out * c["scale"]


def _exact_adjust(c, rows):
    back = c["kind"] == "adjust_grad"
    x = c["logits"][rows].double()
    y = c["grad"][rows].double() if back else x.clone()
    n, V = x.shape
    of = lambda name: c[name][rows].double()[:, None]  # noqa: E731
    if c["history"] is not None:
        t = c["history"][rows].long()
        place = torch.arange(t.shape[1], device=x.device)[None]
        cell = t + V * torch.arange(n, device=x.device)[:, None]
        used = place < c["lengths"][rows][:, None]
        late = used & (place >= c["prompts"][rows][:, None])
        seen = torch.bincount(cell[used], minlength=n * V).view(n, V) > 0
        times = torch.bincount(cell[late], minlength=n * V).view(n, V).double()
        factor = torch.where(seen, torch.where(x > 0, 1.0 / of("repetition"), of("repetition")), 1.0)
        y *= factor
        if not back:
            y -= of("frequency") * times + of("presence") * torch.sign(times)
    if c["bias"] is not None:
        for i in range(c["bias_tokens"].shape[1]):
            y[torch.arange(n, device=x.device), c["bias_tokens"][rows, i].long()] += c["bias"][rows, i].double()
    if c["scale"] is not None:
        y *= of("scale")
    if c["words"] is not None:
        word = c["words"][rows].long()[:, torch.arange(V, device=x.device) // 32]
        y[(word >> (torch.arange(V, device=x.device) % 32)) % 2 == 0] = 0.0 if back else -math.inf
    return y
