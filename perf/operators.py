"""Measured cases of the operators at a model's two ends: what lies before the first layer and behind the last.

A strategy search prices these parts per vocabulary-parallel degree; a training or scoring program runs them:

* ``embed``         rows of the embedding table for given tokens, scaled; a shard of the table gives zeros for the
                    tokens that other shards hold.
* ``embed_grad``    the table's gradient: the gradients of all places that hold the same token, added up.  ``into``:
                    added to the float32 buffer in which a program gathers the gradients of its micro batches.
* ``logprob``       log probabilities of given tokens, the entropy of each row and the ``top`` most likely tokens.
* ``logprob_grad``  the gradient with respect to the logits, from gradients of log probabilities (and of entropies).
* ``norm``          a block's output, normed and gated, joined with the residual stream, and the norm of the sum that
                    the next block (or the head) reads.
* ``norm_grad``     the gradients of stream, block output, weights, biases and gate.

Tokens: small numbers are frequent, as in a vocabulary that was built by merges: P(t) goes by 1 / (t + 1).  Logits: a
wide normal distribution with heavy tails, so that a few stand out; ``masked``: the share of the vocabulary that a grammar rules out
(-inf).  Types: of the table, the logits or the block; ``stream`` of the residual stream.
"""
import math

import numpy as np
import torch

own = False     # False: plain forms.  True: the calls that a user makes of the framework

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZE = {"bf16": 2, "f16": 2, "f32": 4}


def _embed(name, N, R, D, type, scale=1.0, shards=1, shard=0, index="i64"):
    return dict(name=name, kind="embed", N=N, R=R, D=D, type=type, scale=scale, shards=shards, shard=shard, index=index)


def _embed_grad(name, N, R, D, type, scale=1.0, shards=1, shard=0, index="i64", into=False):
    return dict(_embed(name, N, R, D, type, scale, shards, shard, index), kind="embed_grad", into=into)


def _logprob(name, N, V, type, top, masked=0.0, scale=1.0, index="i64"):
    return dict(name=name, kind="logprob", N=N, V=V, type=type, top=top, masked=masked, scale=scale, index=index)


def _logprob_grad(name, N, V, type, entropy, masked=0.0, scale=1.0, index="i64"):
    return dict(name=name, kind="logprob_grad", N=N, V=V, type=type, entropy=entropy, masked=masked, scale=scale, index=index)


def _norm(name, T, D, type, stream, form, post, gates, kind="norm"):
    return dict(name=name, kind=kind, T=T, D=D, type=type, stream=stream, form=form, post=post, gates=gates)


def listed():
    return [
        # one decoding step of 64 requests: the next tokens' rows, scaled
        _embed("embed_decode", 64, 50257, 1024, "f16", scale=32.0),
        # a micro batch of 8 x 4096 tokens, 2-way vocabulary parallel: half the table, zeros for the rest
        _embed("embed_shard", 32768, 64128, 4096, "bf16", shards=2, shard=0),
        # a short fine-tuning batch, odd width, everything in float32
        _embed_grad("embed_grad_short", 777, 32003, 1023, "f32", scale=32.0),
        # the whole table's gradient of a micro batch of 8 x 4096 tokens
        _embed_grad("embed_grad_whole", 32768, 128256, 4096, "bf16"),
        # an eighth of the table, gathered over micro batches in float32
        _embed_grad("embed_grad_shard", 16384, 19008, 5120, "bf16", shards=8, shard=0, index="i32", into=True),
        # one decoding step of 16 requests with the 20 most likely tokens, a grammar leaves half of the vocabulary
        _logprob("logprob_decode", 16, 128256, "bf16", 20, masked=0.5, scale=1.25),
        # a long prompt scored with 5 alternatives a token, odd vocabulary, float32 logits
        _logprob("logprob_score", 4096, 50257, "f32", 5),
        # the loss of a training batch: 8192 tokens, log probabilities and entropy alone
        _logprob("logprob_train", 8192, 128256, "bf16", 0),
        # ... and its gradient
        _logprob_grad("logprob_grad_train", 8192, 128256, "bf16", False),
        # a policy gradient with an entropy bonus on a short batch, odd vocabulary
        _logprob_grad("logprob_grad_policy", 517, 32003, "f16", True, scale=0.8),
        # one decoding step of 8 requests: join and norm, a gate per channel
        _norm("norm_decode", 8, 4096, "bf16", "bf16", "rms", True, 1),
        # the gradient of a micro batch of 4 x 4096 tokens, float32 stream, a gate per sequence, norms with mean and bias
        _norm("norm_grad_train", 16384, 3584, "bf16", "f32", "layer", True, 4, kind="norm_grad"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    most = 4.2e9    # bytes of the largest listed case
    while True:
        kind = rng.choice(["embed", "embed_grad", "embed_grad", "logprob", "logprob", "logprob_grad", "norm", "norm_grad"])
        type, index = rng.choice(["bf16", "bf16", "f16", "f32"]), rng.choice(["i64", "i32"])
        if kind in ("embed", "embed_grad"):
            shards = rng.choice([1, 1, 2, 8])
            R = rng.choice([_log(rng, 500, 160000), 128 * _log(rng, 8, 1200)])
            D = rng.choice([_log(rng, 64, 8192), 64 * _log(rng, 1, 128), 256 * _log(rng, 2, 32)])
            c = dict(kind=kind, N=_log(rng, 1, 65536), R=R, D=D, type=type, scale=rng.choice([1.0, round(D ** 0.5, 3)]),
                     shards=shards, shard=rng.randrange(shards), index=index)
            if kind == "embed_grad":
                c["into"] = rng.random() < 0.4
        elif kind in ("logprob", "logprob_grad"):
            V = rng.choice([_log(rng, 500, 262144), 128 * _log(rng, 8, 2048)])
            c = dict(kind=kind, N=_log(rng, 1, 32768), V=V, type=type, masked=rng.choice([0.0, 0.0, 0.5, 0.99]),
                     scale=rng.choice([1.0, 1.0, 1.25, 0.8]), index=index)
            if kind == "logprob":
                c["top"] = rng.choice([0, 0, 1, 5, 20])
            else:
                c["entropy"] = rng.random() < 0.5
        else:
            D = rng.choice([_log(rng, 64, 8192), 64 * _log(rng, 1, 128), 256 * _log(rng, 2, 32)])
            gates = rng.choice([0, 1, 1, 4])
            T = _log(rng, 1, 65536)
            c = dict(kind=kind, T=T * (4 if gates == 4 else 1), D=D, type=type, stream=rng.choice([type, type, "f32"]),
                     form=rng.choice(["rms", "rms", "layer"]), post=rng.random() < 0.6, gates=gates)
        if 3072 not in c.values() and work(c)["bytes"] <= most:
            return c


# ---- what a pass has to read and write -----------------------------------------------------------------
def _chances(c):
    """P(token) for the tokens that the case's shard holds."""
    V = c["R"] * c["shards"]
    t = np.arange(c["shard"] * c["R"], (c["shard"] + 1) * c["R"], dtype=np.float64)
    return np.log1p(1.0 / (t + 1.0)) / math.log(V + 1.0)


def _held(c):
    """(expected places whose token the shard holds, expected different tokens among them)"""
    p = _chances(c)
    return c["N"] * float(p.sum()), float(-np.expm1(c["N"] * np.log1p(-p)).sum())


def work(c):
    kind, e = c["kind"], SIZE[c["type"]]
    if kind in ("embed", "embed_grad"):
        places, tokens = _held(c)
        ids = c["N"] * (8 if c["index"] == "i64" else 4)
        if kind == "embed":
            return dict(bytes=ids + (tokens + c["N"]) * c["D"] * e, flops=c["N"] * c["D"])
        out = 2 * tokens * c["D"] * 4 if c["into"] else c["R"] * c["D"] * e
        return dict(bytes=ids + places * c["D"] * e + out, flops=places * c["D"])
    if kind in ("logprob", "logprob_grad"):
        n, ids = c["N"] * c["V"], c["N"] * (8 if c["index"] == "i64" else 4)
        if kind == "logprob":
            return dict(bytes=n * e + ids + c["N"] * (12 + 12 * c["top"]), flops=6 * n)
        return dict(bytes=2 * n * e + ids + 8 * c["N"], flops=6 * n)
    n, s = c["T"] * c["D"], SIZE[c["stream"]]
    if kind == "norm":
        return dict(bytes=2 * n * (e + s), flops=(12 if c["post"] else 8) * n)
    return dict(bytes=n * (3 * e + 3 * s), flops=(30 if c["post"] else 16) * n)


# ---- inputs --------------------------------------------------------------------------------------------
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _tokens(g, N, V, index):
    u = torch.rand(N, generator=g, device="cuda", dtype=torch.float64)
    t = (torch.exp(u * math.log(V + 1.0)) - 1.0).floor().clamp_(0, V - 1)
    return t.to(torch.int64 if index == "i64" else torch.int32)


def _normal(g, rows, columns, type, size=1.0, tails=0.0):
    x = torch.empty(rows, columns, dtype=TYPES[type], device="cuda")
    step = max(1, (1 << 28) // max(1, columns))
    for at in range(0, rows, step):
        u = torch.randn(min(step, rows - at), columns, generator=g, device="cuda")
        x[at:at + step] = size * (u + tails * u ** 3 if tails else u)
    return x


def prepare(case, seed):
    c, g = dict(case), _generator(seed)
    if c["kind"] in ("embed", "embed_grad"):
        c["first"] = c["shard"] * c["R"]
        c["tokens"] = _tokens(g, c["N"], c["R"] * c["shards"], c["index"])
        if c["kind"] == "embed":
            c["weight"] = _normal(g, c["R"], c["D"], c["type"], 0.02)
        else:
            c["grad"] = _normal(g, c["N"], c["D"], c["type"], 1e-2)
            if c["into"]:
                c["main"] = _normal(g, c["R"], c["D"], "f32", 1e-2)
        return c
    if c["kind"] in ("logprob", "logprob_grad"):
        N, V = c["N"], c["V"]
        c["logits"] = x = _normal(g, N, V, c["type"], 1.8, 0.08)
        c["tokens"] = t = _tokens(g, N, V, c["index"])
        if c["masked"]:
            out = torch.rand(V, generator=g, device="cuda") < c["masked"]
            out[t.long()] = False
            x.masked_fill_(out, float("-inf"))
        if c["kind"] == "logprob_grad":
            # what the forward pass left, and the gradients that reach it; one row in eight is no target
            c["lse"], c["entropy_of"] = _left(x, c["scale"])
            size = 1.0 if c["type"] == "f16" else 1.0 / N      # a program that trains in f16 scales its loss
            c["d_logp"] = torch.randn(N, generator=g, device="cuda") * size
            c["d_entropy"] = torch.randn(N, generator=g, device="cuda") * (0.01 * size)
            t[::8] = -100
        return c
    T, D, type, stream = c["T"], c["D"], c["type"], c["stream"]
    c["residual"], c["block"] = _normal(g, T, D, stream), _normal(g, T, D, type, 0.5)
    vector = lambda at: (at + 0.1 * torch.randn(D, generator=g, device="cuda")).to(TYPES[type])  # noqa: E731
    c["pre_weight"], c["pre_bias"] = vector(1.0), vector(0.0) if c["form"] == "layer" else None
    c["post_weight"] = vector(1.0) if c["post"] else None
    c["post_bias"] = vector(0.0) if c["post"] and c["form"] == "layer" else None
    c["gate"] = _normal(g, c["gates"], D, type, 0.5) if c["gates"] else None
    c["residual_scale"], c["block_scale"], c["eps"] = 0.98, 1.4, 1e-5
    if c["kind"] == "norm_grad":
        c["stream_out"], _, c["stats"] = _join(c)
        c["d_normed"], c["d_stream"] = _normal(g, T, D, type, 1e-2), _normal(g, T, D, stream, 1e-2)
        del c["residual"]
    return c


# ---- plain forms ---------------------------------------------------------------------------------------
def _left(x, scale):
    """Log of the sum of exponentials and entropy of each row, float32, some rows at a time."""
    lse, entropy = torch.empty(x.shape[0], device=x.device), torch.empty(x.shape[0], device=x.device)
    step = max(1, (1 << 28) // x.shape[1])
    for at in range(0, x.shape[0], step):
        z = x[at:at + step].float() * scale
        top = z.amax(1, keepdim=True)
        e = torch.exp(z - top)
        s = e.sum(1)
        lse[at:at + step] = top[:, 0] + torch.log(s)
        entropy[at:at + step] = torch.log(s) - (e * torch.where(e > 0, z - top, 0.0)).sum(1) / s
    return lse, entropy


def _logprob_plain(c):
    x = c["logits"].float()
    z = x * c["scale"]
    top = z.amax(1, keepdim=True)
    e = torch.exp(z - top)
    s = e.sum(1)
    log_s = torch.log(s)
    entropy = log_s - (e * torch.where(e > 0, z - top, 0.0)).sum(1) / s
    lse = top[:, 0] + log_s
    got = {"logp": z.gather(1, c["tokens"].long()[:, None])[:, 0] - lse, "lse": lse, "entropy": entropy}
    if c["top"]:
        at = torch.sort(x, dim=1, descending=True, stable=True)[1][:, :c["top"]]
        got["top_logp"], got["top_tokens"] = z.gather(1, at) - lse[:, None], at
    return got


def _logprob_grad_plain(c):
    z = c["logits"].float() * c["scale"]
    t = c["tokens"].long()
    held = (t >= 0) & (t < c["V"])
    d = torch.where(held, c["d_logp"], 0.0)
    q = z - c["lse"][:, None]
    p = torch.exp(q)
    g = -d[:, None] * p
    if c["entropy"]:
        g = g - c["d_entropy"][:, None] * torch.where(p > 0, p * (q + c["entropy_of"][:, None]), 0.0)
    g.scatter_add_(1, torch.where(held, t, 0)[:, None], d[:, None])
    return (g * c["scale"]).to(c["logits"].dtype)


def _normed(x, form, weight, bias, eps):
    mean = x.mean(1, keepdim=True) if form == "layer" else torch.zeros_like(x[:, :1])
    rstd = torch.rsqrt((x - mean).square().mean(1, keepdim=True) + eps)
    y = (x - mean) * rstd * weight.float()
    return y + bias.float() if bias is not None else y, mean, rstd


def _rows_of(gate, T):
    """A gate for each row: a gate serves T / (number of gates) rows in turn."""
    return gate.float().repeat_interleave(T // gate.shape[0], 0)


def _join(c):
    b, T = c["block"].float(), c["T"]
    stats = torch.zeros(T, 4, device=b.device)
    if c["post"]:
        b, mean, rstd = _normed(b, c["form"], c["post_weight"], c["post_bias"], c["eps"])
        stats[:, 0:1], stats[:, 1:2] = mean, rstd
    if c["gate"] is not None:
        b = b * _rows_of(c["gate"], T)
    r = c["residual"].float() * c["residual_scale"] + b * c["block_scale"]
    h, mean, rstd = _normed(r, c["form"], c["pre_weight"], c["pre_bias"], c["eps"])
    stats[:, 2:3], stats[:, 3:4] = mean, rstd
    return r.to(TYPES[c["stream"]]), h.to(TYPES[c["type"]]), stats


def _norm_back(dy, hat, rstd, weight, form):
    """Gradient of a norm's input, from that of its output, the normed input without weight, and 1 / deviation."""
    g = dy * weight.float()
    d = g - hat * (g * hat).mean(1, keepdim=True)
    if form == "layer":
        d = d - g.mean(1, keepdim=True)
    return d * rstd


def _norm_grad_plain(c):
    form, T, kind = c["form"], c["T"], TYPES[c["type"]]
    mean_b, rstd_b, mean_r, rstd_r = (c["stats"][:, i:i + 1] for i in range(4))
    dh, b = c["d_normed"].float(), c["block"].float()
    hat_r = (c["stream_out"].float() - mean_r) * rstd_r
    got = {"pre_weight": (dh * hat_r).sum(0).to(kind)}
    if c["pre_bias"] is not None:
        got["pre_bias"] = dh.sum(0).to(kind)
    dr = c["d_stream"].float() + _norm_back(dh, hat_r, rstd_r, c["pre_weight"], form)
    got["residual"] = (dr * c["residual_scale"]).to(TYPES[c["stream"]])
    dn, n = dr * c["block_scale"], b
    if c["post"]:
        hat_b = (b - mean_b) * rstd_b
        n = hat_b * c["post_weight"].float()
        n = n + c["post_bias"].float() if c["post_bias"] is not None else n
    if c["gate"] is not None:
        got["gate"] = (dn * n).reshape(c["gates"], T // c["gates"], c["D"]).sum(1).to(kind)
        dn = dn * _rows_of(c["gate"], T)
    if c["post"]:
        got["post_weight"] = (dn * hat_b).sum(0).to(kind)
        if c["post_bias"] is not None:
            got["post_bias"] = dn.sum(0).to(kind)
        dn = _norm_back(dn, hat_b, rstd_b, c["post_weight"], form)
    got["block"] = dn.to(kind)
    return got


def _embed_plain(c):
    t = c["tokens"].long() - c["first"]
    held = (t >= 0) & (t < c["R"])
    return (c["weight"][torch.where(held, t, 0)].float() * c["scale"] * held[:, None]).to(c["weight"].dtype)


def _embed_grad_plain(c):
    t = c["tokens"].long() - c["first"]
    held = (t >= 0) & (t < c["R"])
    add = c["grad"].float() * c["scale"] * held[:, None]
    total = torch.zeros(c["R"], c["D"], device=add.device).index_add_(0, torch.where(held, t, 0), add)
    if c["into"]:
        return c["main"].add_(total)
    return total.to(c["grad"].dtype)


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
    if kind == "embed":
        return _embed_plain(c)
    if kind == "embed_grad":
        return _embed_grad_plain(c)
    if kind == "logprob":
        return _logprob_plain(c)
    if kind == "logprob_grad":
        return _logprob_grad_plain(c)
    if kind == "norm":
        return _join(c)[:2]
    return _norm_grad_plain(c)


def _run_own(c):
    global _ops
    ops = _ops = _ops or _framework()
    kind = c["kind"]
    if kind == "embed":
        return ops.embedding(c["tokens"], c["weight"], scale=c["scale"], first=c["first"])
    if kind == "embed_grad":
        return ops.embedding_grad(c["tokens"], c["grad"], c["R"], scale=c["scale"], first=c["first"],
                                  into=c["main"] if c["into"] else None)
    if kind == "logprob":
        r = ops.token_logprobs(c["logits"], c["tokens"], scale=c["scale"], entropy=True, top=c["top"])
        got = {"logp": r.logp, "lse": r.lse, "entropy": r.entropy}
        if c["top"]:
            got["top_logp"], got["top_tokens"] = r.top_logp, r.top_tokens
        return got
    if kind == "logprob_grad":
        more = dict(entropy=c["entropy_of"], grad_entropy=c["d_entropy"]) if c["entropy"] else {}
        return ops.token_logprobs_grad(c["logits"], c["tokens"], c["lse"], c["d_logp"], scale=c["scale"], **more)
    pre = ops.Norm(c["form"], c["pre_weight"], c["pre_bias"], c["eps"])
    post = ops.Norm(c["form"], c["post_weight"], c["post_bias"], c["eps"]) if c["post"] else None
    shared = dict(post=post, pre=pre, gate=c["gate"], residual_scale=c["residual_scale"], block_scale=c["block_scale"])
    if kind == "norm":
        r = ops.residual_norm(c["residual"], c["block"], **shared)
        return r.stream, r.normed
    r = ops.residual_norm_grad(c["stream_out"], c["block"], c["stats"], c["d_normed"], c["d_stream"], **shared)
    got = {"residual": r.residual, "block": r.block, "pre_weight": r.pre_weight}
    for name in ("pre_bias", "post_weight", "post_bias", "gate"):
        if getattr(r, name) is not None:
            got[name] = getattr(r, name)
    return got




# ---- the definitions in 64 bits ------------------------------------------------------------------------
def exact(case, seed):
    c = prepare(case, seed)
    kind, f = c["kind"], torch.float64
    if kind in ("embed", "embed_grad"):
        t = c["tokens"].long()
        inside = torch.nonzero((t >= c["first"]) & (t < c["first"] + c["R"]))[:, 0]
        rows = t[inside] - c["first"]
        if kind == "embed":
            y = torch.zeros(c["N"], c["D"], dtype=f, device="cuda")
            y[inside] = c["weight"].index_select(0, rows).to(f) * c["scale"]
            return y
        w = c["main"].to(f) if c["into"] else torch.zeros(c["R"], c["D"], dtype=f, device="cuda")
        # a sum for each token: places in the order of their tokens, differences of running sums per block of columns
        order = torch.argsort(rows, stable=True)
        which, count = torch.unique_consecutive(rows[order], return_counts=True)
        end = torch.cumsum(count, 0)
        for at in range(0, c["D"], 512):
            run_ = torch.cumsum(c["grad"][:, at:at + 512].index_select(0, inside[order]).to(f), 0)
            run_ = torch.cat([torch.zeros_like(run_[:1]), run_])
            w[which, at:at + 512] += c["scale"] * (run_[end] - run_[end - count])
        return w
    if kind in ("logprob", "logprob_grad"):
        step = max(1, (1 << 27) // c["V"])
        parts = [(_exact_logprob if kind == "logprob" else _exact_logprob_grad)(c, slice(at, at + step))
                 for at in range(0, c["N"], step)]
        if kind == "logprob_grad":
            return torch.cat(parts)
        return {k: None if k == "top_tokens" else torch.cat([p[k] for p in parts]) for k in parts[0]}
    return _exact_norm(c) if kind == "norm" else _exact_norm_grad(c)


def _exact_logprob(c, rows):
    z = c["logits"][rows].to(torch.float64) * c["scale"]
    logp = torch.log_softmax(z, 1)
    p = logp.exp()
    got = {"logp": logp.gather(1, c["tokens"][rows].long()[:, None])[:, 0], "lse": torch.logsumexp(z, 1),
           "entropy": -torch.where(p > 0, p * logp, 0.0).sum(1)}
    if c["top"]:
        got["top_logp"], got["top_tokens"] = logp.topk(c["top"], 1)[0], None
    return got


def _exact_logprob_grad(c, rows):
    x = c["logits"][rows].to(torch.float64)
    share = torch.exp(x * c["scale"] - c["lse"][rows].double()[:, None])
    t, d = c["tokens"][rows].long(), c["d_logp"][rows].double()
    d = d * ((t >= 0) & (t < c["V"]))
    hit = torch.zeros_like(x)
    hit[torch.arange(len(t), device="cuda"), t.clamp(0, c["V"] - 1)] = 1.0
    out = d[:, None] * (hit - share)
    if c["entropy"]:
        away = (x * c["scale"]).clamp(min=-1e300) - c["lse"][rows].double()[:, None] + c["entropy_of"][rows].double()[:, None]
        out -= c["d_entropy"][rows].double()[:, None] * share * away
    return out * c["scale"]


def _exact_layer(x, c, which):
    """(output, the input brought to mean and deviation) of one of the two norms"""
    given = c["stats"].double() if "stats" in c else None
    if given is not None:
        at = 0 if which == "post" else 2
        hat = (x - given[:, at:at + 1]) * given[:, at + 1:at + 2]
    elif c["form"] == "layer":
        hat = (x - x.mean(1, keepdim=True)) / (x.var(1, unbiased=False, keepdim=True) + c["eps"]).sqrt()
    else:
        hat = x / ((x * x).mean(1, keepdim=True) + c["eps"]).sqrt()
    y = hat * c[which + "_weight"].double()
    return (y if c[which + "_bias"] is None else y + c[which + "_bias"].double()), hat


def _exact_gate(c):
    if c["gate"] is None:
        return torch.ones(1, 1, 1, dtype=torch.float64, device="cuda")
    return c["gate"].double()[:, None, :]


def _exact_norm(c):
    T, D = c["T"], c["D"]
    b = c["block"].double()
    n = _exact_layer(b, c, "post")[0] if c["post"] else b
    gate = _exact_gate(c)
    r = c["residual_scale"] * c["residual"].double() + c["block_scale"] * (n.view(gate.shape[0], -1, D) * gate).view(T, D)
    return r, _exact_layer(r, c, "pre")[0]


def _exact_norm_grad(c):
    T, D = c["T"], c["D"]
    gate, stats = _exact_gate(c), c["stats"].double()

    def through(g, hat, rstd):
        inner = g - hat * ((g * hat).sum(1, keepdim=True) / D)
        if c["form"] == "layer":
            inner = inner - g.sum(1, keepdim=True) / D
        return inner * rstd

    dh = c["d_normed"].double()
    hat = _exact_layer(c["stream_out"].double(), c, "pre")[1]
    got = {"pre_weight": torch.einsum("td,td->d", dh, hat)}
    if c["pre_bias"] is not None:
        got["pre_bias"] = dh.sum(0)
    total = through(dh * c["pre_weight"].double(), hat, stats[:, 3:4]) + c["d_stream"].double()
    got["residual"] = c["residual_scale"] * total
    total = c["block_scale"] * total
    b = c["block"].double()
    n, hat = _exact_layer(b, c, "post") if c["post"] else (b, None)
    if c["gate"] is not None:
        got["gate"] = (total * n).view(gate.shape[0], -1, D).sum(1)
    total = (total.view(gate.shape[0], -1, D) * gate).view(T, D)
    if c["post"]:
        got["post_weight"] = (total * hat).sum(0)
        if c["post_bias"] is not None:
            got["post_bias"] = total.sum(0)
        total = through(total * c["post_weight"].double(), hat, stats[:, 1:2])
    got["block"] = total
    return got
