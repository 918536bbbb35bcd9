"""Plain forms of the operators in 64 bits, on the CPU, and the bounds their float32 results keep, for the tests."""
import math

import torch

U = 2.0 ** -24                                   # half a unit of float32
HALF_UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
LEAST = {torch.float32: 2.0 ** -126, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -126}   # half the least step near 0


def rounded(ref, dtype):
    """What rounding once to dtype may add to |ref|."""
    return HALF_UNIT[dtype] * 1.01 * ref.abs() + LEAST[dtype]


def close(got, ref, bound, what=""):
    got, bound = got.detach().cpu().double(), bound.expand_as(ref) if isinstance(bound, torch.Tensor) else torch.full_like(ref, bound)
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    same = (got == ref) | (torch.isnan(got) & torch.isnan(ref))
    off = torch.where(same, 0.0, (got - ref).abs() - bound)
    bad = ~(off <= 0)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, first at {torch.nonzero(bad)[0].tolist()}: " \
                          f"{got[bad][0].item()} for {ref[bad][0].item()} within {bound[bad][0].item()}"


# ---- embedding ----
def held(tokens, first, rows):
    t = tokens.long().cpu().reshape(-1) - first
    return torch.where((t >= 0) & (t < rows), t, -1)


def embedding(tokens, weight, scale, first):
    t = held(tokens, first, weight.shape[0])
    y = torch.zeros(t.numel(), weight.shape[1], dtype=torch.float64)
    y[t >= 0] = weight.detach().cpu().double()[t[t >= 0]] * scale
    return y.reshape(*tokens.shape, weight.shape[1])


def embedding_grad(tokens, grad, rows, scale, first):
    """(sums, a bound on the error of float32 sums in any order)"""
    t = held(tokens, first, rows)
    g = grad.detach().cpu().double().reshape(t.numel(), grad.shape[-1])[t >= 0]
    t = t[t >= 0]
    dim = grad.shape[-1]
    total = torch.zeros(rows, dim, dtype=torch.float64).index_add_(0, t, g) * scale
    size = torch.zeros(rows, dim, dtype=torch.float64).index_add_(0, t, g.abs()) * abs(scale)
    count = torch.bincount(t, minlength=rows).double()[:, None]
    return total, (count + 2) * U * size


# ---- log probabilities ----
def logprobs(logits, tokens, scale):
    """logp, lse, entropy, log probabilities of all"""
    z = logits.detach().cpu().double() * scale
    lse = torch.logsumexp(z, -1)
    every = torch.where(torch.isinf(lse)[..., None], -math.inf, z - lse[..., None])
    p = every.exp()
    entropy = -torch.where(p > 0, p * every, torch.where(torch.isnan(p), p, 0.0)).sum(-1)
    t = tokens.long().cpu()
    here = (t >= 0) & (t < logits.shape[-1])
    logp = torch.where(here, every.gather(-1, torch.where(here, t, 0)[..., None])[..., 0], 0.0)
    return logp, lse, entropy, every


def logprob_bound(logits, scale):
    """Of lse, of a log probability, of the entropy.  An exponential is off by a unit of its own, and by its exponent's two
    roundings, whose average over p is at most 2 ln V units; a thread adds up at most V / 256 + 40 of them one after another
    and 20 sums are joined; lse, the largest logit times scale and the token's distance to it are rounded once each."""
    V = logits.shape[-1]
    z = logits.detach().cpu().double() * scale
    size = torch.where(torch.isfinite(z), z.abs(), 0.0).amax(-1)
    ln_v = math.log(max(V, 2))
    of_sum = U * (4 + 4 * ln_v + V / 256 + 60)
    return of_sum + 4 * U * (size + ln_v), of_sum + 8 * U * (2 * size + ln_v), of_sum * (2 + 2 * ln_v) + 8 * U * ln_v


def top_of(logits, k):
    """The k largest, equal ones by number; NaN as -inf."""
    x = logits.detach().cpu().double()
    x = torch.where(torch.isnan(x), -math.inf, x)
    return torch.sort(x, dim=-1, descending=True, stable=True)[1][..., :k]


def logprobs_grad(logits, tokens, lse, d_logp, scale, d_lse=None, entropy=None, d_entropy=None, top=None, d_top=None, first=0, vocab=None):
    """(gradient, sum of the sizes of its terms)"""
    f = lambda t: t.detach().cpu().double()   # noqa: E731
    x = f(logits)
    n, columns = x.shape
    q = x * scale - f(lse)[:, None]
    ruled_out = f(lse) < -1e5
    p = torch.where(ruled_out[:, None], 0.0, q.exp())
    t = tokens.long().cpu()
    d = torch.where((t >= 0) & (t < (vocab or columns)), f(d_logp), 0.0) if d_logp is not None else torch.zeros(n, dtype=torch.float64)
    coefficient, out = d.clone(), torch.zeros_like(x)
    size = torch.zeros_like(x)
    size_c = d.abs()

    def add(at, value):
        at = at - first
        inside = (at >= 0) & (at < columns) & ~ruled_out
        out[torch.arange(n)[inside], at[inside]] += value[inside]
        size[torch.arange(n)[inside], at[inside]] += value[inside].abs()

    add(t, d)
    if d_lse is not None:
        coefficient, size_c = coefficient - f(d_lse), size_c + f(d_lse).abs()
    if d_top is not None:
        for i in range(top.shape[1]):
            add(top[:, i].cpu(), f(d_top)[:, i])
            coefficient, size_c = coefficient + f(d_top)[:, i], size_c + f(d_top)[:, i].abs()
    out, size = out - p * coefficient[:, None], size + p * size_c[:, None]
    if d_entropy is not None:
        away = torch.where(p > 0, q + f(entropy)[:, None], 0.0)
        out, size = out - f(d_entropy)[:, None] * p * away, size + f(d_entropy).abs()[:, None] * p * (q.abs().clamp(max=1e9) + f(entropy).abs()[:, None])
    # p: the exponent's three roundings, each of at most (|x scale| + |lse| + |q|) U, and 2 U of its own; ten products and sums
    big = torch.where(p > 0, (x * scale).abs() + f(lse).abs()[:, None] + q.abs(), 0.0)
    return out * scale, size * scale * U * (16 + (d_top.shape[1] if d_top is not None else 0) + 3 * big)


# ---- residual join and norms ----
def norm(x, given, stats=None):
    """(output, normed without weight, mean, 1 / deviation); ``stats``: (mean, 1 / deviation) to be used instead"""
    if stats is None:
        mean = x.mean(-1, keepdim=True) if given.form == "layer" else torch.zeros_like(x[..., :1])
        rstd = 1 / ((x - mean).square().mean(-1, keepdim=True) + given.eps).sqrt()
    else:
        mean, rstd = stats
    hat = (x - mean) * rstd
    y = hat if given.weight is None else hat * given.weight.detach().cpu().double()
    return (y if given.bias is None else y + given.bias.detach().cpu().double()), hat, mean, rstd


def gate_rows(gate, n, dim):
    g = gate.detach().cpu().double().reshape(-1, dim)
    return g.repeat_interleave(n // g.shape[0], 0)


def residual_norm(residual, block, post, pre, gate, residual_scale, block_scale):
    dim = residual.shape[-1]
    r = residual.detach().cpu().double().reshape(-1, dim) * residual_scale
    if block is not None:
        b = block.detach().cpu().double().reshape(-1, dim)
        b = norm(b, post)[0] if post else b
        r = r + block_scale * (b * gate_rows(gate, b.shape[0], dim) if gate is not None else b)
    return r, (norm(r, pre)[0] if pre else None)


def residual_norm_grad(stream, block, stats, d_normed, d_stream, post, pre, gate, residual_scale, block_scale):
    """{name: (gradient, sum of the sizes of the terms it is added up from)}"""
    dim = stream.shape[-1]
    f = lambda t: t.detach().cpu().double().reshape(-1, dim)   # noqa: E731
    s = stats.cpu().double()
    got = {}

    def back(d, size, hat, given, rstd):
        w = 1.0 if given.weight is None else given.weight.detach().cpu().double()
        u, size = d * w, size * (w.abs() if isinstance(w, torch.Tensor) else w)
        out = u - hat * (u * hat).mean(-1, keepdim=True)
        of = size + hat.abs() * (size * hat.abs()).mean(-1, keepdim=True)
        if given.form == "layer":
            out, of = out - u.mean(-1, keepdim=True), of + size.mean(-1, keepdim=True)
        return out * rstd, of * rstd

    def off(x, mean, rstd):      # hat's own size where x and the mean cancel
        return (x.abs() + mean.abs()) * rstd

    total = f(d_stream) if d_stream is not None else torch.zeros_like(f(stream))
    size = total.abs()
    if pre:
        hat, of_hat = norm(f(stream), pre, (s[:, 2:3], s[:, 3:4]))[1], off(f(stream), s[:, 2:3], s[:, 3:4])
        dh = f(d_normed)
        got["pre_weight"], got["pre_bias"] = ((dh * hat).sum(0), (dh.abs() * of_hat).sum(0)), (dh.sum(0), dh.abs().sum(0))
        more, of = back(dh, dh.abs(), hat, pre, s[:, 3:4])
        total, size = total + more, size + of + more.abs() + (of_hat - hat.abs()) * (dh * hat).abs().mean(-1, keepdim=True) * s[:, 3:4]
    got["residual"] = total * residual_scale, size * residual_scale
    if block is None:
        return got
    d, size = total * block_scale, size * block_scale
    b, hat = f(block), None
    of_b = b.abs()
    if post:
        of_hat = off(b, s[:, 0:1], s[:, 1:2])
        b, hat, _, _ = norm(b, post, (s[:, 0:1], s[:, 1:2]))
        of_b = b.abs() + of_hat * (1.0 if post.weight is None else post.weight.cpu().double().abs())
    if gate is not None:
        groups = gate.reshape(-1, dim).shape[0]
        got["gate"] = tuple(t.reshape(groups, -1, dim).sum(1).reshape(gate.shape) for t in (d * b, size * of_b))
        d, size = d * gate_rows(gate, d.shape[0], dim), size * gate_rows(gate, d.shape[0], dim).abs()
    if post:
        got["post_weight"], got["post_bias"] = ((d * hat).sum(0), (size * of_hat).sum(0)), (d.sum(0), size.sum(0))
        d, size = back(d, size, hat, post, s[:, 1:2])
    got["block"] = d, size
    return got
