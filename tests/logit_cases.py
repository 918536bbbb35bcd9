"""Plain forms of the operators on logits in 64 bits, on the CPU, and the bounds their float32 results keep, for the tests."""
import math

import torch

from operator_cases import U, close, rounded   # noqa: F401

F64 = torch.float64
LEAST_REST = 2.0 ** -22


def f64(t):
    return t.detach().cpu().to(F64)


def of_sum(V):
    """Relative error of a float32 sum of V exponentials.  Each is off by a unit of its own and by its exponent's two roundings, whose average over
    the sum is at most 2 ln V units; a thread adds up at most V / 256 + 40 of them one after another and 20 sums are joined."""
    return U * (4 + 4 * math.log(max(V, 2)) + V / 256 + 60)


# ---- distillation ----
def listed_of(tokens, teacher, vocab):
    """Of each row {token: sum of q} over its used places, in 64 bits (q as logarithms)."""
    rows = []
    for ts, ls in zip(tokens.long().cpu().tolist(), f64(teacher).tolist()):
        got = {}
        for t, v in zip(ts, ls):
            if 0 <= t < vocab and v != -math.inf:
                got.setdefault(t, []).append(v)
        rows.append({t: (v[0] if len(v) == 1 else math.log(sum(math.exp(a) for a in v))) for t, v in got.items()})
    return rows


def distill_row(z, listed, beta, rest):
    """Loss of one row z (float64, differentiable), of buckets; and (p, q, ln p - what it is held against) of each, the rest last."""
    ts = sorted(listed)
    if bool(torch.isneginf(z).all()) or (not rest and not ts):
        return z.sum() * 0.0 if torch.isfinite(z).all() else torch.zeros((), dtype=F64), None
    lse = torch.logsumexp(z, 0)
    lp = [z[t] - lse for t in ts]
    others = torch.ones_like(z, dtype=torch.bool)
    others[ts] = False
    lq = [listed[t] for t in ts]
    have_rest = bool((z[others] > -math.inf).any()) or bool(torch.isnan(z[others]).any())
    if rest:
        r = 1.0 - sum(math.exp(v) for v in lq)
        if r < LEAST_REST:
            r = LEAST_REST if beta == 1.0 else 0.0
        lr = math.log(r) if r > 0 else -math.inf if r == 0 else math.nan
    else:
        norm = math.log(sum(math.exp(v - max(lq)) for v in lq)) + max(lq)
        lq = [v - norm for v in lq]
        lr = -math.inf
    if have_rest:
        lp.append(torch.logsumexp(z[others], 0) - lse)
        lq.append(lr)
    loss = torch.zeros((), dtype=F64)
    shown = []
    for a, b in zip(lp, lq):
        p, q = a.exp(), math.exp(b)
        if beta == 0.0:
            if q != 0.0:
                loss = loss + q * (b - a)
            shown.append((p.item(), q, 0.0))
        elif beta == 1.0:
            if p.item() != 0.0:
                loss = loss + p * (a - b)
            shown.append((p.item(), q, (a - b).item() if p.item() != 0 else 0.0))
        else:
            m = torch.log(beta * q + (1 - beta) * p)
            if q != 0.0:
                loss = loss + beta * q * (b - m)
            if p.item() != 0.0:
                loss = loss + (1 - beta) * p * (a - m)
            shown.append((p.item(), q, (a - m).item() if p.item() != 0 else 0.0))
    return loss, shown


def distillation(logits, tokens, teacher, scale, beta, rest, targets=None):
    """(loss, lse, logp, d loss / d z [n, V], bounds of loss, of lse, of logp, of d loss / d z)"""
    x = f64(logits)
    n, V = x.shape
    listed = listed_of(tokens, teacher, V)
    loss, lse, logp = torch.zeros(n, dtype=F64), torch.zeros(n, dtype=F64), torch.zeros(n, dtype=F64)
    d, b_loss, b_d = torch.zeros_like(x), torch.zeros(n, dtype=F64), torch.zeros_like(x)
    e = of_sum(V)
    for i in range(n):
        level = x[i].max()      # taken off first: next to float32's lowest value 64 bits have no digits for a row either
        level = level if torch.isfinite(level) else torch.zeros((), dtype=F64)
        z = ((x[i] - level) * scale).requires_grad_(True)
        one, shown = distill_row(z, listed[i], beta, rest)
        loss[i] = one.detach()
        if one.requires_grad and shown is not None:
            g, = torch.autograd.grad(one, z)
            d[i] = torch.where(torch.isneginf(z), torch.where(torch.isnan(g), 0.0, g), g).detach()
        relative = torch.logsumexp(z.detach(), 0)
        lse[i] = relative + level * scale
        # Each ln p is off by twice the sum's error: a loss by that times the sum of the sizes of its derivatives.
        mean = sum(p * abs(a) for p, q, a in shown) if shown else 0.0
        mass = sum(q for p, q, a in shown) if shown else 0.0
        b_loss[i] = 2 * e * (2 * mass + 2 * mean + 2) + 2 * U * loss[i].abs()
        if shown:
            p = torch.softmax(z.detach(), 0)
            off = 4 * e * p * (mass + 1 + mean + max([abs(a) for p_, q, a in shown if p_ > 0], default=0.0))
            # of the rest each one's share, of a float32 exponential: three terms of its exponent, three roundings each
            others = torch.ones(V, dtype=torch.bool)
            others[list(listed[i])] = False
            far = (z.detach() - z.detach()[others].max()).abs() if others.any() else torch.zeros(V, dtype=F64)
            far = torch.where(torch.isfinite(far), far, 0.0)
            b_d[i] = off + d[i].abs() * U * (16 + others * 9 * (far + math.log(V) + 1))
        if targets is not None:
            t = int(targets[i])
            logp[i] = z.detach()[t] - relative if 0 <= t < V else 0.0
            if math.isinf(lse[i]) and lse[i] < 0 and 0 <= t < V:
                logp[i] = -math.inf
    bad = torch.isnan(x).any(1) | torch.isposinf(x).any(1)
    loss[bad] = lse[bad] = math.nan
    if targets is not None:
        t = targets.long().cpu()
        logp[bad & (t >= 0) & (t < V)] = math.nan
    d[bad] = math.nan
    size = torch.where(torch.isfinite(lse), lse.abs(), 0.0)
    top = torch.where(torch.isfinite(x), (x * scale).abs(), 0.0).amax(1)
    b_lse = e + 4 * U * (size + top)
    b_logp = e + 4 * U * torch.where(torch.isfinite(logp), logp.abs(), 0.0)
    return loss, lse, logp, d, b_loss, b_lse, b_logp, b_d


def distillation_grad(logits, tokens, stats, d_loss, scale, targets=None, d_lse=None, d_logp=None, first=0, vocab=None):
    """(gradient, a bound) by the stats that are given"""
    x, s = f64(logits), f64(stats)
    n, V = x.shape
    zero = torch.zeros(n, dtype=F64)
    d = f64(d_loss) if d_loss is not None else zero
    l = f64(d_lse) if d_lse is not None else zero
    g = zero
    if d_logp is not None:
        t = targets.long().cpu()
        g = torch.where((t >= 0) & (t < (vocab or V)), f64(d_logp), 0.0)
    dead = torch.isneginf(s[:, 1])
    g, l = torch.where(dead, 0.0, g), torch.where(dead, 0.0, l)
    def share(m, log_s):
        none = torch.isneginf(log_s)
        q = (x - torch.where(none, 0.0, m)[:, None]) * scale - torch.where(none, 0.0, log_s)[:, None]
        q = torch.where(none[:, None], -math.inf, q)
        return q.exp(), torch.where(q > -745, q.abs() + (x * scale - (m * scale)[:, None]).abs() + log_s.abs()[:, None], 0.0)
    w, big_w = share(s[:, 2], s[:, 3])
    p, big_p = share(s[:, 0], s[:, 1])
    # (p of the unlisted is w times that of all of them, whose exponent has three terms)
    of_all = torch.where(torch.isneginf(s[:, 3]), 0.0, (s[:, 2] - s[:, 0]).abs() * scale + s[:, 3].abs() + s[:, 1].abs())[:, None]
    out = d[:, None] * s[:, 4:5] * w
    size = (out.abs() * (1 + big_w))
    for i in range(n):
        for k, t in enumerate(tokens[i].long().cpu().tolist()):
            if t >= 0 and 0 <= t - first < V:
                out[i, t - first] = d[i] * s[i, 5 + k]
                size[i, t - first] = out[i, t - first].abs()
    out = out + (l - g)[:, None] * p
    size = size + (l.abs() + g.abs())[:, None] * p * (1 + big_p + big_w + of_all)
    for i in range(n):
        if g[i] != 0 and 0 <= int(targets[i]) - first < V:
            out[i, int(targets[i]) - first] += g[i]
            size[i, int(targets[i]) - first] += g[i].abs()
    return out * scale, size * scale * U * 16 + 2.0 ** -126


# ---- adjusted logits ----
def counts(tokens, lengths, prompts, n, V, first):
    """(how often each column's token is behind the prompt, whether it is in the history at all)"""
    times, there = torch.zeros(n, V, dtype=F64), torch.zeros(n, V, dtype=torch.bool)
    if tokens is None:
        return times, there
    H = tokens.shape[-1]
    tokens = tokens.long().cpu().reshape(-1, H).expand(n, H) if tokens.dim() == 1 else tokens.long().cpu().reshape(n, H)
    for i in range(n):
        length = H if lengths is None else min(max(int(lengths.reshape(-1)[i]), 0), H)
        prompt = 0 if prompts is None else int(prompts.reshape(-1)[i])
        for k, t in enumerate(tokens[i, :length].tolist()):
            if 0 <= t - first < V:
                there[i, t - first] = True
                times[i, t - first] += k >= prompt
    return times, there


def of_rows(value, otherwise, n):
    if value is None:
        return torch.full((n, 1), otherwise, dtype=F64)
    if not isinstance(value, torch.Tensor):
        return torch.full((n, 1), float(torch.tensor(value, dtype=torch.float32)), dtype=F64)
    return f64(value).reshape(-1, 1).expand(n, 1)


def allowed_of(allowed, n, V, first):
    if allowed is None:
        return torch.ones(n, V, dtype=torch.bool)
    words = allowed.cpu().view(torch.int32).long().reshape(-1, allowed.shape[-1]).expand(n, allowed.shape[-1])
    j = torch.arange(first, first + V)
    return (words[:, j // 32] >> (j % 32)) % 2 != 0


def adjusted(logits, history=None, lengths=None, prompts=None, repetition=None, frequency=None, presence=None, bias_tokens=None, bias=None,
             allowed=None, scale=None, first=0):
    """(result, a bound: each term is rounded once, and there are five)"""
    shape = logits.shape
    x = f64(logits).reshape(-1, shape[-1])
    n, V = x.shape
    times, there = counts(history, lengths, prompts, n, V, first)
    r, f, p, s = (of_rows(v, o, n) for v, o in ((repetition, 1.0), (frequency, 0.0), (presence, 0.0), (scale, 1.0)))
    y = torch.where(there, torch.where(x > 0, x / r, x * r), x)
    y = torch.where(times > 0, y - f * times - p, y)
    size = torch.where(torch.isfinite(x), x.abs(), 0.0) * (r + 1 / r) + f.abs() * times + p.abs()
    if bias is not None and bias.numel():
        B = bias.shape[-1]
        at, value = bias_tokens.long().cpu().reshape(-1, B).expand(n, B), f64(bias).reshape(-1, B).expand(n, B)
        for i in range(n):
            for t, v in zip(at[i].tolist(), value[i].tolist()):
                if 0 <= t - first < V:
                    y[i, t - first] += v
                    size[i, t - first] += (B + 1) * abs(v)
    y, size = y * s, size * s.abs()
    y = torch.where(allowed_of(allowed, n, V, first), y, -math.inf)
    return y.reshape(shape), (8 * U * size).reshape(shape)


def adjusted_grad(logits, grad, history=None, lengths=None, repetition=None, allowed=None, scale=None, first=0):
    shape = logits.shape
    x, g = f64(logits).reshape(-1, shape[-1]), f64(grad).reshape(-1, shape[-1])
    n, V = x.shape
    _, there = counts(history, lengths, None, n, V, first)
    r, s = of_rows(repetition, 1.0, n), of_rows(scale, 1.0, n)
    d = g * s * torch.where(there, torch.where(x > 0, 1 / r, r), 1.0)
    d = torch.where(allowed_of(allowed, n, V, first), d, 0.0)
    return d.reshape(shape), (4 * U * d.abs()).reshape(shape)


def words_of(allowed):
    """[..., tokens] truth values as words of 32 bits."""
    n = allowed.shape[-1]
    bits = torch.zeros(*allowed.shape[:-1], (n + 31) // 32 * 32, dtype=torch.int64)
    bits[..., :n] = allowed.cpu()
    words = (bits.reshape(*allowed.shape[:-1], -1, 32) << torch.arange(32)).sum(-1)
    return torch.where(words >= 2 ** 31, words - 2 ** 32, words).to(torch.int32)
