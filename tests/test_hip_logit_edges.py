"""Calls of the operators on a head's logits at the edges of what they accept, against plain forms in 64 bits (logit_cases.py) or against
the same call made another way."""
import math

import pytest

torch = pytest.importorskip("torch")   # before the library: one HIP runtime in the process

import logit_cases as C   # noqa: E402
from galvatron_dp import model_ends, operators as ops   # noqa: E402
from test_hip_logits import check_distillation, gen, history_of, lists, normal   # noqa: E402

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
INF = math.inf


def test_results_in_the_place_of_what_autograd_does_not_follow():
    """A detached view of a tensor that wants a gradient may be written, and the graph that holds its values says so; a student's gradients
    are the same where its block wants one."""
    g = gen(45)
    leaf = normal(g, 3, 60).requires_grad_(True)
    y = leaf * 5
    kept = (y * y).sum()
    want = ops.adjust_logits(y.detach(), scale=2.0)
    assert torch.equal(ops.adjust_logits(y.detach(), scale=2.0, into=y.detach()), want) and torch.equal(y, want)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        kept.backward()
    with torch.no_grad():
        ops.adjust_logits(leaf, scale=2.0, into=leaf)
    assert torch.equal(leaf * 5, want)
    ends = model_ends.ModelEnds(96, 1000, dtype=BF16, seed=7)
    tokens, targets = torch.randint(0, 1000, (6,), generator=g).cuda(), torch.randint(0, 1000, (6,), generator=g).cuda()
    block = normal(g, 6, 96, dtype=BF16)
    listed, q = lists(g, 6, 1000, 8)
    for weight in (1.0, 0.5):
        teacher = model_ends.Teacher(listed, q, weight=weight)
        a = ends.loss_and_grads(tokens, targets, block, teacher=teacher)
        b = ends.loss_and_grads(tokens, targets, block.clone().requires_grad_(True), teacher=teacher)
        assert all(torch.equal(s, t) for s, t in zip(a, b) if s is not None)


@pytest.mark.parametrize("score", [INF, math.nan], ids=["inf", "nan"])
@pytest.mark.parametrize("beta,rest", [(0.0, True), (0.5, True), (1.0, True), (0.0, False), (0.5, False)])
def test_a_teacher_that_is_no_number(beta, rest, score):
    """At a place that is used: the row's loss and its gradient are NaN, what does not go by the teacher is as it was."""
    g = gen(40)
    for K in (5, 80):
        x = normal(g, 7, 300)
        tokens, teacher = lists(g, 7, 300, K)
        want = ops.distillation(x, tokens, teacher, beta=beta, rest=rest, targets=tokens[:, 0], stats=True)
        teacher[0, 2] = teacher[1, 0] = score
        tokens[2, 3] = tokens[2, 1]                             # of a token in two places
        teacher[2, 3] = score
        x[3, tokens[3, 2]] = -INF                               # of a token that the row rules out
        teacher[3, 2] = score
        listed = torch.zeros(300, dtype=torch.bool, device="cuda").scatter_(0, tokens[4], True)
        x[4, ~listed] = x[4, tokens[4, 2]] = -INF               # ... in a row that has no rest
        teacher[4, 2] = score
        tokens[5, 1], teacher[5, 1] = -1, score                 # at a place that is not used
        r = ops.distillation(x, tokens, teacher, beta=beta, rest=rest, targets=tokens[:, 0], stats=True)
        assert torch.isnan(r.loss).tolist() == [True] * 5 + [False] * 2
        assert torch.equal(r.loss[6], want.loss[6])
        assert torch.isfinite(r.lse).all() and torch.isfinite(r.logp).all()
        assert torch.equal(r.lse[:3], want.lse[:3]) and torch.equal(r.logp[:3], want.logp[:3])
        ones = torch.ones(7, device="cuda")
        grad = ops.distillation_grad(x, tokens, r.stats, ones)
        assert torch.isnan(grad[:4].where(torch.isfinite(x[:4]), math.nan)).all() and not torch.isnan(grad[5:]).any()
        assert torch.isnan(grad[4].gather(0, tokens[4])[torch.isfinite(x[4].gather(0, tokens[4]))]).all()
        parts = [ops.distillation_parts(x[:, a:a + 100], tokens, teacher, first=a) for a in (0, 100, 200)]
        assert torch.isnan(ops.join_distillation(parts, tokens, teacher, 300, beta=beta, rest=rest).loss).tolist() == [True] * 5 + [False] * 2


def listed_by_logsumexp(tokens, teacher, vocab):
    """Of each row {token: log of the sum of q} over its used places, whatever float64 has of q itself."""
    rows = []
    for ts, ls in zip(tokens.long().cpu().tolist(), C.f64(teacher).tolist()):
        got = {}
        for t, v in zip(ts, ls):
            if 0 <= t < vocab and v != -INF:
                got.setdefault(t, []).append(v)
        rows.append({t: max(v) + math.log(sum(math.exp(a - max(v)) for a in v)) for t, v in got.items()})
    return rows


@pytest.mark.parametrize("beta", [0.0, 0.5, 1.0])
def test_unlikely_tokens_in_several_places(beta, monkeypatch):
    """Probabilities that float64 does not hold, or holds with few digits: their sum's logarithm is a number all the same."""
    monkeypatch.setattr(C, "listed_of", listed_by_logsumexp)
    g = gen(41)
    for K in (6, 90):
        x = normal(g, 5, 400, size=2.0)
        tokens, teacher = lists(g, 5, 400, K)
        tokens[0, 1] = tokens[0, 2] = tokens[0, 0]
        teacher[0, :3] = torch.tensor([-800.0, -801.0, -900.0])
        tokens[1, 1] = tokens[1, 0]
        teacher[1, :2] = -1e9                                   # as a grammar's mask leaves them
        tokens[2, 4] = tokens[2, 3]
        teacher[2, 3], teacher[2, 4] = -744.5, -744.0           # a few units of the least number
        tokens[3, 1] = tokens[3, 0]
        teacher[3, 1] = -3e38                                   # next to a likely one
        tokens[4, 2] = tokens[4, 1] = tokens[4, 0]
        teacher[4, 0], teacher[4, 1], teacher[4, 2] = -800.0, -INF, -800.0
        r = check_distillation(x, tokens, teacher, 1.0, beta, True, tokens[:, 0])
        assert torch.isfinite(r.loss).all() and torch.isfinite(r.stats).all()


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("case", [(6, 1000, 1040, 20, 2), (2, 128000, 128256, 100, 1), (1500, 250, 260, 5, 4), (5, 90, 120, 9, 4)], ids=str)
def test_shards_with_columns_behind_the_vocabulary(case, dtype):
    """Tokens from ``vocab`` on are none, for the parts, their join and the gradient alike; their columns are unlisted ones."""
    n, V, padded, K, shards = case
    g = gen(42)
    x = normal(g, n, padded, dtype=dtype, size=2.0)
    tokens, teacher = lists(g, n, padded, K)
    for i, t in ((0, V), (1, padded - 1)):      # (each once)
        tokens[i] = torch.where(tokens[i] == t, tokens[i, 0], tokens[i])
        tokens[i, 0] = t
    targets = torch.randint(-1, padded, (n,), generator=g).cuda()
    targets[0], targets[1] = tokens[0, 0], V - 1
    used, wanted = torch.where(tokens < V, tokens, -1), torch.where(targets < V, targets, -100)
    edges = [padded * i // shards for i in range(shards + 1)]
    of = [x[:, a:b] for a, b in zip(edges, edges[1:])]
    parts = [ops.distillation_parts(s, tokens, teacher, first=a, vocab=V, targets=targets) for s, a in zip(of, edges)]
    r = ops.join_distillation(parts, tokens, teacher, V, beta=0.25, targets=targets, stats=True)
    few = slice(0, 6)
    check_distillation(x[few], used[few], teacher[few], 1.0, 0.25, True, wanted[few], ops.Distillation(*(t[few] for t in r)))
    d_loss, d_logp = torch.rand(n, generator=g).cuda(), torch.rand(n, generator=g).cuda()
    whole = ops.distillation_grad(x, used, r.stats, d_loss, targets=wanted, grad_logp=d_logp)
    pieces = [ops.distillation_grad(s, tokens, r.stats, d_loss, targets=targets, grad_logp=d_logp, first=a, vocab=V) for s, a in zip(of, edges)]
    assert torch.equal(whole, torch.cat(pieces, 1))
    for bad in (-1, 0, 2 ** 31, 2 ** 32):
        with pytest.raises(ValueError, match="vocab"):
            ops.distillation_parts(x, tokens, teacher, first=0, vocab=bad)


@pytest.mark.parametrize("dtype", [None, F32], ids=["same", "float32"])
def test_a_step_that_is_differentiated_or_in_float32(dtype):
    """``ModelEnds.forward`` with adjusted logits: towards the block as without them, and in the type that is asked for."""
    ends = model_ends.ModelEnds(96, 1000, dtype=BF16, seed=7)
    g = gen(44)
    tokens, targets = torch.randint(0, 1000, (6,), generator=g).cuda(), torch.randint(0, 1000, (6,), generator=g).cuda()
    block = normal(g, 6, 96, dtype=BF16)
    adjust = dict(history=history_of(g, 6, 40, 1000), repetition=1.2, frequency=0.5, scale=0.8, **({"dtype": dtype} if dtype else {}))
    plain = block.clone().requires_grad_(True)
    want = ops.token_logprobs(ops.adjust_logits(ends.logits(ends.embed(tokens), plain)[1], **adjust), targets)
    want.logp.sum().backward()
    leaf = block.clone().requires_grad_(True)
    r = ends.forward(tokens, targets, leaf, adjust=adjust)
    r.logp.sum().backward()
    assert torch.equal(r.logp, want.logp) and torch.equal(leaf.grad, plain.grad) and bool((leaf.grad != 0).any())
    with torch.no_grad():
        assert torch.equal(ends.forward(tokens, targets, leaf, adjust=adjust).logp, want.logp)
        listed, q = lists(g, 6, 1000, 8)
        r = ends.forward(tokens, targets, block, teacher=model_ends.Teacher(listed, q), adjust=adjust)
        same = ops.distillation(ops.adjust_logits(ends.logits(ends.embed(tokens), block)[1], **adjust), listed, q, targets=targets)
        assert torch.equal(r.loss, same.loss) and torch.equal(r.logp, same.logp)


def test_missing_tensors_are_named():
    """What a call that did not ask for them leaves as None."""
    g = gen(43)
    x = normal(g, 3, 50)
    tokens, teacher = lists(g, 3, 50, 4)
    r, one = ops.distillation(x, tokens, teacher), torch.ones(3, device="cuda")
    assert r.stats is None
    parts = ops.distillation_parts(x, tokens, teacher, first=0)
    for what, call in (("stats", lambda: ops.distillation_grad(x, tokens, r.stats, one)), ("tokens", lambda: ops.distillation(x, None, teacher)),
                       ("teacher", lambda: ops.distillation(x, tokens, None)), ("tokens", lambda: ops.distillation_parts(x, None, teacher, first=0)),
                       ("teacher", lambda: ops.distillation_parts(x, tokens, None, first=0)), ("tokens", lambda: ops.join_distillation([parts], None, teacher, 50)),
                       ("teacher", lambda: ops.join_distillation([parts], tokens, None, 50))):
        with pytest.raises(ValueError, match=what):
            call()


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("columns", [1, 7, 2049, 50257], ids=str)
def test_gradients_of_adjusted_logits_in_place(columns, dtype):
    """Without a scale what does not change is neither read nor written: the same bits as in a new tensor, rows at any alignment."""
    g = gen(46)
    n = 5
    x = normal(g, n, columns, dtype=dtype)
    history = history_of(g, n, 70, columns)
    ok = torch.rand(n, columns, generator=g) < 0.5
    ok[1], ok[2], ok[3, columns // 3:] = True, False, True
    mask, rep = C.words_of(ok).cuda(), (0.5 + torch.rand(n, generator=g)).cuda()
    for given in (dict(history=history, repetition=1.3), dict(history=history, repetition=rep, allowed=mask), dict(allowed=mask), dict(history=history[:, :0], allowed=mask),
                  dict(history=history, repetition=rep, lengths=torch.tensor([0, 1, 70, 35, 0]).cuda(), allowed=mask[1]), dict()):
        grad = normal(g, n, columns + 9, dtype=dtype)
        for at in (0, 1, 3):
            want = ops.adjust_logits_grad(x, grad[:, at:at + columns], **given)
            ref, bound = C.adjusted_grad(x, grad[:, at:at + columns], **given)
            C.close(want, ref, bound + C.rounded(ref, dtype), "gradient")
            place = grad.clone()
            got = ops.adjust_logits_grad(x, place[:, at:at + columns], into=place[:, at:at + columns], **given)
            assert torch.equal(got, want) and torch.equal(place[:, :at], grad[:, :at]) and torch.equal(place[:, at + columns:], grad[:, at + columns:])


def test_large_adjusted_logits_in_place():
    """More than 256 MB in the place of what is read, in both directions: the same bits as in a new tensor."""
    g = gen(47)
    n, V = 1100, 128250
    x = torch.randn(n, V, device="cuda").to(BF16)
    given = dict(history=torch.randint(0, V, (n, 40), generator=g).cuda(), repetition=1.2, allowed=C.words_of(torch.rand(V, generator=g) < 0.5).cuda())
    more = dict(frequency=0.5, bias_tokens=torch.randint(0, V, (n, 9), generator=g).cuda(), bias=normal(g, n, 9))
    for each in (dict(given, **more), dict(allowed=given["allowed"])):
        want, place = ops.adjust_logits(x, **each), x.clone()
        assert torch.equal(ops.adjust_logits(place, into=place, **each), want)
    for each in (given, dict(allowed=given["allowed"])):
        want, place = ops.adjust_logits_grad(x, x, **each), x.clone()
        assert torch.equal(ops.adjust_logits_grad(x, place, into=place, **each), want)


@pytest.mark.parametrize("listed", [20, 70])
@pytest.mark.parametrize("case", [(600, 262400, BF16), (300, 262400, F32), (4100, 16500, F16)], ids=["bfloat16", "float32", "many rows"])
def test_distillation_gradients_that_are_written_past_the_caches(case, listed):
    """More than 128 MB: the same bits as rows by themselves have, in a new tensor and in the logits' place, with targets that are listed and
    targets that are not."""
    n, V, dtype = case
    g = gen(48)
    x = torch.randn(n, V, device="cuda").to(dtype)
    assert x.numel() * x.element_size() >= 128 << 20
    tokens, teacher = lists(g, 9, V, listed)
    tokens, teacher = tokens.repeat(n // 9 + 1, 1)[:n].contiguous(), teacher.repeat(n // 9 + 1, 1)[:n].contiguous()
    targets = torch.randint(0, V, (n,), generator=g).cuda()
    targets[::3] = tokens[::3, 1]
    r = ops.distillation(x, tokens, teacher, targets=targets, stats=True)
    d, d_logp = torch.rand(n, generator=g).cuda(), torch.rand(n, generator=g).cuda()
    whole = ops.distillation_grad(x, tokens, r.stats, d, targets=targets, grad_logp=d_logp)
    some = torch.cat([torch.arange(8), torch.arange(n // 2, n // 2 + 4), torch.arange(n - 4, n)]).cuda()
    part = ops.distillation_grad(x[some], tokens[some], r.stats[some], d[some], targets=targets[some], grad_logp=d_logp[some])
    assert torch.equal(whole[some], part)
    one = slice(0, 2)
    want, bound = C.distillation_grad(x[one], tokens[one], r.stats[one], d[one], 1.0, targets[one], None, d_logp[one])
    C.close(part[one], want, bound + C.rounded(want, dtype), "gradient by stats")
    # the listed places and the targets, of all rows
    at = torch.cat([tokens, targets[:, None]], 1)
    for a in range(0, n, 97):
        rows = slice(a, a + 97)
        same = ops.distillation_grad(x[rows], tokens[rows], r.stats[rows], d[rows], targets=targets[rows], grad_logp=d_logp[rows])
        assert torch.equal(whole[rows].gather(1, at[rows]), same.gather(1, at[rows]))
    place = x.clone()
    assert torch.equal(ops.distillation_grad(place, tokens, r.stats, d, targets=targets, grad_logp=d_logp, into=place), whole)
