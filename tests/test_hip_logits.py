"""The operators on a head's logits, distillation and adjusted logits, against plain forms in 64 bits (logit_cases.py), at the sizes, lists,
histories and masks where they can go wrong.  Bounds follow from the arithmetic: how many float32 roundings a result is behind, and one
rounding to its type."""
import math
import threading

import pytest

torch = pytest.importorskip("torch")   # before the library: one HIP runtime in the process

import logit_cases as C   # noqa: E402
from galvatron_dp import operators as ops   # noqa: E402

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = [F32, F16, BF16]
INF = math.inf
ids = lambda v: str(v).replace("torch.", "") if isinstance(v, torch.dtype) else None   # noqa: E731


def gen(seed):
    return torch.Generator().manual_seed(seed)


def normal(g, *shape, dtype=F32, size=1.0):
    return (torch.randn(*shape, generator=g) * size).to(dtype).cuda()


def lists(g, n, V, K, mass=None, index=torch.int64, spread=2.0):
    """Different tokens in each row, and log probabilities that leave some for the rest."""
    tokens = torch.stack([torch.randperm(V, generator=g)[:K] for _ in range(n)])
    left = torch.rand(n, 1, generator=g) * 0.6 + 0.3 if mass is None else torch.full((n, 1), mass)
    teacher = torch.log_softmax(spread * torch.randn(n, K, generator=g), 1) + left.log()
    return tokens.to(index).cuda(), teacher.cuda()


def check_distillation(x, tokens, teacher, scale, beta, rest, targets=None, got=None):
    """A call's results, its stats, and the gradients of all of them by both routes."""
    ref = C.distillation(x, tokens, teacher, scale, beta, rest, targets)
    loss, lse, logp, d, b_loss, b_lse, b_logp, b_d = ref
    r = got or ops.distillation(x, tokens, teacher, scale=scale, beta=beta, rest=rest, targets=targets, stats=True)
    C.close(r.loss, loss, b_loss, "loss")
    C.close(r.lse, lse, b_lse, "lse")
    if targets is not None:
        C.close(r.logp, logp, b_logp, "logp")
    else:
        assert r.logp is None
    n, V = x.shape
    g = gen(99)
    d_loss, d_lse = (1 + torch.rand(n, generator=g)).cuda(), torch.randn(n, generator=g).cuda()
    d_logp = torch.randn(n, generator=g).cuda() if targets is not None else None
    out = ops.distillation_grad(x, tokens, r.stats, d_loss, scale=scale, targets=targets, grad_lse=d_lse, grad_logp=d_logp)
    want, bound = C.distillation_grad(x, tokens, r.stats, d_loss, scale, targets, d_lse, d_logp)
    C.close(out, want, bound + C.rounded(want, x.dtype), "gradient by stats")
    one = ops.distillation_grad(x, tokens, r.stats, torch.ones(n, device="cuda"), scale=scale, targets=targets)
    C.close(one, d * scale, b_d * scale + C.rounded(d * scale, x.dtype), "gradient of the loss")
    return r


SIZES = [  # rows, vocabulary, listed
    (1, 1, 1), (1, 2, 1), (3, 5, 2), (4, 5, 5), (7, 33, 4), (5, 64, 64), (64, 1000, 20), (5, 4097, 63), (3, 8190, 65), (3, 50257, 128),
    (2, 128256, 256), (1, 300003, 20), (1100, 517, 20), (1030, 5003, 7),
    (1024, 262400, 20), (1300, 26000, 100)]


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("case", SIZES, ids=str)
def test_distillation_sizes(case, dtype):
    n, V, K = case
    g = gen(n + V)
    x = normal(g, n, V, dtype=dtype, size=2.0)
    tokens, teacher = lists(g, n, V, K, index=torch.int32 if V % 2 else torch.int64)
    targets = torch.randint(-1, V + 1, (n,), generator=g).cuda()
    if n > 40:      # (rows of plain Python arithmetic: some of them)
        r = ops.distillation(x, tokens, teacher, targets=targets, stats=True)
        some = torch.cat([torch.arange(4), torch.arange(n - 4, n)]).cuda()
        part = ops.Distillation(*(t[some] for t in r))
        check_distillation(x[some], tokens[some], teacher[some], 1.0, 0.0, True, targets[some], part)
    else:
        check_distillation(x, tokens, teacher, 1.0, 0.0, True, targets)


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("case", [(2100, 517, 20), (2050, 1000, 100), (3001, 9, 9), (2048, 4090, 256), (2049, 8185, 3)], ids=str)
def test_distillation_of_many_short_rows(case, dtype):
    """A wave for each row: the same bits as rows by themselves have in the gradient, and results within the bounds; lists with unused and
    repeated places among them."""
    n, V, K = case
    g = gen(n + K)
    x = normal(g, n, V, dtype=dtype, size=2.0)
    tokens, teacher = lists(g, 64, V, K)
    tokens, teacher = tokens.repeat(n // 64 + 1, 1)[:n].contiguous(), teacher.repeat(n // 64 + 1, 1)[:n].contiguous()
    if K > 2:
        tokens[1, 1], tokens[2, 0], teacher[3, 2] = tokens[1, 0], -1, -INF
    targets = torch.randint(-1, V + 1, (n,), generator=g).cuda()
    targets[:5] = tokens[:5, 0]
    r = ops.distillation(x, tokens, teacher, beta=0.25, targets=targets, stats=True)
    some = torch.cat([torch.arange(6), torch.arange(n - 2, n)]).cuda()
    check_distillation(x[some], tokens[some], teacher[some], 1.0, 0.25, True, targets[some], ops.Distillation(*(t[some] for t in r)))
    d, d_logp = torch.rand(n, generator=g).cuda(), torch.rand(n, generator=g).cuda()
    whole = ops.distillation_grad(x, tokens, r.stats, d, targets=targets, grad_logp=d_logp)
    part = ops.distillation_grad(x[some], tokens[some], r.stats[some], d[some], targets=targets[some], grad_logp=d_logp[some])
    assert torch.equal(whole[some], part)
    place = x.clone()
    assert torch.equal(ops.distillation_grad(place, tokens, r.stats, d, targets=targets, grad_logp=d_logp, into=place), whole)


def test_logits_that_no_cache_holds():
    """Few rows, but more than 256 MB; results as of rows by themselves."""
    g = gen(15)
    for n, V, dtype in ((600, 262400, BF16), (300, 262400, F32)):
        x = torch.randn(n, V, device="cuda", dtype=dtype)
        for K in (20, 70):
            tokens, teacher = lists(g, 8, V, K)
            tokens, teacher = tokens.repeat(n // 8, 1)[:n].contiguous(), teacher.repeat(n // 8, 1)[:n].contiguous()
            tokens, teacher = torch.cat([tokens, tokens])[:n].contiguous(), torch.cat([teacher, teacher])[:n].contiguous()
            r = ops.distillation(x, tokens, teacher, stats=True)
            some = torch.tensor([0, n // 2, n - 1]).cuda()
            check_distillation(x[some], tokens[some], teacher[some], 1.0, 0.0, True, None, ops.Distillation(*(t if t is None else t[some] for t in r)))


@pytest.mark.parametrize("scale", [1.0, 0.5, 3.25])
@pytest.mark.parametrize("rest", [True, False], ids=["rest", "renormed"])
@pytest.mark.parametrize("beta", [0.0, 0.125, 0.5, 1.0])
def test_distillation_forms(beta, rest, scale):
    if beta == 1.0 and not rest:
        with pytest.raises(ValueError, match="beta 1"):
            ops.distillation(torch.zeros(2, 4, device="cuda"), torch.zeros(2, 1, dtype=torch.int64, device="cuda"), torch.zeros(2, 1, device="cuda"),
                             beta=beta, rest=rest)
        return
    g = gen(5)
    for K in (1, 12, 100):
        x = normal(g, 6, 777, size=2.0)
        tokens, teacher = lists(g, 6, 777, K)
        check_distillation(x, tokens, teacher, scale, beta, rest, tokens[:, 0] if K == 12 else torch.arange(6).cuda() * 50)


@pytest.mark.parametrize("beta", [0.0, 0.25, 1.0])
def test_places_that_are_not_used_and_tokens_in_several(beta):
    g = gen(6)
    for rest in (True, False) if beta < 1 else (True,):
        for K in (9, 70):
            x = normal(g, 8, 400, size=2.0)
            tokens, teacher = lists(g, 8, 400, K)
            tokens[1, 2], tokens[1, 3], tokens[1, 4] = -1, 400, -100        # no tokens
            teacher[2, 1] = teacher[2, 3] = -INF                            # tokens that are of the rest
            tokens[3, 1] = tokens[3, 0]                                     # twice
            tokens[4, 5] = tokens[4, 6] = tokens[4, 2]                      # three times
            tokens[5, 1], teacher[5, 1] = tokens[5, 0], -INF                # a listed one again, at a place that is not used
            teacher[6, 1] = teacher[6, 2] = -INF
            tokens[6, 2] = tokens[6, 1]                                     # one of the rest twice
            teacher[7] = -INF                                               # no list
            targets = torch.stack([tokens[i, (1, 0, 1, 1, 5, 1, 2, 0)[i]] for i in range(8)])
            r = check_distillation(x, tokens, teacher, 1.0, beta, rest, targets)
            assert r.loss[7].item() == 0.0 and not torch.isnan(r.stats).any()


def test_a_list_of_nearly_everything():
    """A rest that float32 cannot tell is none (2^-22 towards the teacher's peaks); next to that the rest counts."""
    g = gen(7)
    x = normal(g, 5, 300, size=2.0)
    tokens, _ = lists(g, 5, 300, 4)
    q = torch.tensor([[0.5, 0.25, 0.125, 0.125], [0.5, 0.25, 0.125, 0.125 - 2.0 ** -21], [0.5, 0.25, 0.125, 0.125 - 2.0 ** -24],
                      [0.7, 0.25, 0.125, 0.125], [1.0, 0.0, 0.0, 0.0]])
    for beta in (0.0, 0.5, 1.0):
        r = check_distillation(x, tokens, q.log().cuda(), 1.0, beta, True)
        assert torch.isfinite(r.loss).all()


@pytest.mark.parametrize("dtype", [F32, BF16], ids=ids)
@pytest.mark.parametrize("beta", [0.0, 0.5, 1.0])
def test_rows_with_little_left_and_far_from_zero(beta, dtype):
    """The rest next to nothing in the student (its share in the gradient is none the less), masks of -inf, -1e9 and the lowest value, levels."""
    g = gen(8)
    low = torch.finfo(dtype).min
    for K in (3, 80):
        x = normal(g, 9, 500, size=2.0)
        tokens, teacher = lists(g, 9, 500, K)
        x[0].scatter_(0, tokens[0], 150.0)                       # p of the rest is e^-150
        listed = torch.zeros(500, dtype=torch.bool, device="cuda").scatter_(0, tokens[1], True)
        x[1, ~listed] = -INF                                     # nothing but the list
        x[2, listed.logical_not()] = -1e9
        x[3, torch.arange(0, 500, 2)] = -INF
        x[3, tokens[3]] = 1.0
        x[4] += 9000.0
        x[5] -= 9000.0
        x[6] = low
        x[7] = -INF
        x[8, tokens[8, 0]] = 90.0                                # one token has nearly all
        x = x.to(dtype)
        r = check_distillation(x, tokens, teacher, 1.0, beta, True, tokens[:, 0])
        assert r.loss[7].item() == 0.0 and r.lse[7].item() == -INF and r.logp[7].item() == -INF
        assert not torch.isnan(r.stats).any()
        grad = ops.distillation_grad(x, tokens, r.stats, torch.ones(9, device="cuda"), targets=tokens[:, 0], grad_logp=torch.ones(9, device="cuda"))
        assert not torch.isnan(grad).any() and (grad[7] == 0).all()


def test_a_listed_token_that_is_ruled_out():
    g = gen(9)
    x = normal(g, 2, 100)
    tokens, teacher = lists(g, 2, 100, 5)
    x[0, tokens[0, 2]] = -INF
    r = check_distillation(x, tokens, teacher, 1.0, 0.0, True)
    assert r.loss[0].item() == INF and torch.isfinite(r.loss[1])
    for beta in (0.5, 1.0):
        assert torch.isfinite(check_distillation(x, tokens, teacher, 1.0, beta, True).loss).all()


@pytest.mark.parametrize("beta", [0.0, 0.5, 1.0])
def test_no_numbers(beta):
    g = gen(10)
    x = normal(g, 6, 100)
    tokens, teacher = lists(g, 6, 100, 5)
    others = [next(j for j in range(100) if j not in set(tokens[i].tolist())) for i in range(6)]
    x[0, others[0]] = x[1, tokens[1, 3]] = math.nan
    x[2, others[2]] = x[3, tokens[3, 1]] = INF
    teacher[4, 2] = math.nan
    targets = tokens[:, 0].clone()
    r = ops.distillation(x, tokens, teacher, beta=beta, targets=targets, stats=True)
    assert torch.isnan(r.loss).tolist() == [True] * 5 + [False]
    assert torch.isnan(r.lse).tolist() == [True] * 4 + [False] * 2 and torch.isnan(r.logp).tolist() == [True] * 4 + [False] * 2
    grad = ops.distillation_grad(x, tokens, r.stats, torch.ones(6, device="cuda"))
    assert torch.isnan(grad[:4]).all() and not torch.isnan(grad[5]).any()
    check_distillation(x[5:], tokens[5:], teacher[5:], 1.0, beta, True, targets[5:])


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_distillation_strides_and_shapes(dtype):
    """Rows within wider ones that begin on no 16 bytes, columns at a stride, leading dimensions, lists and targets with strides."""
    g = gen(11)
    wide = normal(g, 6, 1203, dtype=dtype, size=2.0)
    tokens, teacher = lists(g, 6, 1100, 10)
    targets = tokens.flip(1)[:, 3]
    for x in (wide[:, 1:1101], wide[:, 3:1103], normal(g, 1100, 6, dtype=dtype).t(), wide[::2, 5:1105].expand(3, 1100)):
        n = x.shape[0]
        check_distillation(x, tokens[:n], teacher[:n], 1.0, 0.0, True, targets[:n])
    x = wide[:, 1:1101].reshape(2, 3, 1100)
    r = ops.distillation(x, tokens.reshape(2, 3, 10), teacher.reshape(2, 3, 10), targets=targets.reshape(2, 3), stats=True)
    assert r.loss.shape == r.logp.shape == (2, 3) and r.stats.shape == (2, 3, 15)
    check_distillation(wide[:, 1:1101], tokens, teacher, 1.0, 0.0, True, targets, ops.Distillation(*(t.flatten(0, 1) for t in r)))
    one = ops.distillation(x[0, 0], tokens[0], teacher[0])
    assert one.loss.shape == () and one.loss.item() == r.loss[0, 0].item() and one.stats is None and one.logp is None
    none = ops.distillation(x[:0], tokens[:0].reshape(0, 3, 10), teacher[:0].reshape(0, 3, 10), stats=True)
    assert none.loss.shape == (0, 3) and none.stats.shape == (0, 3, 15)
    assert ops.distillation_grad(x[:0], tokens[:0].reshape(0, 3, 10), none.stats, none.loss).shape == (0, 3, 1100)


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("case", [(3, 1000, 20, 4), (2, 50257, 100, 3), (1500, 260, 5, 2), (5, 9, 9, 9)], ids=str)
def test_distillation_in_shards(case, dtype):
    n, V, K, shards = case
    g = gen(12)
    x = normal(g, n, V, dtype=dtype, size=2.0)
    tokens, teacher = lists(g, n, V, K)
    tokens[0, 0], teacher[0, K // 2] = -1, -INF
    targets = torch.randint(-1, V, (n,), generator=g).cuda()
    edges = [V * i // shards for i in range(shards + 1)]
    of = [x[:, a:b] for a, b in zip(edges, edges[1:])]
    parts = [ops.distillation_parts(s, tokens, teacher, first=a, targets=targets) for s, a in zip(of, edges)]
    r = ops.join_distillation(parts, tokens, teacher, V, beta=0.25, targets=targets, stats=True)
    gathered = ops.DistillationParts(*(torch.stack(t) for t in zip(*parts)))
    for a, b in zip(r, ops.join_distillation(gathered, tokens, teacher, V, beta=0.25, targets=targets, stats=True)):
        assert torch.equal(a, b)
    few = slice(0, 8)
    check_distillation(x[few], tokens[few], teacher[few], 1.0, 0.25, True, targets[few], ops.Distillation(*(t[few] for t in r)))
    d_loss, d_logp = torch.rand(n, generator=g).cuda(), torch.rand(n, generator=g).cuda()
    whole = ops.distillation_grad(x, tokens, r.stats, d_loss, targets=targets, grad_logp=d_logp)
    pieces = [ops.distillation_grad(s, tokens, r.stats, d_loss, targets=targets, grad_logp=d_logp, first=a, vocab=V) for s, a in zip(of, edges)]
    assert torch.equal(whole, torch.cat(pieces, 1))


@pytest.mark.parametrize("beta", [0.0, 0.5, 1.0])
def test_distillation_through_autograd_and_differences(beta):
    """Against the differentiated plain form, and a few logits against differences of it."""
    g = gen(13)
    x = normal(g, 5, 321, size=2.0).requires_grad_(True)
    tokens, teacher = lists(g, 5, 321, 7)
    targets = torch.tensor([0, -100, 320, 5, 400]).cuda()
    targets[3] = tokens[3, 2]
    weight = torch.rand(5, generator=g).cuda()
    r = ops.distillation(x, tokens, teacher, scale=1.5, beta=beta, targets=targets)
    ((r.loss * weight).sum() - 0.5 * r.logp.sum() + 0.1 * (r.lse ** 2).sum()).backward()
    z = x.detach().cpu().double().requires_grad_(True)
    listed = C.listed_of(tokens, teacher, 321)
    w = weight.cpu().double()

    def whole(z, i):
        t = int(targets[i])
        lse = torch.logsumexp(z[i] * 1.5, 0)
        total = w[i] * C.distill_row(z[i] * 1.5, listed[i], beta, True)[0] + 0.1 * lse ** 2
        return total - 0.5 * (z[i, t] * 1.5 - lse) if 0 <= t < 321 else total

    sum(whole(z, i) for i in range(5)).backward()
    _, lse, _, d, _, b_lse, _, b_d = C.distillation(x, tokens, teacher, 1.5, beta, True)
    # of lse^2 and logp: p's exponent has three roundings of some 30 each; lse itself is rounded once
    p = torch.softmax(x.detach().cpu().double() * 1.5, 1)
    bound = 1.5 * (b_d * w[:, None] + (p + 1e-3) * (0.2 * lse.abs()[:, None] + 0.5) * C.U * 300 + 0.2 * p * b_lse[:, None])
    C.close(x.grad, z.grad, bound + C.rounded(z.grad, F32), "autograd")
    h = 1e-5
    for i in range(5):
        for j in (0, 100, int(tokens[i, 0]), int(tokens[i, 6])):
            up, down = z.detach().clone(), z.detach().clone()
            up[i, j] += h
            down[i, j] -= h
            slope = (whole(up, i) - whole(down, i)).item() / (2 * h)
            assert abs(slope - x.grad[i, j].item()) < 1e-6, (i, j)     # (h^2 times third derivatives below 10^3; 10^-15 * 10^2 / h)


def test_distillation_gradients_in_place_and_versions():
    g = gen(14)
    for K in (5, 200):
        x = normal(g, 3, 5000, dtype=BF16, size=2.0)
        tokens, teacher = lists(g, 3, 5000, K)
        targets = torch.tensor([7, 4999, 0]).cuda()
        targets[1] = tokens[1, 0]
        r = ops.distillation(x, tokens, teacher, targets=targets, stats=True)
        d = torch.rand(3, generator=g).cuda()
        want = ops.distillation_grad(x, tokens, r.stats, d, targets=targets, grad_logp=-d)
        buffer = torch.full((3, 5003), 7.0, dtype=BF16, device="cuda")
        got = ops.distillation_grad(x, tokens, r.stats, d, targets=targets, grad_logp=-d, into=buffer[:, 2:5002])
        assert torch.equal(got, want) and (buffer[:, :2] == 7).all() and (buffer[:, 5002:] == 7).all()
        version = x._version
        assert ops.distillation_grad(x, tokens, r.stats, d, targets=targets, grad_logp=-d, into=x) is x
        assert torch.equal(x, want) and x._version > version
    with pytest.raises(ValueError, match="neighbouring"):
        ops.distillation_grad(x, tokens, r.stats, d, into=torch.empty(5000, 3, dtype=BF16, device="cuda").t())
    leaf = normal(g, 3, 50).requires_grad_(True)
    tokens, teacher = lists(g, 3, 50, 5)
    y = leaf * 1
    r = ops.distillation(y, tokens, teacher, stats=True)
    assert r.loss.requires_grad and r.lse.requires_grad and not r.stats.requires_grad
    y.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        r.loss.sum().backward()
    with pytest.raises(ValueError, match="no gradient"):
        ops.distillation(leaf, tokens, teacher.requires_grad_(True))


def test_distillation_refusals():
    x, t, q = torch.zeros(2, 10, device="cuda"), torch.zeros(2, 3, dtype=torch.int64, device="cuda"), torch.zeros(2, 3, device="cuda")
    ok = ops.distillation(x, t, q, stats=True)
    one = torch.zeros(2, dtype=torch.int64, device="cuda")
    bad = [lambda: ops.distillation(x.double(), t, q), lambda: ops.distillation(x, t.float(), q), lambda: ops.distillation(x, t[:1], q),
           lambda: ops.distillation(x, t, q[:, :2]), lambda: ops.distillation(x, t[:, :0], q[:, :0]), lambda: ops.distillation(x, t[0], q[0]),
           lambda: ops.distillation(x, t.repeat(1, 100), q.repeat(1, 100)), lambda: ops.distillation(x, t.cpu(), q), lambda: ops.distillation(x, t, q.cpu()),
           lambda: ops.distillation(x, t, q, scale=0.0), lambda: ops.distillation(x, t, q, scale=INF), lambda: ops.distillation(x, t, q, beta=-0.1),
           lambda: ops.distillation(x, t, q, beta=1.5), lambda: ops.distillation(x, t, q, beta=math.nan), lambda: ops.distillation(x, t, q, targets=one[:1]),
           lambda: ops.distillation(x, t, q, targets=one.float()), lambda: ops.distillation(x, t, q, targets=one.cpu()), lambda: ops.distillation(x[:, :0], t, q),
           lambda: ops.distillation_grad(x, t, ok.stats[:, :-1], ok.loss), lambda: ops.distillation_grad(x, t, ok.stats.double(), ok.loss),
           lambda: ops.distillation_grad(x, t, ok.stats, ok.loss[:1]), lambda: ops.distillation_grad(x, t, ok.stats, grad_logp=ok.loss),
           lambda: ops.distillation_grad(x, t, ok.stats, ok.loss, into=x[:1]), lambda: ops.distillation_grad(x, t, ok.stats, ok.loss, into=x.half()),
           lambda: ops.distillation_grad(x, t, ok.stats, ok.loss, first=-1), lambda: ops.distillation_parts(x[None], t, q, first=0),
           lambda: ops.distillation_parts(x, t, q, first=2 ** 31 - 5), lambda: ops.join_distillation([], t, q, 10),
           lambda: ops.join_distillation([ops.distillation_parts(x, t, q, first=0)], t[:, :2], q[:, :2], 10),
           lambda: ops.join_distillation([ops.distillation_parts(x, t, q, first=0)] * 65, t, q, 650),
           lambda: ops.join_distillation([ops.distillation_parts(x, t, q, first=0)], t, q, 0)]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was not refused")


# ---- adjusted logits ---------------------------------------------------------------------------------------
def history_of(g, n, H, V, index=torch.int64):
    t = torch.randint(-1, V + 2, (n, H), generator=g)
    t[torch.rand(n, H, generator=g) < 0.3] = V // 2
    return t.to(index).cuda()


def check_adjusted(x, dtype=None, **given):
    got = ops.adjust_logits(x, dtype=dtype, **given)
    ref, bound = C.adjusted(x, **given)
    assert got.dtype == (dtype or x.dtype)
    C.close(got, ref, bound + C.rounded(ref, got.dtype), "adjusted")
    back = {k: v for k, v in given.items() if k in ("history", "lengths", "repetition", "allowed", "scale", "first")}
    grad = normal(gen(98), *x.shape, dtype=got.dtype)
    d = ops.adjust_logits_grad(x, grad, **back)
    want, bound = C.adjusted_grad(x, grad, **back)
    assert d.dtype == x.dtype
    C.close(d, want, bound + C.rounded(want, x.dtype), "gradient")
    bits = lambda t: t.view(torch.int32 if t.dtype == F32 else torch.int16)   # noqa: E731
    place = x.clone(memory_format=torch.contiguous_format)
    same = ops.adjust_logits(place, **given)
    assert ops.adjust_logits(place, into=place, **given) is place
    assert torch.equal(bits(place), bits(same))
    return got


ADJUST = [  # rows, vocabulary, places
    (1, 1, 1), (2, 7, 0), (3, 33, 5), (1, 1000, 1), (4, 4099, 3000), (2, 8192, 100), (2, 16390, 257), (3, 50257, 700), (1, 128256, 2049), (1030, 40, 9)]


@pytest.mark.parametrize("out", [None, F32], ids=["same", "float32"])
@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("case", ADJUST, ids=str)
def test_adjusted_sizes(case, dtype, out):
    n, V, H = case
    g = gen(n + V)
    x = normal(g, n, V, dtype=dtype, size=2.0)
    each = lambda lo, hi: (lo + (hi - lo) * torch.rand(n, generator=g)).cuda()   # noqa: E731
    B = min(V, 13)
    check_adjusted(x, out, history=history_of(g, n, H, V, torch.int32 if V % 2 else torch.int64),
                   lengths=torch.randint(0, H + 1, (n,), generator=g).to(torch.int32 if H % 2 else torch.int64).cuda(),
                   prompts=torch.randint(0, H // 2 + 1, (n,), generator=g).cuda(), repetition=each(0.5, 2), frequency=each(-0.5, 1),
                   presence=each(-0.5, 1), bias_tokens=torch.randint(0, V, (n, B), generator=g).cuda(), bias=normal(g, n, B, size=3.0),
                   allowed=C.words_of(torch.rand(n, V, generator=g) < 0.6).cuda(), scale=each(0.5, 2))


@pytest.mark.parametrize("parts", ["history", "bias", "mask", "scale", "history bias", "mask scale", "history mask", "history bias mask"])
def test_adjusted_parts(parts):
    """Each part alone and some together, numbers for all rows, one history, one list of biases and one mask for all rows."""
    g = gen(20)
    for dtype in TYPES:
        x = normal(g, 4, 3001, dtype=dtype, size=2.0)
        given = {}
        if "history" in parts:
            given.update(history=history_of(g, 1, 90, 3001)[0], repetition=1.3, frequency=0.25, presence=0.5)
        if "bias" in parts:
            given.update(bias_tokens=torch.tensor([5, 3000, 5, -1, 3001, 0], dtype=torch.int32).cuda(), bias=normal(g, 6, size=3.0))
        if "mask" in parts:
            given.update(allowed=C.words_of(torch.rand(3001, generator=g) < 0.05).cuda())
        if "scale" in parts:
            given.update(scale=0.7)
        check_adjusted(x, **given)
        if parts == "history":
            check_adjusted(x, history=given["history"], frequency=1.0)
            check_adjusted(x, history=given["history"][None].expand(4, 90), repetition=0.5)


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_masks(dtype):
    """Rows that are left nothing or everything, NaN and inf in masked places, words with more tokens than the vocabulary, uint32."""
    g = gen(21)
    x = normal(g, 6, 1037, dtype=dtype)
    ok = torch.rand(6, 1037, generator=g) < 0.5
    ok[0], ok[1] = False, True
    ok[2], ok[2, 1036] = False, True
    x[3, ~ok[3].cuda()] = math.nan
    x[4, ~ok[4].cuda()] = INF
    x[5] = -INF
    words = C.words_of(ok)
    words = torch.cat([words, torch.full((6, 3), -1, dtype=torch.int32)], 1)
    words[:, 32] |= ~((1 << (1037 % 32)) - 1)            # tokens behind the last
    got = check_adjusted(x, allowed=words.cuda())
    assert (got[0] == -INF).all() and torch.equal(got[1], x[1]) and not torch.isnan(got).any()
    assert torch.equal(got, ops.adjust_logits(x, allowed=words.cuda().view(torch.uint32)))
    grad = torch.full((6, 1037), math.nan, dtype=dtype, device="cuda")
    d = ops.adjust_logits_grad(x, grad, allowed=words.cuda())
    assert torch.equal(torch.isnan(d).cpu(), ok)
    logp = ops.token_logprobs(got, torch.zeros(6, dtype=torch.int64, device="cuda"))
    assert logp.lse[0].item() == -INF and torch.isfinite(logp.lse[1:5]).all()


def test_in_place_writes_only_what_changes():
    """Quiet NaNs with a payload, which no arithmetic leaves alone, stay where nothing changes."""
    g = gen(22)
    x = normal(g, 3, 2049)
    bits = x.view(torch.int32)
    bits[:, ::7] = 0x7FA00001
    ok = torch.rand(3, 2049, generator=g) < 0.5
    ok[1] = True
    before = bits.clone()
    ops.adjust_logits(x, history=torch.tensor([[1, 1, 2048, -1]] * 3).cuda(), frequency=1.0, allowed=C.words_of(ok).cuda(), into=x)
    same = bits == before
    assert same[1, 8:2040].all() and not same[1, 1] and not same[1, 2048]     # (16 bytes at a time)
    assert (x.cpu()[~ok] == -INF).all()


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_adjusted_strides_shapes_and_shards(dtype):
    g = gen(23)
    n, V, H = 6, 1111, 40
    wide = normal(g, n, 1200, dtype=dtype, size=2.0)
    history = history_of(g, n, 2 * H, V)[:, ::2]
    kept = history_of(g, n, 100, V)[:, 3:43]
    mask = C.words_of(torch.rand(n, 1300, generator=g) < 0.5).cuda()
    rep = (1 + torch.rand(2 * n, generator=g)).cuda()[::2]
    for x in (wide[:, 1:1112], wide[:, 3:1114], normal(g, V, n, dtype=dtype).t()):
        check_adjusted(x, history=history, repetition=rep, allowed=mask[:, :35], scale=rep)
        check_adjusted(x, history=kept, repetition=rep, frequency=0.1, allowed=mask[:, 2:40])
    x = wide[:, :V].reshape(2, 3, V)
    lengths = torch.randint(0, H, (2, 3), generator=g).cuda()
    whole = dict(history=kept.reshape(2, 3, 40), lengths=lengths, prompts=lengths // 2, repetition=rep.reshape(2, 3), presence=0.5,
                 bias_tokens=torch.randint(0, V, (2, 3, 5), generator=g).cuda(), bias=normal(g, 2, 3, 5), allowed=mask.reshape(2, 3, -1), scale=1.5)
    got = ops.adjust_logits(x, **whole)
    ref, bound = C.adjusted(x, **whole)
    C.close(got, ref, bound + C.rounded(ref, dtype))
    edges = [0, 1, 400, 417, 1110, 1111]
    pieces = [ops.adjust_logits(x[..., a:b], first=a, **whole) for a, b in zip(edges, edges[1:])]
    assert torch.equal(torch.cat(pieces, -1), got)
    back = {k: whole[k] for k in ("history", "lengths", "repetition", "allowed", "scale")}
    grad = normal(g, 2, 3, V, dtype=dtype)
    d = ops.adjust_logits_grad(x, grad, **back)
    pieces = [ops.adjust_logits_grad(x[..., a:b], grad[..., a:b], first=a, **back) for a, b in zip(edges, edges[1:])]
    assert torch.equal(torch.cat(pieces, -1), d)
    place = grad.clone()
    assert torch.equal(ops.adjust_logits_grad(x, place, into=place, **back), d)
    one = ops.adjust_logits(x[0, 0], history=kept[0], repetition=1.5)
    assert torch.equal(one, ops.adjust_logits(x[:1, 0], history=kept[:1], repetition=1.5)[0])
    assert ops.adjust_logits(x[:0], history=kept.reshape(2, 3, 40)[:0]).shape == (0, 3, V)
    # lengths and prompts from outside their ranges
    odd = torch.tensor([-5, 1000, 0, 40, 41, 3]).cuda()
    assert torch.equal(ops.adjust_logits(wide[:, :V], history=kept, lengths=odd, prompts=-odd, frequency=1.0),
                       ops.adjust_logits(wide[:, :V], history=kept, lengths=odd.clamp(0, 40), frequency=1.0))


def test_many_biases_and_long_histories():
    g = gen(24)
    x = normal(g, 2, 9000)
    tokens = torch.randint(0, 9000, (2, 1024), generator=g)
    tokens[0, 500:520] = tokens[0, 3]
    check_adjusted(x, bias_tokens=tokens.cuda(), bias=normal(g, 2, 1024))
    check_adjusted(x, bias_tokens=tokens[:, :0].cuda(), bias=torch.zeros(2, 0, device="cuda"), scale=2.0)
    # entries of 32 bits and all the biases that a row may have: the most LDS that a call takes
    wide, long = normal(g, 2, 40000, dtype=BF16), history_of(g, 2, 17000, 40000)
    check_adjusted(wide, history=long, repetition=1.1, frequency=0.01, bias_tokens=torch.randint(0, 40000, (2, 1024), generator=g).cuda(), bias=normal(g, 2, 1024))
    check_adjusted(x, history=history_of(g, 2, 70001, 9000), repetition=1.1, frequency=0.01, prompts=torch.tensor([70000, 35000]).cuda())


@pytest.mark.parametrize("places", [0, 40, 17000])
def test_adjusted_logits_that_no_cache_holds(places):
    """More than 256 MB: the same bits as rows by themselves have."""
    g = gen(26)
    n, V = 1100, 128250
    x = torch.randn(n, V, device="cuda").to(BF16)
    given = dict(allowed=C.words_of(torch.rand(V, generator=g) < 0.5).cuda(), scale=(0.5 + torch.rand(n, generator=g)).cuda())
    if places:
        given.update(history=torch.randint(0, V, (n, places), generator=g).cuda(), repetition=(0.5 + torch.rand(n, generator=g)).cuda())
    more = dict(given, bias_tokens=torch.randint(0, V, (n, 9), generator=g).cuda(), bias=normal(g, n, 9)) if places else given
    some = torch.tensor([0, 1, n // 2, n - 1]).cuda()
    of = lambda d: {k: v if v.dim() == 1 and k == "allowed" else v[some] for k, v in d.items()}   # noqa: E731
    y = ops.adjust_logits(x, **more)
    part = ops.adjust_logits(x[some], **of(more))
    assert torch.equal(y[some], part)
    ref, bound = C.adjusted(x[some[:1]], **{k: v if k == "allowed" else v[:1] for k, v in of(more).items()})
    C.close(part[:1], ref, bound + C.rounded(ref, BF16))
    d = ops.adjust_logits_grad(x, x, **given)
    assert torch.equal(d[some], ops.adjust_logits_grad(x[some], x[some], **of(given)))


def test_adjusted_through_autograd():
    g = gen(25)
    x = normal(g, 3, 700, size=2.0)
    history = history_of(g, 3, 50, 700)
    given = dict(history=history, repetition=torch.tensor([1.0, 1.5, 0.75]).cuda(), frequency=0.5, allowed=C.words_of(torch.rand(3, 700, generator=g) < 0.5).cuda(),
                 scale=0.5)
    weight = normal(g, 3, 700)
    for dtype in (None, F32):
        for kind in TYPES:
            leaf = x.clone().to(kind).requires_grad_(True)
            y = ops.adjust_logits(leaf, dtype=dtype, **given)
            torch.where(torch.isfinite(y), y.float() * weight, 0.0).sum().backward()
            d = torch.where(torch.isfinite(y), weight, 0.0).to(y.dtype)
            want = ops.adjust_logits_grad(leaf.detach(), d, history, repetition=given["repetition"], allowed=given["allowed"], scale=0.5)
            assert torch.equal(leaf.grad, want)
    # differences of the plain form, away from 0 where a repetition has a kink
    ref = lambda z: C.adjusted(z, **{**given, "allowed": None})[0]   # noqa: E731
    z, h = x.cpu().double(), 1e-4
    leaf = x.clone().requires_grad_(True)
    (ops.adjust_logits(leaf, **{**given, "allowed": None}) * weight).sum().backward()
    for i, j in ((0, 350), (1, 350), (2, 350), (1, 3), (2, 699)):
        assert abs(z[i, j]) > h
        up, down = z.clone(), z.clone()
        up[i, j] += h
        down[i, j] -= h
        slope = ((ref(up) - ref(down)) * weight.cpu().double()).sum().item() / (2 * h)
        assert abs(slope - leaf.grad[i, j].item()) <= 1e-6 * (1 + abs(slope)), (i, j)
    plain = x.clone().requires_grad_(True)       # without a repetition nothing is kept but the mask and the scale
    ops.adjust_logits(plain, history, frequency=1.0, scale=2.0).sum().backward()
    assert (plain.grad == 2.0).all()
    with pytest.raises(ValueError, match="into"):
        ops.adjust_logits(plain, scale=2.0, into=torch.empty_like(x))
    with pytest.raises(ValueError, match="no gradient"):
        ops.adjust_logits(plain, scale=torch.ones(3, device="cuda", requires_grad=True))
    y = x.clone()
    version = y._version
    ops.adjust_logits(y, scale=2.0, into=y)
    assert y._version > version


def test_adjust_refusals():
    x, h = torch.zeros(2, 70, device="cuda"), torch.zeros(2, 3, dtype=torch.int64, device="cuda")
    v, m = torch.ones(2, device="cuda"), torch.zeros(2, 3, dtype=torch.int32, device="cuda")
    b = torch.zeros(2, 3, device="cuda")
    bad = [lambda: ops.adjust_logits(x.double()), lambda: ops.adjust_logits(x, h.float()), lambda: ops.adjust_logits(x, h[:1]), lambda: ops.adjust_logits(x, h.cpu()),
           lambda: ops.adjust_logits(x, h, lengths=v), lambda: ops.adjust_logits(x, h, lengths=h[:1, 0]), lambda: ops.adjust_logits(x, h, lengths=3),
           lambda: ops.adjust_logits(x, h, prompts=h), lambda: ops.adjust_logits(x, h, repetition=0.0), lambda: ops.adjust_logits(x, h, repetition=-1.0),
           lambda: ops.adjust_logits(x, h, repetition=v[:1]), lambda: ops.adjust_logits(x, h, frequency=math.nan), lambda: ops.adjust_logits(x, h, presence=INF),
           lambda: ops.adjust_logits(x, repetition=1.5), lambda: ops.adjust_logits(x, lengths=h[:, 0]), lambda: ops.adjust_logits(x, scale=0.0),
           lambda: ops.adjust_logits(x, scale=v.cpu()), lambda: ops.adjust_logits(x, scale=-1.0), lambda: ops.adjust_logits(x, bias=b), lambda: ops.adjust_logits(x, bias_tokens=h),
           lambda: ops.adjust_logits(x, bias_tokens=h, bias=b[:, :2]), lambda: ops.adjust_logits(x, bias_tokens=h.repeat(1, 400), bias=b.repeat(1, 400)),
           lambda: ops.adjust_logits(x, bias_tokens=h.float(), bias=b), lambda: ops.adjust_logits(x, allowed=m[:, :2]), lambda: ops.adjust_logits(x, allowed=m.long()),
           lambda: ops.adjust_logits(x, allowed=m > 0), lambda: ops.adjust_logits(x, allowed=m[:1]), lambda: ops.adjust_logits(x, allowed=m, first=64),
           lambda: ops.adjust_logits(x, allowed=m.cpu()), lambda: ops.adjust_logits(x, dtype=F16), lambda: ops.adjust_logits(x.half(), dtype=BF16),
           lambda: ops.adjust_logits(x, first=-1), lambda: ops.adjust_logits(x, into=x[:1]), lambda: ops.adjust_logits(x.half(), into=x, dtype=F16),
           lambda: ops.adjust_logits(x, into=torch.zeros(70, 2, device="cuda").t()), lambda: ops.adjust_logits_grad(x, x[:1]), lambda: ops.adjust_logits_grad(x, x.half()),
           lambda: ops.adjust_logits_grad(x, x, into=x.half()), lambda: ops.adjust_logits_grad(x, x, repetition=2.0)]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was not refused")


# ---- together, streams, graphs -----------------------------------------------------------------------------
def test_a_teacher_trains_a_student():
    """A teacher's adjusted logits, its most likely tokens, the student's loss by them and its gradient, as a program runs them."""
    g = gen(30)
    n, V, K = 12, 5000, 20
    student, teacher_logits = normal(g, n, V, size=2.0).requires_grad_(True), normal(g, n, V, dtype=BF16, size=2.0)
    words = C.words_of(torch.rand(V, generator=g) < 0.5).cuda()
    targets = torch.randint(0, V, (n,), generator=g).cuda()
    with torch.no_grad():
        chosen = ops.adjust_logits(teacher_logits, allowed=words, scale=0.5, dtype=F32)
        t = ops.token_logprobs(chosen, targets, top=K)
    masked = ops.adjust_logits(student, allowed=words)
    r = ops.distillation(masked, t.top_tokens, t.top_logp, scale=0.5, targets=targets)
    assert torch.isfinite(r.loss).all() and (r.loss > 0).all()
    r.loss.mean().backward()
    ok = C.allowed_of(words, 1, V, 0)[0]
    z = torch.where(ok, student.detach().cpu().double(), -INF)
    d = C.distillation(z.float(), t.top_tokens, t.top_logp, 0.5, 0.0, True)
    C.close(r.loss, d[0], d[4], "loss")
    C.close(student.grad, d[3] * 0.5 / n, d[7] * 0.5 / n + 4 * C.U * d[3].abs(), "gradient")
    assert (student.grad.cpu()[:, ~ok] == 0).all()


def calls(g, n=5, V=6000):
    """(function of x, inputs) of each operator, for streams and graphs"""
    tokens, teacher = lists(g, n, V, 30)
    history, words = history_of(g, n, 500, V), C.words_of(torch.rand(n, V, generator=g) < 0.5).cuda()
    ones = torch.ones(n, device="cuda")

    def distill(x):
        r = ops.distillation(x, tokens, teacher, beta=0.5, targets=tokens[:, 0], stats=True)
        return r.loss, r.lse, r.logp, ops.distillation_grad(x, tokens, r.stats, ones, targets=tokens[:, 0], grad_logp=ones)

    def adjust(x):
        y = ops.adjust_logits(x, history, repetition=1.25, frequency=0.5, allowed=words, scale=ones * 0.5)
        return y, ops.adjust_logits_grad(x, x, history, repetition=1.25, allowed=words, scale=ones * 0.5)

    return distill, adjust


def test_streams_other_than_the_default():
    g = gen(31)
    x = normal(g, 5, 6000)
    for f in calls(g):
        want = f(x)
        torch.cuda.synchronize()
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            y = torch.empty_like(x)
            for _ in range(3):       # work that has to come first
                y.copy_(x)
                y.mul_(1.0)
            got = f(y)
        stream.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_two_threads():
    g = gen(32)
    x, (distill, adjust) = normal(g, 5, 6000), calls(g)
    want, failed = {distill: distill(x), adjust: adjust(x)}, []
    torch.cuda.synchronize()

    def work(f):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got = f(x)
                torch.cuda.current_stream().synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, want[f])):
                    failed.append(f)
                    return

    threads = [threading.Thread(target=work, args=(f,)) for f in (distill, adjust, distill, adjust)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed


def test_captured_and_replayed():
    """Two graphs in one pool, replayed in turn with eager calls and new inputs between them."""
    g = gen(33)
    fs = calls(g)
    static = [normal(g, 5, 6000), normal(g, 5, 6000)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for f, x in zip(fs, static):
            f(x)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs, results = [], []
    for f, x in zip(fs, static):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=graphs[0].pool() if graphs else None):
            results.append(f(x))
        graphs.append(graph)
    for turn in range(4):
        for i in (0, 1):
            static[i].copy_(normal(g, 5, 6000, size=1.0 + turn))
            graphs[i].replay()
            torch.cuda.synchronize()
            got = [t.clone() for t in results[i]]
            for a, b in zip(got, fs[i](static[i])):
                assert torch.equal(a, b), (turn, i)


def test_offsets_above_32_bits():
    """Rows behind the first 2^31 elements of their tensor."""
    n, V = 3, 800_000_000
    if torch.cuda.mem_get_info()[0] < 12 * 2 ** 30:
        pytest.skip("needs 12 GiB")
    g = gen(34)
    base = torch.empty(n * V, dtype=BF16, device="cuda")
    x = base.as_strided((n, 2000), (V, 1))
    x.copy_(normal(g, n, 2000, dtype=BF16))
    tokens, teacher = lists(g, n, 2000, 8)
    r = check_distillation(x, tokens, teacher, 1.0, 0.0, True)
    want = ops.distillation_grad(x.contiguous(), tokens, r.stats, r.loss)
    y = base.as_strided((n, 2000), (V, 1), 4000)
    assert torch.equal(ops.distillation_grad(x, tokens, r.stats, r.loss, into=y), want)
    want = ops.adjust_logits(x.contiguous(), history=tokens, frequency=1.0, scale=2.0)
    assert torch.equal(ops.adjust_logits(x, history=tokens, frequency=1.0, scale=2.0, into=x), want)
