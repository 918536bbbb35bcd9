"""The operators at a model's two ends against plain forms in 64 bits (operator_cases.py), at the sizes, strides and masks where
they can go wrong.  Bounds follow from the operators' arithmetic: how many float32 roundings a result is behind, and one
rounding to its type."""
import math

import pytest

torch = pytest.importorskip("torch")   # before the library: one HIP runtime in the process

import operator_cases as C   # noqa: E402
from galvatron_dp import operators as ops   # noqa: E402

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = [F32, F16, BF16]
ids = lambda v: str(v).replace("torch.", "") if isinstance(v, torch.dtype) else None   # noqa: E731


def gen(seed):
    return torch.Generator().manual_seed(seed)


def normal(g, *shape, dtype=F32, size=1.0):
    return (torch.randn(*shape, generator=g) * size).to(dtype).cuda()


def tokens_of(g, n, vocab, dtype=torch.int64, frequent=0.3):
    t = torch.randint(0, vocab, (n,), generator=g)
    t[torch.rand(n, generator=g) < frequent] = vocab // 3
    return t.to(dtype).cuda()


# ---- embedding ---------------------------------------------------------------------------------------------
EMBED = [  # tokens, rows, dim, first, scale
    (1, 1, 1, 0, 1.0), (3, 5, 7, 0, 2.0), (64, 1000, 64, 0, 8.0), (65, 257, 100, 40, 0.5), (700, 300, 1023, 0, 1.0),
    (513, 2000, 1024, 1000, 31.9), (9000, 90, 36, 0, 1.0), (33, 70, 8200, 0, 1.0), (0, 5, 8, 0, 1.0), (5, 0, 8, 0, 1.0)]


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("case", EMBED, ids=str)
def test_embedding(case, dtype):
    n, rows, dim, first, scale = case
    g = gen(1)
    w = normal(g, rows, dim, dtype=dtype)
    t = tokens_of(g, n, rows + 2 * first + 1, torch.int32 if n % 2 else torch.int64)
    if n > 2:
        t[0], t[1] = -1, rows + first     # of no shard, and the first of the next one
    got = ops.embedding(t, w, scale=scale, first=first)
    assert got.dtype == dtype
    ref = C.embedding(t, w, scale, first)
    C.close(got, ref, C.rounded(ref, dtype) + C.U * 1.01 * ref.abs())


@pytest.mark.parametrize("out", TYPES, ids=ids)
@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_embedding_types_strides_and_shapes(dtype, out):
    """A table within a wider one, from its second column on (no row begins on 16 bytes), tokens with strides."""
    g = gen(2)
    w = normal(g, 50, 73, dtype=dtype)[:, 1:65]
    t = tokens_of(g, 60, 50).reshape(5, 12)[:, ::2]
    got = ops.embedding(t, w, scale=1.7, dtype=out)
    assert got.shape == (5, 6, 64) and got.dtype == out
    ref = C.embedding(t, w, 1.7, 0)
    C.close(got, ref, C.rounded(ref, out) + 2 * C.U * ref.abs())


GRAD = [  # tokens, rows, dim, first, scale, share of one token
    (1, 1, 1, 0, 1.0, 0.0), (2, 3, 5, 0, 2.0, 1.0), (64, 1000, 64, 0, 8.0, 0.3), (65, 257, 100, 40, 0.5, 0.3),
    (700, 300, 1023, 0, 1.0, 0.1), (5000, 700, 24, 300, 1.0, 0.5), (3000, 2, 8, 0, 1.0, 0.5), (4097, 9, 2056, 0, 1.5, 1.0),
    (1000, 140001, 4, 0, 1.0, 0.2), (70000, 3000, 8, 1000, 1.0, 0.05), (0, 7, 16, 0, 1.0, 0.0), (9, 0, 16, 0, 1.0, 0.0)]


@pytest.mark.parametrize("into", [False, True], ids=["all", "into"])
@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("case", GRAD, ids=str)
def test_embedding_grad(case, dtype, into):
    n, rows, dim, first, scale, frequent = case
    g = gen(3)
    t = tokens_of(g, n, rows + 2 * first + 1, torch.int32 if n % 2 else torch.int64, frequent)
    d = normal(g, n, dim, dtype=dtype)
    ref, bound = C.embedding_grad(t, d, rows, scale, first)
    if into:
        main = normal(g, rows, dim)
        before = main.cpu().double()
        assert ops.embedding_grad(t, d, rows, scale=scale, first=first, into=main) is main
        C.close(main, before + ref, bound + C.rounded(before + ref, F32))
        assert torch.equal(main.cpu().double()[bound.amax(1) == 0], before[bound.amax(1) == 0])
    else:
        got = ops.embedding_grad(t, d, rows, scale=scale, first=first)
        C.close(got, ref, bound + C.rounded(ref, dtype))
        again = ops.embedding_grad(t, d, rows, scale=scale, first=first)
        assert torch.equal(got, again), "the same inputs give the same bits"


def test_embedding_grad_types_strides_and_broadcast():
    g = gen(4)
    t = tokens_of(g, 48, 20).reshape(6, 8)
    wide = normal(g, 6, 8, 41, dtype=BF16)
    for d in (wide[..., 1:33], torch.ones(1, 1, 32, device="cuda").expand(6, 8, 32), torch.tensor(0.5, device="cuda").expand(6, 8, 32),
              normal(g, 6, 32, 8).transpose(1, 2), normal(g, 8, 6, 32, dtype=F16).transpose(0, 1)):
        for dtype in TYPES:
            ref, bound = C.embedding_grad(t, d, 20, 1.0, 0)
            C.close(ops.embedding_grad(t, d, 20, dtype=dtype), ref, bound + C.rounded(ref, dtype))
    main = torch.zeros(20, 65, dtype=BF16, device="cuda")[:, 1:33]      # rows within a wider buffer
    ops.embedding_grad(t, wide[..., 1:33], 20, into=main)
    ref, bound = C.embedding_grad(t, wide[..., 1:33], 20, 1.0, 0)
    C.close(main, ref, bound + C.rounded(ref, BF16))
    assert not main._base[:, 0].any() and not main._base[:, 33:].any()


def test_embedding_shards_add_up_and_autograd():
    g = gen(5)
    w = normal(g, 96, 40).requires_grad_()
    t = tokens_of(g, 200, 96)
    d = normal(g, 200, 40)
    whole = ops.embedding(t, w, scale=3.0)
    parts = [ops.embedding(t, w[a:a + 32], scale=3.0, first=a) for a in (0, 32, 64)]
    assert torch.equal(whole, sum(parts))
    grad, = torch.autograd.grad(whole, w, d)
    ref, bound = C.embedding_grad(t, d, 96, 3.0, 0)
    C.close(grad, ref, bound + C.rounded(ref, F32))
    grad, = torch.autograd.grad(ops.embedding(t, w, scale=3.0).sum(), w)      # a gradient that all places share
    ref, bound = C.embedding_grad(t, torch.ones(200, 40), 96, 3.0, 0)
    C.close(grad, ref, bound + C.rounded(ref, F32))
    # differences: the lookup is linear, so they are exact up to rounding
    v = normal(g, 96, 40)
    up, down = ((ops.embedding(t, (w + s * v).detach(), scale=3.0).double() * d).sum() for s in (0.5, -0.5))
    along = (torch.autograd.grad(ops.embedding(t, w, scale=3.0), w, d)[0].double() * v).sum()
    size = (C.embedding(t, w, 3.0, 0).abs() * d.cpu().abs()).sum().item() + (C.embedding(t, v, 3.0, 0).abs() * d.cpu().abs()).sum().item()
    assert abs((up - down - along).item()) <= 300 * C.U * size


# ---- log probabilities ---------------------------------------------------------------------------------------
LOGPROB = [  # rows, vocab, top, scale
    (1, 1, 1, 1.0), (3, 2, 2, 1.0), (5, 7, 7, 0.5), (2, 31, 20, 1.25), (4, 500, 64, 1.0), (3, 4097, 5, 2.0), (2, 50257, 20, 1.0),
    (1, 70001, 1, 1.0), (2, 262144 + 5, 3, 0.8), (1, 600003, 64, 1.0), (2100, 333, 4, 1.0), (2048, 2065, 20, 1.0), (0, 9, 2, 1.0)]


def check_logprobs(x, t, r, scale, top):
    logp, lse, entropy, every = C.logprobs(x, t, scale)
    of_lse, of_logp, of_entropy = C.logprob_bound(x, scale)
    C.close(r.lse, lse, of_lse, "lse")
    C.close(r.logp, logp, of_logp, "logp")
    C.close(r.entropy, entropy, of_entropy, "entropy")
    if top:
        at = C.top_of(x, top)
        assert torch.equal(r.top_tokens.cpu(), at)
        C.close(r.top_logp, every.gather(-1, at), of_logp[..., None], "top_logp")


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("case", LOGPROB, ids=str)
def test_token_logprobs(case, dtype):
    n, vocab, top, scale = case
    g = gen(6)
    x = normal(g, n, vocab, dtype=dtype, size=3.0)
    t = tokens_of(g, n, vocab, torch.int32 if n % 2 else torch.int64)
    if n > 1:
        t[-1] = -100
    if n > 2:
        t[-2] = vocab
    r = ops.token_logprobs(x, t, scale=scale, entropy=True, top=top)
    check_logprobs(x, t, r, scale, top)
    plain = ops.token_logprobs(x, t, scale=scale)
    assert plain.entropy is None and plain.top_logp is None and plain.top_tokens is None
    C.close(plain.logp, r.logp.cpu().double(), C.logprob_bound(x, scale)[1])


@pytest.mark.parametrize("n", [6, 2054])      # rows in slices, and whole
@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_token_logprobs_masks(dtype, n):
    """Tokens ruled out by -inf and by the type's lowest value; rows of which nothing is left; NaN and +inf; ties."""
    g = gen(7)
    vocab, top = 9001, 6
    x = normal(g, n, vocab, dtype=dtype, size=2.0)
    t = tokens_of(g, n, vocab)
    low = torch.finfo(dtype).min
    out = (torch.rand(vocab, generator=g) < 0.7).cuda()
    out[t[:2]] = False
    x[0, out] = -math.inf
    x[1, out] = low
    x[2] = -math.inf
    x[3] = low
    x[4, 17], x[5, 33] = math.nan, math.inf
    x[5, 40] = -math.inf
    t[2] = 5
    if n > 6:
        x[6] = -math.inf
        x[6, 8998:] = torch.tensor([0.0, -0.0, 1.0], dtype=dtype)     # fewer than top are left; 0 and -0 are equal
        x[7] = 1.5                                                    # all equal
        t[6], t[7] = 3, 9000                                          # a token that is ruled out
    r = ops.token_logprobs(x, t, entropy=True, top=top)
    logp, lse, entropy, every = C.logprobs(x, t, 1.0)
    of_lse, of_logp, of_entropy = C.logprob_bound(x, 1.0)
    assert torch.isnan(r.lse[4:6]).all() and torch.isnan(r.logp[4:6]).all() and torch.isnan(r.entropy[4:6]).all()
    assert r.lse[2] == -math.inf and r.logp[2] == -math.inf and r.entropy[2] == 0 and (r.top_logp[2] == -math.inf).all()
    if dtype != F16:       # the row of the lowest value: all alike
        assert abs(r.logp[3].item() + math.log(vocab)) < 1e-4 and abs(r.entropy[3].item() - math.log(vocab)) < 1e-4
    good = torch.tensor([i for i in range(n) if i not in (2, 3, 4, 5)])
    for got, ref, bound in ((r.lse, lse, of_lse), (r.logp, logp, of_logp), (r.entropy, entropy, torch.full_like(lse, of_entropy))):
        C.close(got[good.cuda()], ref[good], bound[good])
    at = C.top_of(x, top)
    at[5] = r.top_tokens[5].cpu()
    assert r.top_tokens[5, 0] == 33
    assert torch.equal(r.top_tokens.cpu(), at)
    C.close(r.top_logp[good.cuda()], every.gather(-1, at)[good], of_logp[good, None])


def test_token_logprobs_strides_and_shapes():
    g = gen(8)
    wide = normal(g, 4, 6, 1111, dtype=BF16, size=2.0)
    t = tokens_of(g, 24, 1000).reshape(4, 6)
    for x in (wide[..., 1:1001], wide[..., 7:1007], wide[..., ::1][..., :1000], normal(g, 4, 1000, 6).transpose(1, 2),
              normal(g, 1, 1, 1000).expand(4, 6, 1000)):
        r = ops.token_logprobs(x, t, entropy=True, top=3)
        assert r.logp.shape == (4, 6) and r.top_tokens.shape == (4, 6, 3)
        check_logprobs(x, t, r, 1.0, 3)
    one = normal(g, 777)
    r = ops.token_logprobs(one, torch.tensor(5, device="cuda"), entropy=True, top=2)
    assert r.logp.shape == ()
    check_logprobs(one, torch.tensor(5), r, 1.0, 2)


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("cuts", [(0, 100), (0, 33, 100), (0, 1, 2, 50, 99, 100)], ids=str)
def test_parts_of_a_vocabulary(cuts, dtype):
    """Shards of any sizes, some smaller than the alternatives asked for, joined: the same as the whole, and its gradient."""
    g = gen(9)
    n, scale, top = 37, 1.3, 8
    vocab = 90 * cuts[-1] + 7
    cuts = [90 * c if c > 2 else c for c in cuts[:-1]] + [vocab]
    x = normal(g, n, vocab, dtype=dtype, size=2.0)
    x[3] = -math.inf
    x[4, : vocab // 2] = -math.inf
    t = tokens_of(g, n, vocab)
    t[5], t[4] = -100, vocab - 1
    shards = [x[:, a:b] for a, b in zip(cuts, cuts[1:])]
    parts = [ops.logprob_parts(s, t, first=a, scale=scale, top=top) for s, a in zip(shards, cuts)]
    r = ops.join_logprobs(parts, t, vocab, scale=scale, entropy=True)
    whole = ops.token_logprobs(x, t, scale=scale, entropy=True, top=top)
    of_lse, of_logp, of_entropy = C.logprob_bound(x, scale)
    for got, ref, bound in ((r.logp, whole.logp, of_logp), (r.lse, whole.lse, of_lse), (r.entropy, whole.entropy, torch.tensor(of_entropy)),
                            (r.top_logp, whole.top_logp, of_logp[:, None])):
        C.close(got, ref.cpu().double(), 2 * bound)
    assert torch.equal(r.top_tokens, whole.top_tokens)
    d, dh, dt = normal(g, n), normal(g, n), normal(g, n, top)
    grads = [ops.token_logprobs_grad(s, t, r.lse, d, scale=scale, entropy=r.entropy, grad_entropy=dh, top_tokens=r.top_tokens,
                                     grad_top=dt, first=a, vocab=vocab) for s, a in zip(shards, cuts)]
    ref, bound = C.logprobs_grad(x, t, r.lse, d, scale, entropy=r.entropy, d_entropy=dh, top=r.top_tokens, d_top=dt)
    C.close(torch.cat(grads, 1), ref, bound + C.rounded(ref, dtype))


@pytest.mark.parametrize("top,best", [(64, "last"), (64, "spread"), (33, "first")])
def test_join_of_64_parts(top, best):
    """As many parts and alternatives as there may be; the best all in one part, or in all of them."""
    g = gen(19)
    x = normal(g, 3, 64 * 70, size=2.0)
    if best != "spread":
        at = 63 * 70 if best == "last" else 0
        x[:, at:at + 70] += 100.0
    t = tokens_of(g, 3, 64 * 70)
    parts = [ops.logprob_parts(x[:, 70 * i:70 * (i + 1)], t, first=70 * i, top=top) for i in range(64)]
    check_logprobs(x, t, ops.join_logprobs(parts, t, 64 * 70, entropy=True), 1.0, top)


def test_offsets_above_32_bits():
    """Tensors of more than 2^31 elements: what lies at their ends."""
    g = gen(20)
    big = torch.empty(17000, 128256, dtype=BF16, device="cuda")
    big[-2:] = normal(g, 2, 128256, dtype=BF16, size=2.0)
    big[:-2] = 0
    t = torch.zeros(17000, dtype=torch.int64, device="cuda")
    t[-2:] = torch.tensor([128255, 7])
    r = ops.token_logprobs(big, t, entropy=True, top=3)
    check_logprobs(big[-2:], t[-2:], ops.TokenLogprobs(*(f[-2:] for f in r)), 1.0, 3)
    d = torch.ones(17000, device="cuda")
    ref, bound = C.logprobs_grad(big[-2:], t[-2:], r.lse[-2:], d[-2:], 1.0)
    ops.token_logprobs_grad(big, t, r.lse, d, into=big)
    C.close(big[-2:], ref, bound + C.rounded(ref, BF16))
    flat = big.view(-1)[:530000 * 4096].view(530000, 4096)      # a table, and a stream
    flat[-3:] = normal(g, 3, 4096, dtype=BF16)
    last = torch.tensor([529999, 529997, 530000, 529999], device="cuda")
    assert torch.equal(ops.embedding(last, flat)[[0, 1]], flat[[529999, 529997]])
    pre = norm_of(g, "rms", 4096, BF16)
    out = ops.residual_norm(flat, flat, pre=pre, stats=True)
    ref_stream, ref_normed = C.residual_norm(flat[-3:], flat[-3:], None, pre, None, 1.0, 1.0)
    C.close(out.stream[-3:], ref_stream, C.rounded(ref_stream, BF16))
    C.close(out.normed[-3:], ref_normed, norm_bound(ref_stream, pre, 8 * C.U * ref_stream.abs()) + C.rounded(ref_normed, BF16))
    d = normal(g, 4, 4096, dtype=BF16)
    grad = ops.embedding_grad(last, d, 530000)
    ref, bound = C.embedding_grad(last.cpu() - 529990, d, 10, 1.0, 0)
    C.close(grad[-10:], ref, bound + C.rounded(ref, BF16))
    assert not grad[:-10].any()


LOGPROB_GRAD = [(1, 1, 1.0), (3, 7, 0.5), (4, 500, 1.0), (3, 4097, 2.0), (2, 50257, 1.0), (300, 1025, 1.0), (2, 300001, 1.0), (0, 9, 1.0)]


@pytest.mark.parametrize("terms", ["logp", "lse", "entropy", "top", "all"])
@pytest.mark.parametrize("dtype", TYPES, ids=ids)
@pytest.mark.parametrize("case", LOGPROB_GRAD, ids=str)
def test_token_logprobs_grad(case, dtype, terms):
    n, vocab, scale = case
    g = gen(10)
    x = normal(g, n, vocab, dtype=dtype, size=2.0)
    t = tokens_of(g, n, vocab)
    if n > 2:
        t[0] = -100
        x[1, : vocab // 2] = -math.inf
        t[1] = vocab - 1
    k = min(3, vocab)
    r = ops.token_logprobs(x, t, scale=scale, entropy=True, top=k)
    if n > 2:
        t[2] = r.top_tokens[2, 1]        # the token is among the most likely ones
        x[n - 1] = -math.inf
        r.lse[n - 1] = -math.inf
    every = terms == "all"
    d = normal(g, n) if terms == "logp" or every else None
    more = {}
    if terms == "lse" or every:
        more["d_lse"] = normal(g, n)
    if terms == "entropy" or every:
        more.update(entropy=r.entropy, d_entropy=normal(g, n))
    if terms == "top" or every:
        more.update(top=r.top_tokens, d_top=normal(g, n, k))
    ref, bound = C.logprobs_grad(x, t, r.lse, d, scale, **more)
    names = {"d_lse": "grad_lse", "d_entropy": "grad_entropy", "top": "top_tokens", "d_top": "grad_top"}
    given = {names.get(a, a): b for a, b in more.items()}
    got = ops.token_logprobs_grad(x, t, r.lse, d, scale=scale, **given)
    C.close(got, ref, bound + C.rounded(ref, dtype))
    if vocab > 8:      # in rows that begin elsewhere than the logits', and in the logits' place
        other = torch.empty(n, vocab + 3, dtype=dtype, device="cuda")[:, 1:vocab + 1]
        assert torch.equal(ops.token_logprobs_grad(x, t, r.lse, d, scale=scale, into=other, **given), got)
        assert ops.token_logprobs_grad(x, t, r.lse, d, scale=scale, into=x, **given) is x and torch.equal(x, got)


def test_token_logprobs_autograd_and_differences():
    """Along a random direction the difference quotient of the operator's own float32 results is the gradient's product: with steps of
    2^-5 the cubic term is below 2^-10 * 2 of the direction's cube, rounding 2^5 times the results'."""
    g = gen(11)
    n, vocab = 12, 700
    x = normal(g, n, vocab, size=2.0)
    t = tokens_of(g, n, vocab)
    t[0] = -1
    a, b, c, d = normal(g, n), normal(g, n), normal(g, n, 4), normal(g, n)

    def loss(x):
        r = ops.token_logprobs(x, t, scale=0.9, entropy=True, top=4)
        return (r.logp * a).sum() + (r.entropy * b).sum() + (r.top_logp * c).sum() + (r.lse * d).sum()

    leaf = x.clone().requires_grad_()
    grad, = torch.autograd.grad(loss(leaf), leaf)
    for seed in range(3):
        v = normal(gen(100 + seed), n, vocab)
        v = v / v.norm()
        h = 2.0 ** -5
        along = ((loss(x + h * v) - loss(x - h * v)).double() / (2 * h)).item()
        size = a.abs().sum() + b.abs().sum() + c.abs().sum() + d.abs().sum()
        assert abs(along - (grad.double() * v).sum().item()) <= size.item() * (2.0 ** -9 + 64 * C.U * 20 / (2 * h))
    only = torch.autograd.grad(ops.token_logprobs(leaf, t).logp.sum(), leaf)[0]
    lse = ops.token_logprobs(x, t).lse
    ref, bound = C.logprobs_grad(x, t, lse, torch.ones(n), 1.0)
    C.close(only, ref, bound + C.rounded(ref, F32))


# ---- residual join and norms -----------------------------------------------------------------------------------
def norm_of(g, form, dim, dtype, weight=True):
    if form is None:
        return None
    w = (1 + 0.2 * normal(g, dim)).to(dtype) if weight else None
    return ops.Norm(form, w, (0.2 * normal(g, dim)).to(dtype) if weight and form == "layer" else None, 1e-5)


NORM = [  # rows, dim, post, pre, gates, types of block and stream
    (1, 1, "rms", "rms", 1, F32, F32), (2, 7, "layer", "layer", 2, BF16, BF16), (6, 64, None, "rms", 0, F16, F16),
    (5, 100, "rms", "layer", 5, BF16, F32), (8, 512, "rms", "rms", 2, BF16, BF16), (9, 1023, "layer", "layer", 3, F32, F32),
    (700, 72, "rms", "rms", 1, BF16, BF16), (1200, 16, "layer", "rms", 4, F16, F32), (600, 8, "rms", "layer", 300, BF16, BF16),
    (1024, 24, "rms", "rms", 1024, BF16, F32), (12, 2048, "rms", "layer", 4, F16, F16), (3, 4104, "layer", "rms", 3, BF16, BF16),
    (4, 8200, "rms", "layer", 2, BF16, F32), (2, 16384, "layer", "layer", 1, F32, F32), (2, 16383, "layer", "rms", 2, BF16, F32),
    (3, 16384, "layer", "rms", 0, F16, F16), (5, 4097, "rms", "rms", 1, F16, F32), (7, 96, "rms", None, 1, BF16, BF16),
    (7, 90, None, None, 7, F32, F32), (6, 3000, "layer", "layer", 3, BF16, BF16), (4, 3001, "rms", "rms", 1, F16, F16),
    (4, 5120, "layer", "layer", 4, F16, F32), (4, 7000, "rms", "rms", 2, BF16, BF16), (6, 7001, "layer", "layer", 1, BF16, F32),
    (2000, 2500, "layer", "layer", 4, BF16, BF16), (900, 4500, "rms", "layer", 1, F16, F32), (3, 12288, "rms", "rms", 1, BF16, BF16),
    (4, 9000, "layer", "layer", 2, F16, F32), (300, 12300, "rms", "rms", 1, BF16, BF16)]


def norm_inputs(case, seed=12):
    n, dim, post, pre, gates, dtype, stream = case
    g = gen(seed)
    r, b = normal(g, n, dim, dtype=stream, size=2.0), normal(g, n, dim, dtype=dtype)
    post, pre = norm_of(g, post, dim, dtype), norm_of(g, pre, dim, F32 if n % 2 else dtype)
    gate = normal(g, gates, dim, dtype=dtype) if gates else None
    return g, r, b, dict(post=post, pre=pre, gate=gate, residual_scale=0.9, block_scale=1.3)


def norm_bound(x, given, off):
    """Of norm(x) where x is off by ``off``: the row's sums are of dim terms in threads of at most 64 and 80 joined, so mean and deviation are
    off by at most 150 U of the row's size; x - mean, the products and sums add 8 U each."""
    y, hat, mean, rstd = C.norm(x, given)
    size = x.abs().amax(-1, keepdim=True) + mean.abs()
    w = 1.0 if given.weight is None else given.weight.cpu().double().abs()
    far = off.amax(-1, keepdim=True) if isinstance(off, torch.Tensor) else off
    relative = rstd * (150 * C.U * size + 3 * far)
    return w * (relative + hat.abs() * relative + 160 * C.U * hat.abs()) + 8 * C.U * y.abs()


@pytest.mark.parametrize("case", NORM, ids=str)
def test_residual_norm(case):
    n, dim, _, _, _, dtype, stream = case
    g, r, b, given = norm_inputs(case)
    got = ops.residual_norm(r, b, **given)
    ref_stream, ref_normed = C.residual_norm(r, b, given["post"], given["pre"], given["gate"], 0.9, 1.3)
    x = b.cpu().double()
    off = norm_bound(x, given["post"], 0.0) if given["post"] else torch.zeros_like(x)
    gate = C.gate_rows(given["gate"], n, dim).abs() if given["gate"] is not None else 1.0
    off = off * gate * 1.3 + 8 * C.U * (r.cpu().double().abs() + ref_stream.abs())
    assert got.stream.dtype == stream
    C.close(got.stream, ref_stream, off + C.rounded(ref_stream, stream), "stream")
    if given["pre"]:
        assert got.normed.dtype == dtype
        C.close(got.normed, ref_normed, norm_bound(ref_stream, given["pre"], off) + C.rounded(ref_normed, dtype), "normed")
    else:
        assert got.normed is None


def check_norm_grad(got, stream, block, stats, dh, ds, given, what=""):
    """Behind each term are some 30 roundings, and sums of at most 64 terms in a thread, of dim / 64 waves' and of n / 512 rows' at most."""
    ref = C.residual_norm_grad(stream, block, stats, dh, ds, given["post"], given["pre"], given["gate"], given["residual_scale"], given["block_scale"])
    for name, (value, size) in ref.items():
        t = getattr(got, name)
        if t is not None:
            C.close(t, value.reshape(t.shape), 200 * C.U * size.reshape(t.shape) + C.rounded(value.reshape(t.shape), t.dtype), f"{what} {name}")


@pytest.mark.parametrize("with_stream", [True, False], ids=["stream", "no_stream"])
@pytest.mark.parametrize("case", NORM, ids=str)
def test_residual_norm_grad(case, with_stream):
    n, dim, _, pre, _, dtype, stream = case
    if pre is None and not with_stream:
        pytest.skip("no gradient at all")
    g, r, b, given = norm_inputs(case)
    out = ops.residual_norm(r, b, stats=True, **given)
    dh = normal(g, n, dim, dtype=dtype) if pre else None
    ds = normal(g, n, dim, dtype=stream) if with_stream else None
    got = ops.residual_norm_grad(out.stream, b, out.stats, dh, ds, **given)
    check_norm_grad(got, out.stream, b, out.stats, dh, ds, given)
    again = ops.residual_norm_grad(out.stream, b, out.stats, dh, ds, **given)
    assert all(x is None and y is None or torch.equal(x, y) for x, y in zip(got, again)), "the same inputs give the same bits"


def test_residual_norm_without_block_and_without_rows():
    g = gen(13)
    r = normal(g, 3, 5, 96)
    pre = norm_of(g, "rms", 96, BF16)
    out = ops.residual_norm(r, pre=pre)
    assert out.stream is r and out.normed.dtype == BF16 and out.stats is None
    ref = C.norm(r.cpu().double(), pre)[0]
    C.close(out.normed, ref, norm_bound(r.cpu().double(), pre, 0.0) + C.rounded(ref, BF16))
    halved = ops.residual_norm(r, pre=pre, residual_scale=0.5)
    assert torch.equal(halved.stream, r * 0.5)
    bare = ops.residual_norm(r, pre=ops.Norm("layer"))
    ref = C.norm(r.cpu().double(), ops.Norm("layer"))[0]
    C.close(bare.normed, ref, norm_bound(r.cpu().double(), ops.Norm("layer"), 0.0) + C.rounded(ref, F32))
    empty = ops.residual_norm(r[:0], r[:0], stats=True, pre=norm_of(g, "layer", 96, F32), gate=normal(g, 96))
    assert empty.normed.shape == (0, 5, 96)
    given = dict(pre=norm_of(g, "layer", 96, F32), post=norm_of(g, "rms", 96, F32), gate=normal(g, 96))
    none = ops.residual_norm_grad(r[:0], r[:0], empty.stats, r[:0], r[:0], **given)
    assert all(not t.any() for t in (none.pre_weight, none.pre_bias, none.post_weight, none.gate)) and none.residual.shape == (0, 5, 96)


def test_residual_norm_strides():
    g = gen(14)
    wide_r, wide_b = normal(g, 6, 131), normal(g, 6, 140, dtype=BF16)
    r, b = wide_r[:, 3:83], wide_b[:, 1:81]
    given = dict(post=norm_of(g, "rms", 80, BF16), pre=ops.Norm("layer", normal(g, 160)[::2], normal(g, 81)[1:]), gate=normal(g, 160)[::2],
                 residual_scale=0.9, block_scale=1.3)
    got, same = (ops.residual_norm(*x, stats=True, **given) for x in ((r, b), (r.clone(), b.clone())))
    assert all(torch.allclose(x.float(), y.float(), rtol=0.01, atol=1e-5) for x, y in zip(got, same))
    ref = C.residual_norm(r, b, given["post"], given["pre"], given["gate"], 0.9, 1.3)[1]
    assert (got.normed.cpu().double() - ref).abs().max() <= 2.0 ** -8 * ref.abs().max()
    dh, ds = normal(g, 6, 90, dtype=BF16)[:, 5:85], torch.tensor(0.25, device="cuda").expand(6, 80)
    check_norm_grad(ops.residual_norm_grad(got.stream, b, got.stats, dh, ds, **given), got.stream, b, got.stats, dh, ds, given)


def test_residual_norm_autograd_and_differences():
    """Central differences of a float32 loss along a direction: the cubic term of steps of 2^-7 is below 2^-14 * 8 of the loss's size."""
    g = gen(15)
    n, dim = 6, 48
    inputs = dict(r=normal(g, n, dim), b=normal(g, n, dim), pw=1 + 0.2 * normal(g, dim), pb=normal(g, dim), w=1 + 0.2 * normal(g, dim), wb=normal(g, dim),
                  gate=normal(g, 2, dim))
    a, c = normal(g, n, dim), normal(g, n, dim)

    def loss(r, b, pw, pb, w, wb, gate):
        out = ops.residual_norm(r, b, post=ops.Norm("layer", pw, pb), pre=ops.Norm("layer", w, wb), gate=gate, residual_scale=0.8, block_scale=1.2)
        return (out.stream * a).double().sum() + (out.normed * c).double().sum()

    leaves = {k: v.clone().requires_grad_() for k, v in inputs.items()}
    grads = dict(zip(leaves, torch.autograd.grad(loss(**leaves), list(leaves.values()))))
    for name in inputs:
        v = normal(g, *inputs[name].shape)
        v = v / v.norm()
        h = 2.0 ** -7
        step = lambda s: loss(**{**inputs, name: inputs[name] + s * h * v})   # noqa: B023, E731
        along = ((step(1) - step(-1)) / (2 * h)).item()
        size = (a.abs().sum() + c.abs().sum()).item()
        assert abs(along - (grads[name].double() * v).sum().item()) <= size * (2.0 ** -11 + 20 * C.U / h), name
    # the stream alone: the norm before the next block has no part in its gradient
    alone = torch.autograd.grad(ops.residual_norm(leaves["r"], leaves["b"], pre=ops.Norm("rms", leaves["w"])).stream.sum(), [leaves["r"], leaves["b"]])
    assert all(torch.equal(x, torch.ones_like(x)) for x in alone)


# ---- as they are used ------------------------------------------------------------------------------------------
def test_together_on_another_stream_and_in_a_graph():
    """Lookup, join, log probabilities and their gradients in a row, on a stream of their own, and captured: every replay, with eager work in
    between, gives the eager bits."""
    g = gen(16)
    vocab, dim, n = 1003, 64, 96
    w, head = normal(g, vocab, dim, dtype=BF16), normal(g, dim, vocab, dtype=BF16, size=0.1)
    t, b, pre, gate = tokens_of(g, n, vocab), normal(g, n, dim, dtype=BF16), norm_of(g, "rms", dim, BF16), normal(g, 3, dim, dtype=BF16)
    target = torch.roll(t, -1)
    post = norm_of(g, "rms", dim, BF16)

    def step():
        x = ops.embedding(t, w, scale=8.0)
        out = ops.residual_norm(x, b, post=post, pre=pre, gate=gate, stats=True)
        logits = out.normed @ head
        r = ops.token_logprobs(logits, target, entropy=True, top=5)
        d = ops.token_logprobs_grad(logits, target, r.lse, torch.ones_like(r.lse) / n, entropy=r.entropy, grad_entropy=r.entropy)
        dh = d @ head.t().contiguous()
        back = ops.residual_norm_grad(out.stream, b, out.stats, dh, post=post, pre=pre, gate=gate)
        return [*r, d, back.residual, back.pre_weight, back.gate, ops.embedding_grad(t, back.residual, vocab, scale=8.0)]

    eager = [x.clone() for x in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(eager, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for _ in range(4):
        for x in captured:
            x.zero_()
        torch.cuda.synchronize()
        graph.replay()
        again = step()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(eager, captured)) and all(torch.equal(x, y) for x, y in zip(eager, again))


def test_refusals():
    w, t = torch.ones(5, 8, device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda")
    x = torch.zeros(3, 9, device="cuda")
    lse = torch.zeros(3, device="cuda")
    norm = ops.Norm("rms")
    bad = [lambda: ops.embedding(t.float(), w), lambda: ops.embedding(t, w.double()), lambda: ops.embedding(t, w.t()), lambda: ops.embedding(t, w[0]),
           lambda: ops.embedding(t, w, dtype=torch.float64), lambda: ops.embedding(t.cpu(), w), lambda: ops.embedding(t, w.cpu()),
           lambda: ops.embedding_grad(t, w, 5), lambda: ops.embedding_grad(t, w[:3], -1), lambda: ops.embedding_grad(t, w[:3], 5, into=w[:4]),
           lambda: ops.embedding_grad(t, w[:3], 5, into=w, dtype=F16), lambda: ops.embedding_grad(t, w[:3], 8, into=torch.ones(8, 8, device="cuda").t()),
           lambda: ops.token_logprobs(x, t[:2]), lambda: ops.token_logprobs(x, t, top=10), lambda: ops.token_logprobs(x, t, top=65),
           lambda: ops.token_logprobs(x, t, top=-1), lambda: ops.token_logprobs(x, t, scale=0.0), lambda: ops.token_logprobs(x, t, scale=math.nan),
           lambda: ops.token_logprobs(x, t, scale=-1.0), lambda: ops.token_logprobs(x[:, :0], t), lambda: ops.token_logprobs(x.double(), t),
           lambda: ops.token_logprobs(x.cpu(), t), lambda: ops.token_logprobs_grad(x, t, lse[:2], lse), lambda: ops.token_logprobs_grad(x, t, lse, lse[:1]),
           lambda: ops.token_logprobs_grad(x, t, lse, lse, entropy=lse), lambda: ops.token_logprobs_grad(x, t, lse, lse, into=x[:2]),
           lambda: ops.token_logprobs_grad(x, t, lse, grad_top=x), lambda: ops.token_logprobs_grad(x, t, lse, lse, first=-1),
           lambda: ops.logprob_parts(x, t, first=2 ** 31 - 5), lambda: ops.logprob_parts(lse, t, first=0),
           lambda: ops.join_logprobs([ops.logprob_parts(x, t, first=0)] * 65, t, 9), lambda: ops.join_logprobs([ops.logprob_parts(x, t, first=0)], t, 0),
           lambda: ops.residual_norm(x), lambda: ops.residual_norm(x, post=norm, pre=norm), lambda: ops.residual_norm(x, x[:2], pre=norm),
           lambda: ops.residual_norm(x, x.half(), pre=ops.Norm("max")), lambda: ops.residual_norm(x.half(), x, pre=norm),
           lambda: ops.residual_norm(x, x, pre=ops.Norm("rms", lse)), lambda: ops.residual_norm(x, x, pre=norm, gate=x[:2]),
           lambda: ops.residual_norm(x, x, pre=ops.Norm("rms", None, None, -1.0)), lambda: ops.residual_norm(x, x, pre=ops.Norm("rms", None, None, math.nan)),
           lambda: ops.residual_norm(torch.zeros(1, 16385, device="cuda"), pre=norm), lambda: ops.residual_norm(x[:, :0], x[:, :0], pre=norm),
           lambda: ops.residual_norm(x, x, pre=ops.Norm("layer", x[0], x[0].half())), lambda: ops.residual_norm_grad(x, x, x[:, :4], None, None, pre=norm),
           lambda: ops.residual_norm_grad(x, x, x[:, :3], x, pre=norm), lambda: ops.residual_norm_grad(x, None, x[:, :4], x, pre=norm, post=norm),
           lambda: ops.residual_norm_grad(x, x, x[:, :4], x.half(), pre=norm)]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"number {i} was not refused")
    torch.cuda.synchronize()
