"""Calls of the operators at their edges, against plain forms in 64 bits written here: rows far from zero, lists that are out of order,
memory that is written in place, single and missing rows, outputs that a program changes."""
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


# ---- lists of the parts, in any order and more than once ----------------------------------------------------
@pytest.mark.parametrize("parts,top", [(64, 64), (8, 20), (3, 7), (2, 1)])
@pytest.mark.parametrize("order", ["reversed", "shuffled", "repeated"])
def test_join_of_lists_that_parts_do_not_leave(parts, top, order):
    """What a caller hands over stays within the kernel's memory and every place is written: the largest logits of all lists, equal ones by
    number; a token that is listed twice is there twice."""
    g = gen(31)
    n, width = 3, 70
    x = normal(g, n, parts * width, size=2.0)
    t = torch.randint(0, parts * width, (n,), generator=g).cuda()
    made = [ops.logprob_parts(x[:, width * i:width * (i + 1)], t, first=width * i, top=top) for i in range(parts)]
    if order == "repeated":
        made = [made[0]] * parts
    else:
        at = torch.arange(top - 1, -1, -1) if order == "reversed" else torch.randperm(top, generator=g)
        made = [p._replace(top_logits=p.top_logits[:, at.cuda()], top_tokens=p.top_tokens[:, at.cuda()]) for p in made]
    got = ops.join_logprobs(made, t, parts * width)
    logits, tokens = (torch.cat([getattr(p, f).cpu() for p in made], 1) for f in ("top_logits", "top_tokens"))
    for row in range(n):
        best = sorted(zip((-logits[row]).tolist(), tokens[row].tolist()))[:top]
        assert got.top_tokens[row].tolist() == [token for _, token in best]
        ref = torch.tensor([-v for v, _ in best], dtype=torch.float64) - got.lse[row].double().cpu()
        # lse is rounded, and so are the logit's distance and the logarithm that top_logp is made of
        C.close(got.top_logp[row], ref, 8 * C.U * (2 * logits[row].double().abs().max() + 10))

# ---- gradients of rows far from zero ------------------------------------------------------------------------
def far_rows(g, dtype, vocab):
    """Rows of finite logits at any level, of masks alone, and one of which nothing is left."""
    low = torch.finfo(dtype).min
    step = {F32: 1.0, F16: 32.0, BF16: 512.0}[dtype]        # what the type can tell apart there
    at = {F32: -1.2e5, F16: -6.0e4, BF16: -1.2e5}[dtype]
    x = torch.randn(7, vocab, generator=g)
    x[1] = at + step * torch.randint(0, 4, (vocab,), generator=g)
    x[2] = low
    x[3] = at if dtype == F16 else -1e9
    x[4] = -at + step * torch.randint(0, 4, (vocab,), generator=g)
    x[5] = low
    x[5, vocab // 2:] = torch.randn(vocab - vocab // 2, generator=g)
    x[6] = -math.inf
    return x.to(dtype).cuda()


def softmax_grads(x, t, scale, a, b, c, d, top, columns=slice(None)):
    """(gradient of a logp + b entropy + c top_logp + d lse, a bound on its float32 error), from the definition: the shift by the largest
    logit cancels exactly.  A probability's exponent has three roundings of its own size, the logarithm of the sum those of its terms."""
    x = x.detach().cpu().double()
    n, vocab = x.shape
    z = (x - x.amax(1, keepdim=True).clamp(min=-1e300)) * scale
    q = z - torch.logsumexp(z, 1, keepdim=True).clamp(min=-1e300)
    p = q.exp()
    alive = torch.isfinite(x).any(1)
    a, b, c, d = (v.cpu().double() for v in (a, b, c, d))
    rows = torch.arange(n)
    entropy = -torch.where(p > 0, p * q, 0.0).sum(1)
    hit, of_hit = torch.zeros(n, vocab, dtype=torch.float64), torch.zeros(n, vocab, dtype=torch.float64)
    held = (t.cpu() >= 0) & (t.cpu() < vocab)
    a = a * held
    hit[rows[held], t.cpu()[held]] += a[held]
    of_hit[rows[held], t.cpu()[held]] += a[held].abs()
    for i in range(c.shape[1]):
        hit[rows, top[:, i].cpu()] += c[:, i]
        of_hit[rows, top[:, i].cpu()] += c[:, i].abs()
    weight, of_weight = (a + c.sum(1) - d)[:, None], (a.abs() + c.abs().sum(1) + d.abs())[:, None]
    away = torch.where(p > 0, q + entropy[:, None], 0.0)
    grad = hit - p * (weight + b[:, None] * away)
    size = of_hit + p * (of_weight + b.abs()[:, None] * (torch.where(p > 0, q.abs(), 0.0) + entropy[:, None]))
    ln_v = math.log(max(vocab, 2))
    relative = C.U * (80 + 8 * ln_v + vocab / 256 + c.shape[1] + 8 * torch.where(p > 0, q.abs(), 0.0))
    off = size * relative + p * b.abs()[:, None] * C.logprob_bound(torch.zeros(1, vocab), 1.0)[2]
    grad, off = (torch.where(alive[:, None], v, 0.0)[:, columns] * scale for v in (grad, off))
    return grad, off


@pytest.mark.parametrize("scale", [1.0, 1.25, 0.5], ids=str)
@pytest.mark.parametrize("vocab", [9, 2500, 70001])
@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_gradients_do_not_go_by_the_level_of_a_row(dtype, vocab, scale):
    """A row's logits may lie anywhere: its gradient is the softmax's, as its log probabilities are, and zeros where nothing is left."""
    g = gen(32)
    x = far_rows(g, dtype, vocab).requires_grad_()
    n, k = x.shape[0], 3
    t = torch.randint(0, vocab, (n,), generator=g).cuda()
    t[0] = -100
    a, b, c, d = normal(g, n), normal(g, n), normal(g, n, k), normal(g, n)
    r = ops.token_logprobs(x, t, scale=scale, entropy=True, top=k)
    used = torch.isfinite(r.lse)                      # (float32's lowest value times 1.25 has no float32)
    loss = (r.logp[used] * a[used]).sum() + (r.entropy * b).sum() + (r.top_logp[used] * c[used]).sum() + (r.lse[used] * d[used]).sum()
    got, = torch.autograd.grad(loss, x)
    u = used.float()
    ref, off = softmax_grads(x, t, scale, a * u, b, c * u[:, None], d * u, r.top_tokens)
    C.close(got, ref, off + C.rounded(ref, dtype))
    # by hand, in the logits' place, and of a vocabulary in shards
    stats = torch.empty(n, 2, device="cuda")
    with torch.no_grad():
        r = ops.token_logprobs(x, t, scale=scale, entropy=True, top=k, row_stats=stats)
        given = dict(scale=scale, entropy=r.entropy, grad_entropy=b, top_tokens=r.top_tokens, grad_top=c, grad_lse=d)
        ref, off = softmax_grads(x, t, scale, a, b, c, d, r.top_tokens)
        place = x.detach().clone()
        C.close(ops.token_logprobs_grad(place, t, None, a, row_stats=stats, into=place, **given), ref, off + C.rounded(ref, dtype))
        cut = vocab // 3
        shards = [x.detach()[:, :cut], x.detach()[:, cut:]]
        of_join = torch.empty(n, 2, device="cuda")
        parts = [ops.logprob_parts(s, t, first=f, scale=scale, top=k) for s, f in zip(shards, (0, cut))]
        j = ops.join_logprobs(parts, t, vocab, scale=scale, entropy=True, row_stats=of_join)
        assert torch.equal(j.top_tokens, r.top_tokens)
        given.update(entropy=j.entropy, vocab=vocab)
        for s, f in zip(shards, (0, cut)):
            part, of_part = softmax_grads(x, t, scale, a, b, c, d, r.top_tokens, slice(f, f + s.shape[1]))
            C.close(ops.token_logprobs_grad(s, t, None, a, row_stats=of_join, first=f, **given), part, of_part + C.rounded(part, dtype))


def test_gradient_at_a_low_temperature():
    g = gen(33)
    x = (normal(g, 4, 300) * 1e-4 - 20.0).requires_grad_()
    t = torch.randint(0, 300, (4,), generator=g).cuda()
    one, none = torch.ones(4, device="cuda"), torch.zeros(4, device="cuda")
    got, = torch.autograd.grad(ops.token_logprobs(x, t, scale=1e4).logp.sum(), x)
    ref, off = softmax_grads(x, t, 1e4, one, none, torch.zeros(4, 0), none, None)
    C.close(got, ref, off + C.rounded(ref, F32))


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_gradient_from_lse_alone(dtype):
    """float32 holds lse to one part in 2^24: by hand from lse alone a row's probabilities are those of the lse that is given, and a row below
    -2^24, where it says nothing of the sum any more, has zeros."""
    g = gen(34)
    x = far_rows(g, dtype, 600)
    t = torch.randint(0, 600, (7,), generator=g).cuda()
    r = ops.token_logprobs(x, t)
    got = ops.token_logprobs_grad(x, t, r.lse, torch.ones(7, device="cuda")).cpu().double()
    f = x.cpu().double()
    p = (f - r.lse.cpu().double()[:, None]).exp()
    dead = r.lse.cpu() < -2.0 ** 24
    assert dead.tolist() == [False, False, dtype != F16, dtype != F16, False, False, True]
    ref = torch.where(dead[:, None], 0.0, -p)
    ref[torch.arange(7)[~dead], t.cpu()[~dead]] += 1.0
    off = C.U * (24 + 6 * (f - r.lse.cpu().double()[:, None]).abs().clamp(max=200.0)) * (p.clamp(max=2.0) + 1.0)
    C.close(got, ref, off + C.rounded(ref, dtype))


def test_row_stats_are_the_largest_logit_and_the_logarithm_of_the_sum():
    g = gen(35)
    x = normal(g, 5, 40000, size=2.0)
    x[4] = -math.inf
    t = torch.zeros(5, dtype=torch.int64, device="cuda")
    for rows, cut in ((slice(0, 5), 40000), (slice(0, 5), 100)):      # a row in slices, and whole
        stats = torch.empty(5, 2, device="cuda")
        ops.token_logprobs(x[rows, :cut], t, scale=0.7, row_stats=stats)
        f = x[rows, :cut].cpu().double()
        assert torch.equal(stats[:, 0].cpu().double(), f.amax(1))
        ref = torch.logsumexp((f - f.amax(1, keepdim=True).clamp(min=-1e300)) * 0.7, 1)
        C.close(stats[:, 1], ref, C.logprob_bound(torch.zeros(1, cut), 1.0)[0][0].item())
    x = x[:3]
    for bad in (torch.empty(3, 2), torch.empty(2, 2, device="cuda"), torch.empty(3, 2, device="cuda", dtype=F16), torch.empty(2, 3, device="cuda").t()):
        with pytest.raises(ValueError, match="row_stats"):
            ops.token_logprobs(x, t[:3], row_stats=bad)
        with pytest.raises(ValueError, match="row_stats"):
            ops.token_logprobs_grad(x, t[:3], None, t[:3].float(), row_stats=bad)
    with pytest.raises(ValueError, match="row_stats"):
        ops.token_logprobs_grad(x, t[:3], None, t[:3].float())


# ---- what is written in place ---------------------------------------------------------------------------------
def test_autograd_sees_what_is_written_in_place():
    """Of logits that a graph holds, and of buffers: overwritten behind autograd's back they would give a wrong gradient without an error."""
    g = gen(36)
    w, t = normal(g, 3, 9).requires_grad_(), torch.tensor([1, 2, 3], device="cuda")
    one = torch.ones(3, device="cuda")
    logits = w * 2.0
    r = ops.token_logprobs(logits, t)
    ops.token_logprobs_grad(logits.detach(), t, r.lse.detach(), one, into=logits.detach())
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        r.logp.sum().backward()
    stats = torch.empty(3, 2, device="cuda")
    r = ops.token_logprobs(w, t, row_stats=stats)
    ops.token_logprobs(w.detach() + 1.0, t, row_stats=stats)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        r.logp.sum().backward()
    main = torch.zeros(9, 4, device="cuda")
    squares = (main * w.new_ones(1).requires_grad_()).square().sum() + (main * main.new_ones(9, 4).requires_grad_()).sum()
    ops.embedding_grad(t, torch.ones(3, 4, device="cuda"), 9, into=main)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        squares.backward()
    parts = [ops.logprob_parts(w.detach()[:, a:a + 3], t, first=a) for a in (0, 3, 6)]
    before = stats._version
    ops.join_logprobs(parts, t, 9, row_stats=stats)
    assert stats._version > before
    # nothing to write: nothing has changed.  And in inference mode there are no versions
    before = main._version
    ops.embedding_grad(t[:0], torch.ones(0, 4, device="cuda"), 9, into=main)
    assert main._version == before
    with torch.inference_mode():
        x = torch.randn(3, 9, device="cuda")
        assert ops.token_logprobs_grad(x, t, ops.token_logprobs(x, t).lse, one, into=x) is x
        ops.embedding_grad(t, torch.ones(3, 4, device="cuda"), 9, into=torch.zeros(9, 4, device="cuda"))
    assert ops.token_logprobs_grad(x, t, ops.token_logprobs(x, t).lse, one, into=x) is x


# ---- outputs are a program's own ------------------------------------------------------------------------------
def test_outputs_can_be_changed_in_place():
    """Each is a tensor of its own: changing one is allowed, does not touch the others and is no change of them for autograd."""
    g = gen(37)
    x, t = normal(g, 4, 50), torch.tensor([1, -100, 3, 4], device="cuda")
    weights = torch.tensor([1.0, 2.0, 3.0, 4.0], device="cuda").requires_grad_()
    leaf = x.clone().requires_grad_()
    parts = [ops.logprob_parts(x, t, first=0)]
    for r in (ops.token_logprobs(x, t, entropy=True), ops.token_logprobs(leaf, t, entropy=True), ops.join_logprobs(parts, t, 50, entropy=True)):
        lse, entropy = r.lse.detach().clone(), r.entropy.detach().clone()
        squares = r.lse.square().sum() + (r.entropy * weights).sum()
        r.logp.masked_fill_(t < 0, 7.0)
        r.logp.mul_(weights)
        assert r.logp[1] == 14.0 and torch.equal(r.lse, lse) and torch.equal(r.entropy, entropy)
        (squares + r.logp.sum()).backward()
    # the gradient knows of the change: the place that was filled has none
    ref = x.cpu().double()
    p = torch.softmax(ref, 1)
    q, entropy = torch.log_softmax(ref, 1), -(p * torch.log_softmax(ref, 1)).sum(1, keepdim=True)
    w = weights.detach().cpu().double()[:, None]
    hit = torch.zeros(4, 50, dtype=torch.float64)
    hit[[0, 2, 3], [1, 3, 4]] = 1.0
    held = hit.sum(1, keepdim=True)
    want = w * (hit - held * p) - w * p * (q + entropy) + 2 * torch.logsumexp(ref, 1, keepdim=True) * p
    size = w * (hit + p) + w * p * (q.abs() + entropy) + 2 * torch.logsumexp(ref, 1, keepdim=True) * p
    C.close(leaf.grad, want, C.U * 200 * size)
    with torch.no_grad():
        r = ops.token_logprobs(leaf, t, entropy=True)
        r.entropy.zero_()
    (r.logp * weights).sum().backward()


# ---- single rows, and none --------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_gradient_in_the_place_of_one_padded_row(dtype):
    g = gen(38)
    for shape, cut in (((4, 1008), 1), ((2, 3, 1008), 1), ((5, 40), 1)):
        padded = normal(g, *shape, dtype=dtype, size=2.0)
        rest = padded.clone()
        x = padded[:cut, ..., :37] if len(shape) == 2 else padded[:cut, :1, :37]
        t = torch.full(x.shape[:-1], 5, device="cuda")
        r = ops.token_logprobs(x, t)
        one = torch.ones(x.shape[:-1], device="cuda")
        want = ops.token_logprobs_grad(x, t, r.lse, one)
        assert ops.token_logprobs_grad(x, t, r.lse, one, into=x) is x
        assert torch.equal(x, want)
        rest[(slice(0, 1),) * (len(shape) - 1) + (slice(0, 37),)] = want
        assert torch.equal(padded, rest), "what lies beside the row stays"


# ---- what a program leaves out or mixes up is a ValueError that names it ----------------------------------------
def test_norm_gradient_without_stats_is_refused():
    x = torch.zeros(3, 8, device="cuda")
    with pytest.raises(ValueError, match="stats"):
        ops.residual_norm_grad(x, x, None, x, pre=ops.Norm("rms"))


def test_norm_weights_of_other_types_are_refused():
    x, w = torch.zeros(3, 8, device="cuda"), torch.ones(8, device="cuda", dtype=torch.float64)
    for t in (x, x.half()):
        for block in (None, t):
            with pytest.raises(ValueError, match="weight"):
                ops.residual_norm(t, block, pre=ops.Norm("rms", w))


def test_parts_that_do_not_belong_together_are_refused():
    x, t = torch.zeros(3, 8, device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda")
    one, more, fewer = ops.logprob_parts(x, t, first=0, top=1), ops.logprob_parts(x, t, first=8, top=2), ops.logprob_parts(x[:2], t[:2], first=8, top=1)
    for bad in ([], [one, more], [one, fewer]):
        with pytest.raises(ValueError, match="parts"):
            ops.join_logprobs(bad, t, 16)


@pytest.mark.parametrize("dtype", TYPES, ids=ids)
def test_no_rows_with_a_gate_for_each(dtype):
    """An empty batch has no gates either: nothing to do, and gradients of zeros for what is there."""
    g = gen(39)
    x, w, gate = normal(g, 0, 5, 24, dtype=dtype), normal(g, 24, dtype=dtype), normal(g, 0, 24, dtype=dtype)
    post, pre = ops.Norm("layer", w, w), ops.Norm("rms", w)
    out = ops.residual_norm(x, x, post=post, pre=pre, gate=gate, stats=True)
    assert out.stream.shape == out.normed.shape == (0, 5, 24)
    got = ops.residual_norm_grad(out.stream, x, out.stats, x, x, post=post, pre=pre, gate=gate)
    assert got.gate.shape == (0, 24) and got.block.shape == (0, 5, 24) and not got.pre_weight.any() and not got.post_bias.any()
    leaf = gate.clone().requires_grad_()
    ops.residual_norm(x, x, pre=pre, gate=leaf).normed.sum().backward()
    assert leaf.grad.shape == (0, 24)
    with pytest.raises(ValueError, match="gate"):
        ops.residual_norm(normal(g, 2, 24, dtype=dtype), normal(g, 2, 24, dtype=dtype), pre=pre, gate=gate)


def test_norm_statistics_are_there_where_they_are_asked_for():
    """With gradients as without."""
    x = normal(gen(40), 3, 8)
    for t in (x, x.clone().requires_grad_()):
        assert ops.residual_norm(t, pre=ops.Norm("rms")).stats is None
        assert ops.residual_norm(t, t, pre=ops.Norm("rms"), stats=True).stats.shape == (3, 4)


# ---- from several threads ------------------------------------------------------------------------------------------
def test_calls_of_two_threads():
    """Each thread has its own stream, workspaces and errors."""
    import threading
    g = gen(41)
    x, t, d = normal(g, 20, 70001, dtype=BF16, size=2.0), torch.randint(0, 70001, (20,), generator=g).cuda(), normal(g, 20, 64)
    torch.cuda.synchronize()

    def step():
        r = ops.token_logprobs(x, t, entropy=True, top=20)
        return [*r, ops.token_logprobs_grad(x, t, r.lse, r.logp), ops.embedding_grad(t, d, 70001)]

    want, got, refused = step(), {}, {}

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            try:
                for _ in range(20):
                    got[i] = step()
                    try:
                        ops.token_logprobs(x, t, top=65) if i else ops.token_logprobs(x, t, scale=0.0)
                    except ValueError as e:
                        refused[i] = str(e)
            finally:
                torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for one in threads:
        one.start()
    for one in threads:
        one.join()
    assert all(torch.equal(a, b) for i in range(2) for a, b in zip(got[i], want))
    assert "scale" in refused[0] and "top" in refused[1]
