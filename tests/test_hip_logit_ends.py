"""The operators on logits run together with a model's ends: a student that learns from a teacher's most likely tokens, against float64 autograd
on the CPU, a decoding step under a grammar with penalties, shards of the vocabulary, and the command that measures the ends."""
import math

import pytest

torch = pytest.importorskip("torch")

import logit_cases as C   # noqa: E402
import operator_cases as O   # noqa: E402
from galvatron_dp import model_ends, operators as ops, profile_configs   # noqa: E402

pytestmark = pytest.mark.gpu


def inputs(vocab, hidden, dtype, seed, *shape):
    g = torch.Generator().manual_seed(seed)
    tokens, targets = torch.randint(0, vocab, shape, generator=g).cuda(), torch.randint(0, vocab, shape, generator=g).cuda()
    return tokens, targets, torch.randn(*shape, hidden, generator=g).to(dtype).cuda()


def plain_logits(ends, tokens, block):
    table, head, weight, b = (t.detach().cpu().double().requires_grad_() for t in (ends.table, ends.head, ends.norm.weight, block))
    x = O.norm(table[tokens.cpu()] * ends.scale + b, ends.norm._replace(weight=None, bias=None))[0] * weight
    return x @ head.t(), (table, weight, head, b)


@pytest.mark.parametrize("weight", [1.0, 0.75])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_a_student_learns_from_a_teacher(dtype, weight):
    student = model_ends.ModelEnds(96, 1000, dtype=dtype, scale=2.0, seed=3)
    master = model_ends.ModelEnds(64, 1000, dtype=dtype, seed=5)
    tokens, targets, block = inputs(1000, 96, dtype, 4, 2, 20)
    targets[0, :5] = -100
    _, _, other = inputs(1000, 64, dtype, 6, 2, 20)
    taught = master.forward(tokens, targets, other, top=20)
    teacher = model_ends.Teacher(taught.top_tokens, taught.top_logp, beta=0.25, weight=weight)
    r = student.forward(tokens, targets, block, teacher=teacher)
    got = student.loss_and_grads(tokens, targets, block, teacher=teacher)
    z, leaves = plain_logits(student, tokens, block)
    flat, listed = z.reshape(40, 1000), C.listed_of(taught.top_tokens.reshape(40, 20), taught.top_logp.reshape(40, 20), 1000)
    t, loss, held = targets.cpu().reshape(40), 0.0, int((targets >= 0).sum())
    for i in range(40):
        if t[i] >= 0:
            each = C.distill_row(flat[i], listed[i], 0.25, True)[0]
            loss = loss + weight * each - (1 - weight) * torch.log_softmax(flat[i], 0)[t[i]]
    loss = loss / held
    grads = torch.autograd.grad(loss, leaves)
    # what lies between the ends is rounded to the type four times over (stream, normed, logits, their gradient), and the head's products are sums
    # of 96 or 1000 terms: relative to the largest gradient 40 half units of the type, and of float32 sums 1000
    unit = 40 * O.HALF_UNIT[dtype] + 1000 * O.U
    assert abs(got.loss.item() - loss.item()) <= unit * abs(loss.item())
    assert got.entropy is None and r.loss.shape == (2, 20)
    for x, ref in zip((got.embedding, got.norm, got.head, got.block), grads):
        assert (x.cpu().double() - ref).abs().max() <= unit * ref.abs().max()
    with pytest.raises(ValueError, match="teacher"):
        student.forward(tokens, targets, block, teacher=teacher, top=3)


def test_a_student_in_shards():
    whole = model_ends.ModelEnds(64, 900, dtype=torch.float32, seed=5)
    tokens, targets, block = inputs(900, 64, torch.float32, 6, 2, 31)
    shards = [model_ends.ModelEnds(64, 900, dtype=torch.float32, shards=3, shard=i) for i in range(3)]
    for i, s in enumerate(shards):
        s.table, s.head, s.norm = whole.table[300 * i:300 * (i + 1)], whole.head[300 * i:300 * (i + 1)], whole.norm
    listed = torch.stack([torch.randperm(900, generator=torch.Generator().manual_seed(i))[:7] for i in range(62)]).reshape(2, 31, 7).cuda()
    logp = torch.log_softmax(torch.arange(7.0).cuda().expand(2, 31, 7), -1) - 0.25
    teacher = model_ends.Teacher(listed, logp)
    want = whole.forward(tokens, targets, block, teacher=teacher)
    stream = sum(s.embed(tokens) for s in shards)
    parts = [ops.distillation_parts(s.logits(stream, block)[1].reshape(62, 300), listed.reshape(62, 7), logp.reshape(62, 7), first=s.first,
                                    targets=targets.reshape(62)) for s in shards]
    got = ops.join_distillation(parts, listed.reshape(62, 7), logp.reshape(62, 7), 900, targets=targets.reshape(62))
    # (the shards' heads are products of other sizes: sums of 64 terms in another order)
    assert torch.allclose(got.loss, want.loss.reshape(62), atol=2e-5) and torch.allclose(got.logp, want.logp.reshape(62), atol=2e-5)
    assert isinstance(shards[1].forward(tokens, targets, block, teacher=teacher), ops.DistillationParts)


def test_a_decoding_step_under_a_grammar():
    """Penalties for what a request has had, a mask that leaves it some tokens, and the log probabilities of those."""
    ends = model_ends.ModelEnds(96, 1000, dtype=torch.bfloat16, seed=7)
    tokens, targets, block = inputs(1000, 96, torch.bfloat16, 8, 6)
    g = torch.Generator().manual_seed(9)
    ok = torch.rand(6, 1000, generator=g) < 0.02
    ok[0], ok[0, 17] = False, True
    history = torch.randint(0, 1000, (6, 40), generator=g).cuda()
    adjust = dict(history=history, repetition=1.2, frequency=0.5, allowed=C.words_of(ok).cuda(), scale=0.8)
    plain = ends.logits(ends.embed(tokens), block)[1]
    r = ends.forward(tokens, targets, block, top=5, adjust=adjust)
    want = ops.token_logprobs(ops.adjust_logits(plain, **adjust), targets, top=5)
    assert all(torch.equal(a, b) for a, b in zip(r, want) if a is not None)
    assert r.top_tokens[0, 0].item() == 17 and r.top_logp[0].tolist() == [0.0] + [-math.inf] * 4
    picked = r.top_tokens.cpu()
    assert all(ok[i, picked[i, k]] for i in range(6) for k in range(5) if r.top_logp[i, k] > -math.inf)


def test_the_command_measures_a_students_ends(tmp_path):
    path = tmp_path / "computation_profiling_bf16_small.json"
    given = ["--hidden", "128", "--vocab", "2000", "--seq", "64", "--bsz", "1", "2", "--teacher", "20"]
    times = model_ends.main(given + ["--backward", "--profile", str(path)])
    config = profile_configs.read_json_config(str(path))
    assert all(config["layertype_other_bsz%d_seq64" % b] == times[b, 64] > 0 for b in (1, 2))
    assert model_ends.main(given + ["--shards", "4"]).keys() == times.keys()
    with pytest.raises(SystemExit):
        model_ends.main(given[:-1] + ["300"])
