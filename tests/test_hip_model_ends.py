"""The operators run together as a model's ends, against float64 autograd on the CPU, and the profile entries they are measured for."""
import json

import pytest

torch = pytest.importorskip("torch")

import operator_cases as C   # noqa: E402
from galvatron_dp import model_ends, operators as ops, profile_configs   # noqa: E402

pytestmark = pytest.mark.gpu


def plain(ends, tokens, targets, block):
    """(loss, gradients of table, norm weight, head, block), float64"""
    table, head, weight, b = (t.detach().cpu().double().requires_grad_() for t in (ends.table, ends.head, ends.norm.weight, block))
    stream = table[tokens.cpu()] * ends.scale + b
    given = ends.norm._replace(weight=None, bias=None)
    x = C.norm(stream, given)[0] * weight
    if ends.norm.bias is not None:
        x = x + ends.norm.bias.cpu().double()
    logp = torch.log_softmax(x @ head.t(), -1)
    t = targets.cpu()
    held = (t >= 0) & (t < ends.vocab)
    loss = -(logp.gather(-1, torch.where(held, t, 0)[..., None])[..., 0] * held).sum() / held.sum()
    return loss.detach(), torch.autograd.grad(loss, (table, weight, head, b))


@pytest.mark.parametrize("norm", ["rms", "layer"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_loss_and_grads(dtype, norm):
    ends = model_ends.ModelEnds(96, 1000, dtype=dtype, norm=norm, scale=2.0, seed=3)
    g = torch.Generator().manual_seed(4)
    tokens, targets = torch.randint(0, 1000, (3, 50), generator=g).cuda(), torch.randint(0, 1000, (3, 50), generator=g).cuda()
    targets[0, :7] = -100
    block = torch.randn(3, 50, 96, generator=g).to(dtype).cuda()
    main = torch.zeros(1000, 96, device="cuda")
    got = ends.loss_and_grads(tokens, targets, block, into=main)
    loss, grads = plain(ends, tokens, targets, block)
    # what lies between the ends is rounded to the type four times over (stream, normed, logits, their gradient), and the head's products are sums
    # of 96 or 1000 terms: relative to the largest gradient 40 half units of the type, and of float32 sums 1000
    unit = 40 * C.HALF_UNIT[dtype] + 1000 * C.U
    assert abs(got.loss.item() - loss.item()) <= unit * abs(loss.item())
    for x, ref in zip((got.embedding, got.norm, got.head, got.block), grads):
        assert (x.cpu().double() - ref).abs().max() <= unit * ref.abs().max()
    assert got.embedding is main


def test_shards_join_to_the_whole():
    whole = model_ends.ModelEnds(64, 900, dtype=torch.float32, seed=5)
    g = torch.Generator().manual_seed(6)
    tokens, targets = torch.randint(0, 900, (2, 31), generator=g).cuda(), torch.randint(0, 900, (2, 31), generator=g).cuda()
    block = torch.randn(2, 31, 64, generator=g).cuda()
    shards = [model_ends.ModelEnds(64, 900, dtype=torch.float32, shards=3, shard=i) for i in range(3)]
    for i, s in enumerate(shards):
        s.table, s.head, s.norm = whole.table[300 * i:300 * (i + 1)], whole.head[300 * i:300 * (i + 1)], whole.norm
    stream = sum(s.embed(tokens) for s in shards)
    assert torch.equal(stream, whole.embed(tokens))
    parts = [ops.logprob_parts(s.logits(stream, block)[1].reshape(62, 300), targets.reshape(62), first=s.first, top=4) for s in shards]
    got = ops.join_logprobs(parts, targets.reshape(62), 900)
    want = whole.forward(tokens, targets, block, top=4)
    assert torch.allclose(got.logp, want.logp.reshape(62), atol=2e-5) and torch.equal(got.top_tokens, want.top_tokens.reshape(62, 4))
    assert isinstance(shards[1].forward(tokens, targets, block), ops.LogprobParts)
    with pytest.raises(ValueError):
        shards[0].loss_and_grads(tokens, targets, block)
    with pytest.raises(ValueError):
        model_ends.ModelEnds(64, 901, shards=3)


def test_profile_entries_are_what_the_search_reads(tmp_path):
    path = tmp_path / "computation_profiling_bf16_small.json"
    layers = {"layertype_0_bsz%d_seq64" % b: 1.5 for b in range(1, 9)}
    path.write_text(json.dumps(layers))
    times = model_ends.main(["--hidden", "128", "--vocab", "2000", "--seq", "64", "--bsz"] + [str(b) for b in range(1, 9)] + ["--backward", "--profile", str(path)])
    config = profile_configs.read_json_config(str(path))
    assert {k: v for k, v in config.items() if k in layers} == layers
    assert all(config["layertype_other_bsz%d_seq64" % b] == times[b, 64] > 0 for b in range(1, 9))
    _, other = profile_configs.fit_layer_times(config, "batch", 1, [64])
    assert other[0].shape == (2,)
