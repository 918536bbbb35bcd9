"""A model's ends in float16: the loss is scaled before its gradients are rounded, or refused."""
import pytest

torch = pytest.importorskip("torch")

import operator_cases as C   # noqa: E402
from galvatron_dp import model_ends   # noqa: E402
from test_hip_model_ends import plain   # noqa: E402

F16 = torch.float16


def test_float16_needs_a_scale_of_the_loss():
    ends = model_ends.ModelEnds(8, 30, dtype=F16, device="cpu")
    t = torch.zeros(3, dtype=torch.int64)
    with pytest.raises(ValueError, match="loss_scale"):
        ends.loss_and_grads(t, t, torch.zeros(3, 8, dtype=F16))
    for bad in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="loss_scale"):
            ends.loss_and_grads(t, t, torch.zeros(3, 8, dtype=F16), loss_scale=bad)


@pytest.mark.gpu
def test_gradients_in_float16_keep_the_softmax():
    """4096 targets and 40000 tokens: a share of 1 / 40000 of a mean over 4096 is 6e-9, below a tenth of float16's least step.  Scaled, the
    gradients of tokens that are never a target, which have nothing but such shares, are there to float16's precision."""
    ends = model_ends.ModelEnds(64, 40000, dtype=F16, seed=7)
    g = torch.Generator().manual_seed(8)
    tokens, targets = (torch.randint(0, 20000, (4, 1024), generator=g).cuda() for _ in range(2))
    targets[0, :9] = -100
    block = torch.randn(4, 1024, 64, generator=g).half().cuda()
    scale = 4096.0 * 16
    got = ends.loss_and_grads(tokens, targets, block, loss_scale=scale)
    loss, grads = plain(ends, tokens, targets, block)
    # rounded to float16 four times on the way (as in the test of the other types), 4096 terms to a float32 sum
    unit = 40 * C.HALF_UNIT[F16] + 4096 * C.U
    assert abs(got.loss.item() - loss.item()) <= unit * abs(loss.item())
    for name, ref in zip(("embedding", "norm", "head", "block"), grads):
        x = getattr(got, name).cpu().double() / scale
        assert (x - ref).abs().max() <= unit * ref.abs().max(), name
    never = torch.ones(40000, dtype=torch.bool)
    never[targets[targets >= 0].cpu()] = False
    head, ref = got.head.cpu().double()[never] / scale, grads[2][never]
    assert (head - ref).abs().max() <= unit * ref.abs().max()
    assert (head != 0).double().mean() > 0.99
    main = torch.zeros(40000, 64, device="cuda")
    again = ends.loss_and_grads(tokens, targets, block, into=main, loss_scale=scale)
    assert again.embedding is main and (main.cpu().double() / scale - grads[0]).abs().max() <= unit * grads[0].abs().max()


@pytest.mark.gpu
def test_scaled_loss_of_the_other_types_and_the_command():
    ends = model_ends.ModelEnds(32, 300, dtype=torch.float32)
    t = torch.arange(40, device="cuda").reshape(2, 20)
    block = torch.ones(2, 20, 32, device="cuda")
    one, many = ends.loss_and_grads(t, t, block), ends.loss_and_grads(t, t, block, loss_scale=64.0)
    assert torch.equal(one.loss, many.loss)
    for x, y in zip(one[2:], many[2:]):
        assert torch.equal(x * 64.0, y)          # (a power of two: the same digits)
    model_ends.main(["--hidden", "64", "--vocab", "500", "--seq", "32", "--precision", "fp16", "--backward"])


@pytest.mark.gpu
def test_another_default_type_of_the_program():
    ends = model_ends.ModelEnds(32, 300, dtype=torch.bfloat16)
    t, block = torch.arange(40, device="cuda").reshape(2, 20), torch.ones(2, 20, 32, device="cuda", dtype=torch.bfloat16)
    want = ends.loss_and_grads(t, t, block)
    torch.set_default_dtype(torch.bfloat16)
    try:
        got = ends.loss_and_grads(t, t, block)
    finally:
        torch.set_default_dtype(torch.float32)
    # (the shares of the mean are divided in the default type: one rounding of it more in each gradient)
    for x, y in zip(got, want):
        assert (x.double() - y.double()).abs().max() <= 4 * C.HALF_UNIT[torch.bfloat16] * y.double().abs().max()
