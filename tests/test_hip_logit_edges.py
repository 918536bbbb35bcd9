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
