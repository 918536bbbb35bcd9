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
