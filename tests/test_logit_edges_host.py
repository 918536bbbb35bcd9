"""CPU-only checks of calls of the operators on logits that are refused before any device work."""
import ctypes

import pytest

torch = pytest.importorskip("torch")

from galvatron_dp import _lib, operators as ops   # noqa: E402
import test_logits_host as H   # noqa: E402


def test_parts_of_a_vocabulary_that_is_none_are_refused():
    lib = ops._ops()
    assert lib.gdp_distill_parts(ctypes.byref(H.part(whole_vocab=-1)), None) == _lib.GDP_E_BADARG
    assert lib.gdp_last_error().startswith(b"gdp_distill: whole_vocab")
    assert lib.gdp_distill_parts(ctypes.byref(H.part(n=0, whole_vocab=90)), None) == _lib.GDP_OK


def test_results_over_a_tensor_that_wants_a_gradient_are_refused():
    """Autograd would go on with the history of what it held."""
    x, t, s, v = torch.zeros(3, 70), torch.zeros(3, 4, dtype=torch.int64), torch.zeros(3, 9), torch.ones(3)
    leaf = torch.zeros(3, 70, requires_grad=True)
    for into in (leaf, leaf * 5, (leaf * 5)[:, :]):
        for call in (lambda: ops.adjust_logits(x, scale=2.0, into=into), lambda: ops.adjust_logits_grad(x, x, into=into), lambda: ops.distillation_grad(x, t, s, v, into=into),
                     lambda: ops.distillation_grad(into, t, s, v, into=into)):
            with pytest.raises(ValueError, match="detach"):
                call()
            with torch.no_grad(), pytest.raises(ValueError, match="HIP device"):
                call()
    for call in (lambda: ops.adjust_logits(x, into=leaf.detach()), lambda: ops.distillation_grad(x, t, s, v, into=(leaf * 5).detach())):
        with pytest.raises(ValueError, match="HIP device"):
            call()
