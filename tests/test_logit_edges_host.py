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
