"""CPU-only checks of the boundary of the operators on logits: records have the header's layout, calls are refused on the host before any device
work (no kernel is launched here), workspaces, and what is compiled."""
import ctypes
import os
import re
import shutil
import subprocess

import pytest

torch = pytest.importorskip("torch")

from galvatron_dp import _lib, operators as ops   # noqa: E402
import test_operators_host as H   # noqa: E402

P = H.P
RECORDS = (ops.gdp_distill, ops.gdp_distill_part, ops.gdp_distill_joint, ops.gdp_distill_grad, ops.gdp_adjust_history, ops.gdp_adjust,
           ops.gdp_adjust_grad)


def test_limits_are_the_headers():
    text = open(H.HEADER).read()
    assert int(re.search(r"GDP_MAX_LISTED (\d+)", text)[1]) == ops.MAX_LISTED
    assert int(re.search(r"GDP_MAX_BIASES (\d+)", text)[1]) == ops.MAX_BIASES


def test_records_have_the_headers_layout(tmp_path):
    if shutil.which("gcc") is None:
        pytest.skip("no gcc")
    lines = ['#include "%s"' % H.HEADER, "#include <stdio.h>", "int main(void) {"]
    for r in RECORDS:
        lines += ['printf("%%zu\\n", sizeof(%s));' % r.__name__]
        lines += ['printf("%%zu\\n", offsetof(%s, %s));' % (r.__name__, f[0]) for f in r._fields_]
    (tmp_path / "a.c").write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", str(tmp_path / "a.c"), "-o", str(tmp_path / "a")], check=True)
    got = [int(v) for v in subprocess.run([str(tmp_path / "a")], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [v for r in RECORDS for v in [ctypes.sizeof(r)] + [getattr(r, f[0]).offset for f in r._fields_]]


def distill(**over):
    given = dict(n=4, vocab=100, logits=P, logits_stride=100, logits_type=2, list_type=1, target_type=1, listed=3, tokens=P, teacher=P, targets=P,
                 scale=1.0, beta=0.5, rest=1, loss=P, lse=P, logp=P, stats=P, workspace=P, workspace_bytes=1 << 30)
    return ops.gdp_distill(**{**given, **over})


def part(**over):
    given = dict(n=4, vocab=100, first=0, logits=P, logits_stride=100, logits_type=2, list_type=1, target_type=1, listed=3, tokens=P, teacher=P,
                 targets=P, scale=1.0, sums=P, listed_logits=P, workspace=P, workspace_bytes=1 << 30)
    return ops.gdp_distill_part(**{**given, **over})


def joint(**over):
    given = dict(n=4, vocab=100, parts=2, list_type=1, target_type=1, listed=3, tokens=P, teacher=P, targets=P, scale=1.0, beta=0.5, rest=1, sums=P,
                 listed_logits=P, loss=P, lse=P, logp=P, stats=P)
    return ops.gdp_distill_joint(**{**given, **over})


def distill_grad(**over):
    given = dict(n=4, vocab=100, first=0, whole_vocab=100, logits=P, logits_stride=100, logits_type=2, list_type=1, target_type=1, listed=3, tokens=P,
                 targets=P, stats=P, grad_loss=P, grad_logp=P, scale=1.0, out=2 * P, out_stride=100)
    return ops.gdp_distill_grad(**{**given, **over})


def history(**over):
    given = dict(tokens=P, places=10, stride=10, token_type=1, length_type=1, prompt_type=1, repetition=1.5, frequency=0.5, presence=0.0,
                 lengths=P, prompts=P)
    return ops.gdp_adjust_history(**{**given, **over})


def adjust(**over):
    given = dict(n=4, vocab=100, first=0, logits=P, logits_stride=100, logits_type=2, out_type=2, history=history(), bias_tokens=P, bias=P,
                 bias_stride=5, biases=5, bias_token_type=1, allowed=P, allowed_stride=4, words=4, scales=None, scale=1.0, out=2 * P,
                 out_stride=100)
    return ops.gdp_adjust(**{**given, **over})


def adjust_grad(grad=3 * P, grad_stride=100, **over):
    return ops.gdp_adjust_grad(adjust(**over), grad, grad_stride)


SIZES = [dict(n=-1), dict(vocab=0), dict(vocab=(1 << 22) + 1), dict(n=(1 << 21) + 1), dict(logits_type=3), dict(logits=None), dict(logits_stride=-5), dict(logits=P + 1)]
LISTS = [dict(list_type=2), dict(target_type=2), dict(listed=0), dict(listed=257), dict(listed=-1), dict(tokens=None), dict(tokens=P + 4), dict(targets=P + 4),
         dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf"))]
TEACHER = [dict(teacher=None), dict(teacher=P + 2)]
FORMS = [dict(beta=-0.5), dict(beta=1.5), dict(beta=float("nan")), dict(beta=1.0, rest=0), dict(loss=None), dict(lse=None), dict(logp=None), dict(targets=None), dict(stats=P + 2)]
SPACE = [dict(vocab=1 << 20, workspace_bytes=16), dict(vocab=1 << 20, workspace=P + 8), dict(vocab=1 << 20, workspace=None), dict(n=1 << 21, vocab=1 << 22, logits_type=0)]
BAD = [("gdp_distill_forward", distill, o) for o in SIZES + LISTS + TEACHER + FORMS + SPACE]
BAD += [("gdp_distill_parts", part, o) for o in SIZES + LISTS + TEACHER + SPACE + [
    dict(first=-1), dict(first=(1 << 31) - 100), dict(sums=None), dict(sums=P + 4), dict(listed_logits=None), dict(listed_logits=P + 2)]]
BAD += [("gdp_distill_join", joint, o) for o in LISTS + TEACHER + FORMS + [
    dict(n=-1), dict(n=(1 << 21) + 1), dict(vocab=0), dict(vocab=1 << 31), dict(parts=0), dict(parts=65), dict(sums=None), dict(sums=P + 4), dict(listed_logits=None)]]
BAD += [("gdp_distill_backward", distill_grad, o) for o in SIZES + LISTS + [
    dict(first=-1), dict(whole_vocab=0), dict(stats=None), dict(stats=P + 2), dict(targets=None), dict(grad_loss=P + 1), dict(grad_lse=P + 2), dict(grad_logp=P + 3),
    dict(out=None), dict(out=2 * P + 1), dict(out_stride=99), dict(out=P, logits_stride=120)]]
GIVEN = [dict(first=-1), dict(first=(1 << 31) - 100), dict(out_type=3), dict(logits_type=1), dict(scale=0.0), dict(scale=float("inf")), dict(scale=float("nan")), dict(scales=P + 2),
         dict(biases=-1), dict(biases=1025), dict(words=3), dict(first=60), dict(allowed=P + 2), dict(allowed_stride=-1), dict(out=None), dict(out_stride=99), dict(out=2 * P + 1),
         dict(bias_tokens=None), dict(bias=None), dict(bias=P + 2), dict(bias_tokens=P + 4), dict(bias_token_type=2), dict(bias_stride=-1)]
GIVEN += [dict(history=history(**o)) for o in (
    dict(places=-1), dict(places=(1 << 29) + 1), dict(stride=-1), dict(token_type=2), dict(length_type=2), dict(prompt_type=-1), dict(repetition=0.0), dict(repetition=-1.0),
    dict(repetition=float("nan")), dict(frequency=float("inf")), dict(presence=float("nan")), dict(tokens=P + 4), dict(lengths=P + 4), dict(prompts=P + 4),
    dict(repetitions=P + 1), dict(frequencies=P + 2), dict(presences=P + 3))]
BAD += [("gdp_adjust_forward", adjust, o) for o in SIZES + GIVEN + [dict(out=P, out_type=0), dict(out=P, logits_stride=120)]]
BAD += [("gdp_adjust_backward", adjust_grad, o) for o in SIZES + GIVEN + [dict(grad=None), dict(grad=P + 1), dict(grad_stride=-1), dict(grad=2 * P, out_type=0), dict(grad=2 * P, grad_stride=120)]]
show = lambda v: v if isinstance(v, str) else "" if callable(v) else ",".join(f"{k}" for k in v)   # noqa: E731


@pytest.mark.parametrize("name,make,over", BAD, ids=show)
def test_refused_on_the_host(name, make, over):
    lib = ops._ops()
    assert getattr(lib, name)(ctypes.byref(make(**over)), None) == _lib.GDP_E_BADARG
    assert lib.gdp_last_error().startswith(b"gdp_")


def test_nothing_to_do():
    lib = ops._ops()
    for name, record in (("gdp_distill_forward", distill(n=0, logits=None)), ("gdp_distill_parts", part(n=0, logits=None)), ("gdp_distill_join", joint(n=0, sums=None)),
                         ("gdp_distill_backward", distill_grad(n=0, logits=None)), ("gdp_adjust_forward", adjust(n=0, logits=None)),
                         ("gdp_adjust_backward", adjust_grad(n=0, logits=None, grad=None))):
        assert getattr(lib, name)(ctypes.byref(record), None) == _lib.GDP_OK, name


def test_workspaces():
    lib, size = ops._ops(), ctypes.c_size_t()

    def of(*sizes):
        rc = lib.gdp_distill_workspace(*sizes, ctypes.byref(size))
        return size.value if rc == 0 else rc

    for bad in ((-1, 5, 0, 1), (1, 0, 0, 1), (1, 5, 3, 1), (1, 5, 0, 0), (1, 5, 0, 257)):
        assert of(*bad) == _lib.GDP_E_BADARG
    assert lib.gdp_distill_workspace(1, 5, 0, 1, None) == _lib.GDP_E_BADARG
    assert of(4096, 50000, 2, 20) == of(2050, 1000, 2, 100) == 0            # a workgroup, or a wave, for each row
    assert of(4096, 50000, 2, 100) == 4096 * (16 + 4 * 100)                 # long lists, finished apart
    assert 2 * 16 + 4 * 20 <= of(1, 128000, 2, 20) <= 64 * 16 + 4 * 20 + 512  # sums of each slice, the listed logits once
    assert of(1 << 21, 1 << 22, 2, 256) >= (1 << 21) * (16 * 16 + 4 * 256)  # 2^18 columns of a slice at most


def test_tensors_have_to_be_on_a_device():
    """No CPU path: the operators say so before they touch the library."""
    x, t, q, v = torch.zeros(3, 70), torch.zeros(3, 4, dtype=torch.int64), torch.zeros(3, 4), torch.zeros(3)
    for call in (lambda: ops.distillation(x, t, q), lambda: ops.distillation_grad(x, t, torch.zeros(3, 9), v), lambda: ops.distillation_parts(x, t, q, first=0),
                 lambda: ops.join_distillation(ops.DistillationParts(torch.zeros(1, 3, 4), torch.zeros(1, 3, 4)), t, q, 70), lambda: ops.adjust_logits(x, t),
                 lambda: ops.adjust_logits_grad(x, x, t)):
        with pytest.raises(ValueError, match="HIP device"):
            call()


def test_tangents_are_refused():
    """Forward-mode derivatives would be dropped without a word: the operators say that they have none, whichever tensor carries one."""
    import torch.autograd.forward_ad as fw
    x, t, q, v = torch.zeros(3, 70), torch.zeros(3, 4, dtype=torch.int64), torch.zeros(3, 4), torch.ones(3)
    s, parts = torch.zeros(3, 9), ops.DistillationParts(torch.zeros(1, 3, 4), torch.zeros(1, 3, 4))
    calls = [lambda d: ops.distillation(d(x), t, q), lambda d: ops.distillation(x, t, d(q)), lambda d: ops.distillation_parts(d(x), t, q, first=0),
             lambda d: ops.distillation_parts(x, t, d(q), first=0), lambda d: ops.join_distillation(parts._replace(sums=d(parts.sums)), t, q, 70),
             lambda d: ops.join_distillation(parts, t, d(q), 70), lambda d: ops.distillation_grad(d(x), t, s, v), lambda d: ops.distillation_grad(x, t, d(s), v),
             lambda d: ops.distillation_grad(x, t, s, d(v)), lambda d: ops.distillation_grad(x, t, s, grad_lse=d(v)), lambda d: ops.distillation_grad(x, t, s, v, into=d(x)),
             lambda d: ops.adjust_logits(d(x)), lambda d: ops.adjust_logits(x, t, repetition=d(v)), lambda d: ops.adjust_logits(x, t, frequency=d(v)),
             lambda d: ops.adjust_logits(x, t, presence=d(v)), lambda d: ops.adjust_logits(x, bias_tokens=t, bias=d(q)), lambda d: ops.adjust_logits(x, scale=d(v)),
             lambda d: ops.adjust_logits_grad(d(x), x), lambda d: ops.adjust_logits_grad(x, d(x)), lambda d: ops.adjust_logits_grad(x, x, t, repetition=d(v))]
    for i, call in enumerate(calls):
        with fw.dual_level():
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call(lambda p: fw.make_dual(p.clone(), torch.ones_like(p)))
                pytest.fail(f"call {i}")


@pytest.mark.skipif(shutil.which("nm") is None, reason="no nm")
def test_every_kernel_has_calls_that_reach_it():
    """Scans: few or many listed places, many with the finish behind them where that is short or by the join; a wave a row, or four or eight that read in or past the caches; gradients by
    a wave or four.  Adjusted logits: results of the logits' type or float32;
    no table, entries of 16 or 32 bits (long histories: four vectors a thread), two bits for the gradient; one vector a thread, or four, read
    in or past the caches."""
    names = subprocess.run(["nm", "-C", _lib.LIB_PATH], capture_output=True, text=True, check=True).stdout
    clean = re.sub(r"\(anonymous namespace\)::|ops::", "", names)
    got = {(k, *re.sub(r"\(\w+\)", "", a).split(", ")) for k, a in re.findall(r" ((?:distill|adjust)_\w*kernel)<([^>]*)>", clean)}
    types = ("F32", "F16", "BF16")
    want = {("distill_join_kernel", p) for p in "14"} | {("distill_grad_kernel", t, w) for t in types for w in "14"}
    forms = (("false", "1"), ("false", "4"), ("true", "4"), ("false", "8"), ("true", "8"))
    want |= {("distill_scan_kernel", t, p, "true", *form) for t in types for p in "14" for form in forms if p == "1" or form[0] == "false"}
    want |= {("distill_scan_kernel", t, "4", "false", *form) for t in types for form in forms}
    sizes = (("1", "false"), ("4", "false"), ("4", "true"))
    for t in types:
        for o in {t, "F32"}:
            for back, tables in (("false", "01"), ("true", "03")):
                want |= {("adjust_kernel", t, o, table, back, *size) for table in tables for size in sizes}
            want |= {("adjust_kernel", t, o, "2", "false", "4", past) for past in ("false", "true")}
    assert got == want


def test_the_command_refuses_lists_that_are_too_long(capsys):
    from galvatron_dp import model_ends
    for given in (["--vocab", "2000", "--teacher", "257"], ["--vocab", "20", "--teacher", "21"], ["--vocab", "20", "--teacher", "-1"]):
        with pytest.raises(SystemExit):
            model_ends.main(["--hidden", "64"] + given)
        assert "--teacher" in capsys.readouterr().err
