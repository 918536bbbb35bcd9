"""CPU-only checks of the operators' boundary: the library exports what their header declares, the records have its layout,
and calls are refused on the host, before any device work (no kernel is launched here)."""
import ctypes
import os
import re
import shutil
import subprocess

import pytest

torch = pytest.importorskip("torch")

from galvatron_dp import _lib, operators as ops   # noqa: E402

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "galvatron_ops_hip.h")
RECORDS = (ops.gdp_embed, ops.gdp_embed_grad, ops.gdp_logprob, ops.gdp_logprob_part, ops.gdp_logprob_joint,
           ops.gdp_logprob_grad, ops.gdp_norm_params, ops.gdp_norm, ops.gdp_norm_grad)


def test_header_symbols_are_exported():
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    names = set(re.findall(r"\bint (gdp_[a-z_]+)\s*\(", text))
    assert names == set(ops.EXPORTED_SYMBOLS)
    for n in names:
        assert getattr(_lib.lib(), n) is not None
    assert int(re.search(r"GDP_MAX_TOP (\d+)", text)[1]) == ops.MAX_TOP
    assert int(re.search(r"GDP_MAX_NORM_DIM (\d+)", text)[1]) == ops.MAX_NORM_DIM


def test_records_have_the_headers_layout(tmp_path):
    """Every member's offset, as a C compiler lays the header's structures out."""
    if shutil.which("gcc") is None:
        pytest.skip("no gcc")
    lines = ['#include "%s"' % HEADER, "#include <stdio.h>", "int main(void) {"]
    for r in RECORDS:
        lines += ['printf("%%zu\\n", sizeof(%s));' % r.__name__]
        lines += ['printf("%%zu\\n", offsetof(%s, %s));' % (r.__name__, f[0]) for f in r._fields_]
    (tmp_path / "a.c").write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", str(tmp_path / "a.c"), "-o", str(tmp_path / "a")], check=True)
    got = [int(v) for v in subprocess.run([str(tmp_path / "a")], capture_output=True, text=True, check=True).stdout.split()]
    want = [v for r in RECORDS for v in [ctypes.sizeof(r)] + [getattr(r, f[0]).offset for f in r._fields_]]
    assert got == want


P = 1 << 20     # an address that nothing reads: every call below is refused or has nothing to do


def embed(**over):
    given = dict(n=4, rows=8, dim=16, first=0, tokens=P, token_type=1, weight_type=0, out_type=0, scale=1.0, weight=P, weight_stride=16,
                 out=P, out_stride=16)
    return ops.gdp_embed(**{**given, **over})


def embed_grad(**over):
    given = dict(n=4, rows=8, dim=16, first=0, tokens=P, token_type=1, grad_type=0, out_type=0, accumulate=0, scale=1.0, grad=P,
                 grad_stride=16, out=P, out_stride=16, workspace=P, workspace_bytes=1 << 30)
    return ops.gdp_embed_grad(**{**given, **over})


def logprob(**over):
    given = dict(n=4, vocab=100, logits=P, logits_stride=100, logits_type=2, token_type=1, tokens=P, scale=1.0, top=2, logp=P, lse=P,
                 entropy=P, top_logp=P, top_tokens=P, workspace=P, workspace_bytes=1 << 30)
    return ops.gdp_logprob(**{**given, **over})


def part(**over):
    given = dict(n=4, vocab=100, first=0, logits=P, logits_stride=100, logits_type=2, token_type=1, tokens=P, scale=1.0, top=2, stats=P,
                 top_logits=P, top_tokens=P, workspace=P, workspace_bytes=1 << 30)
    return ops.gdp_logprob_part(**{**given, **over})


def joint(**over):
    given = dict(n=4, vocab=100, parts=2, top=2, scale=1.0, token_type=1, tokens=P, stats=P, top_logits=P, top_tokens=P, logp=P, lse=P,
                 entropy=P, top_logp=P, out_tokens=P)
    return ops.gdp_logprob_joint(**{**given, **over})


def logprob_grad(**over):
    given = dict(n=4, vocab=100, first=0, whole_vocab=100, logits=P, logits_stride=100, logits_type=2, token_type=1, tokens=P, scale=1.0,
                 top=0, lse=P, grad_logp=P, out=2 * P, out_stride=100)
    return ops.gdp_logprob_grad(**{**given, **over})


def side(**over):
    return ops.gdp_norm_params(**{**dict(form=1, type=0, eps=1e-5, weight=P, bias=P), **over})


def norm(**over):
    given = dict(n=4, dim=16, type=2, stream_type=0, residual=P, residual_stride=16, block=P, block_stride=16, post=side(), pre=side(), gate=P,
                 gates=2, gate_stride=16, gate_type=2, residual_scale=1.0, block_scale=1.0, stream=P, stream_stride=16, normed=P,
                 normed_stride=16, stats=P)
    return ops.gdp_norm(**{**given, **over})


def norm_grad(**over):
    given = dict(n=4, dim=16, type=2, stream_type=0, stream=P, stream_stride=16, block=P, block_stride=16, stats=P, grad_normed=P,
                 grad_normed_stride=16, grad_stream=P, grad_stream_stride=16, post=side(), pre=side(), gate=P, gates=2, gate_stride=16,
                 gate_type=2, residual_scale=1.0, block_scale=1.0, grad_residual=P, grad_residual_stride=16, grad_block=P,
                 grad_block_stride=16, grad_pre_weight=P, grad_pre_bias=P, grad_post_weight=P, grad_post_bias=P, grad_gate=P,
                 workspace=P, workspace_bytes=1 << 30)
    return ops.gdp_norm_grad(**{**given, **over})


BAD = [("gdp_embed_forward", embed, o) for o in (
    dict(n=-1), dict(rows=-1), dict(dim=-1), dict(first=-1), dict(n=1 << 26), dict(rows=(1 << 27) + 1), dict(dim=(1 << 20) + 1), dict(weight_type=3), dict(out_type=-1),
    dict(token_type=2), dict(tokens=None), dict(weight=None), dict(out=None), dict(weight_stride=-16), dict(out_stride=15), dict(weight_stride=1 << 60),
    dict(weight=P + 2), dict(out=P + 1), dict(tokens=P + 4))]
BAD += [("gdp_embed_backward", embed_grad, o) for o in (
    dict(n=-1), dict(rows=-1), dict(dim=-1), dict(first=-1), dict(grad_type=3), dict(out_type=5), dict(token_type=7), dict(tokens=None), dict(grad=None), dict(out=None),
    dict(workspace=None), dict(workspace=P + 16), dict(workspace_bytes=10), dict(grad_stride=-1), dict(out_stride=8), dict(grad=P + 1), dict(tokens=P + 2))]
BAD += [(name, make, o) for name, make in (("gdp_logprob_forward", logprob), ("gdp_logprob_parts", part)) for o in (
    dict(n=-1), dict(vocab=0), dict(vocab=(1 << 22) + 1), dict(n=(1 << 21) + 1), dict(logits_type=3), dict(token_type=2), dict(top=-1), dict(top=65),
    dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(logits=None), dict(tokens=None), dict(top_tokens=None),
    dict(logits_stride=-5), dict(logits=P + 1), dict(tokens=P + 4), dict(n=1 << 20, vocab=1 << 22, logits_type=0),
    dict(vocab=1 << 20, workspace_bytes=16), dict(vocab=1 << 20, workspace=P + 8), dict(vocab=1 << 20, workspace=None))]
BAD += [("gdp_logprob_forward", logprob, o) for o in (dict(top=40, vocab=39), dict(logp=None), dict(lse=None), dict(entropy=None), dict(top_logp=None))]
BAD += [("gdp_logprob_parts", part, o) for o in (dict(first=-1), dict(first=(1 << 31) - 100), dict(stats=None), dict(stats=P + 4), dict(top_logits=None))]
BAD += [("gdp_logprob_join", joint, o) for o in (
    dict(n=-1), dict(n=(1 << 21) + 1), dict(vocab=0), dict(vocab=1 << 31), dict(parts=0), dict(parts=65), dict(top=-1), dict(top=65), dict(top=3, vocab=2), dict(token_type=2),
    dict(scale=0.0), dict(tokens=None), dict(stats=None), dict(logp=None), dict(lse=None), dict(entropy=None), dict(top_logits=None), dict(top_tokens=None),
    dict(top_logp=None), dict(out_tokens=None), dict(stats=P + 4), dict(tokens=P + 2))]
BAD += [("gdp_logprob_backward", logprob_grad, o) for o in (
    dict(n=-1), dict(vocab=0), dict(first=-1), dict(whole_vocab=0), dict(logits_type=9), dict(token_type=2), dict(scale=0.0), dict(logits=None), dict(out=None),
    dict(tokens=None), dict(lse=None), dict(entropy=P), dict(grad_entropy=P), dict(top=1), dict(top=65), dict(out_stride=99), dict(out=P, logits_stride=120), dict(out=2 * P + 1))]
BAD += [("gdp_norm_forward", norm, o) for o in (
    dict(n=-1), dict(n=1 << 22), dict(dim=0), dict(dim=16385), dict(type=3), dict(stream_type=1), dict(post=side(form=3)), dict(pre=side(type=4)), dict(pre=side(eps=-1.0)),
    dict(post=side(eps=float("nan"))), dict(pre=side(weight=P + 2)), dict(post=side(bias=P + 1)), dict(block=None), dict(block=None, gate=None), dict(gates=3), dict(gates=0),
    dict(gate_type=8), dict(gate=P + 1), dict(gate_stride=-1), dict(residual=None), dict(normed=None), dict(pre=side(form=0)), dict(pre=side(form=0), normed=None, stream=None),
    dict(residual_stride=-1), dict(stream_stride=15), dict(normed_stride=0), dict(residual=P + 2), dict(block=P + 1), dict(stats=P + 8))]
BAD += [("gdp_norm_backward", norm_grad, o) for o in (
    dict(n=-1), dict(dim=0), dict(dim=16385), dict(stream_type=1), dict(post=side(form=-1)), dict(block=None), dict(gates=3), dict(gate=None), dict(pre=side(form=0)),
    dict(post=side(form=0)), dict(stats=None), dict(stats=P + 4), dict(grad_normed=None), dict(stream=None), dict(workspace=None), dict(workspace=P + 4), dict(workspace_bytes=64),
    dict(grad_residual_stride=15), dict(grad_block_stride=3), dict(grad_stream=P + 2), dict(grad_block=P + 1))]


@pytest.mark.parametrize("name,make,over", BAD, ids=lambda v: v if isinstance(v, str) else "" if callable(v) else ",".join(v))
def test_refused_on_the_host(name, make, over):
    ops._ops()
    lib = _lib.lib()
    assert getattr(lib, name)(ctypes.byref(make(**over)), None) == _lib.GDP_E_BADARG
    assert lib.gdp_last_error().startswith(b"gdp_")


def test_null_and_nothing_to_do():
    lib = ops._ops()
    for name in ops.EXPORTED_SYMBOLS:
        if not name.endswith("workspace"):
            assert getattr(lib, name)(None, None) == _lib.GDP_E_BADARG
    for name, record in (("gdp_embed_forward", embed(n=0, tokens=None, out=None)), ("gdp_embed_forward", embed(dim=0)),
                         ("gdp_embed_backward", embed_grad(rows=0, out=None)), ("gdp_embed_backward", embed_grad(n=0, tokens=None, grad=None, accumulate=1)),
                         ("gdp_logprob_forward", logprob(n=0, logits=None)), ("gdp_logprob_parts", part(n=0, logits=None)), ("gdp_logprob_join", joint(n=0, stats=None)),
                         ("gdp_logprob_backward", logprob_grad(n=0, logits=None)), ("gdp_norm_forward", norm(n=0, residual=None))):
        assert getattr(lib, name)(ctypes.byref(record), None) == _lib.GDP_OK, name


def test_workspaces():
    lib, size = ops._ops(), ctypes.c_size_t()

    def of(name, *sizes):
        rc = getattr(lib, name)(*sizes, ctypes.byref(size))
        return size.value if rc == 0 else rc

    assert of("gdp_embed_grad_workspace", -1, 1, 1) == _lib.GDP_E_BADARG
    assert of("gdp_logprob_workspace", 1, 0, 0, 0) == _lib.GDP_E_BADARG
    assert of("gdp_norm_grad_workspace", 6, 8, 4) == _lib.GDP_E_BADARG
    assert lib.gdp_embed_grad_workspace(1, 1, 1, None) == _lib.GDP_E_BADARG
    # the order of the tokens, two numbers a row, two partial sums for each piece of 16 to 128 places
    n, rows, dim = 5000, 700, 1024
    assert 8 * n + 8 * rows + n // 128 * 2 * dim * 4 <= of("gdp_embed_grad_workspace", n, rows, dim) <= 8 * n + 16 * rows + (n // 16 + 1) * 2 * dim * 4 + 4096
    assert of("gdp_logprob_workspace", 4096, 50000, 2, 20) == 0              # a workgroup for each row
    assert 0 < of("gdp_logprob_workspace", 1, 128000, 2, 20) <= 64 * (16 + 8 * 20) + 1024
    assert of("gdp_norm_grad_workspace", 1, 64, 0) == 5 * 64 * 4
    assert of("gdp_norm_grad_workspace", 1 << 20, 64, 4) <= 4096 * 5 * 64 * 4


def test_tensors_have_to_be_on_a_device():
    """No CPU path: the operators say so before they touch the library."""
    t, w, x = torch.zeros(3, dtype=torch.int64), torch.ones(5, 8), torch.zeros(3, 9)
    for call in (lambda: ops.embedding(t, w), lambda: ops.embedding_grad(t, w[:3], 5), lambda: ops.token_logprobs(x, t),
                 lambda: ops.token_logprobs_grad(x, t, x[:, 0], x[:, 0]), lambda: ops.logprob_parts(x, t, first=0),
                 lambda: ops.join_logprobs(ops.LogprobParts(torch.zeros(1, 3, 4), torch.zeros(1, 3, 0), torch.zeros(1, 3, 0, dtype=torch.int32)), t, 9),
                 lambda: ops.residual_norm(x, x, pre=ops.Norm("rms")), lambda: ops.residual_norm_grad(x, x, torch.zeros(3, 4), x, pre=ops.Norm("rms"))):
        with pytest.raises(ValueError, match="HIP device"):
            call()


def test_one_runtime_in_the_process():
    """The library loaded before torch brings a HIP runtime of its own, whose streams torch's are not: the operators refuse that process."""
    code = ("import sys; sys.path.insert(0, %r)\nfrom galvatron_dp import _lib\n_lib.lib()\nfrom galvatron_dp import operators\n"
            "n = len({l.split()[-1] for l in open('/proc/self/maps') if 'libamdhip64' in l})\n"
            "try:\n    operators._ops()\n    print('bound', n)\nexcept RuntimeError as e:\n    print('refused', n, 'import torch' in str(e))\n")
    out = subprocess.run(["python3", "-c", code % os.path.join(ROOT, "hetu-galvatron_amd")], capture_output=True, text=True).stdout.split()
    assert out in (["bound", "1"], ["refused", "2", "True"]), out
