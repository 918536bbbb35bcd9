"""CPU-only checks of the operators' boundary at its edges: records with row statistics, refusals on the host before any device work."""
import ctypes
import os
import re
import shutil
import subprocess

import pytest

torch = pytest.importorskip("torch")

from galvatron_dp import _lib, operators as ops   # noqa: E402
import test_operators_host as H   # noqa: E402

STATS = {"gdp_logprob_forward_stats": (ops.gdp_logprob_stats, H.logprob), "gdp_logprob_join_stats": (ops.gdp_logprob_joint_stats, H.joint),
         "gdp_logprob_backward_stats": (ops.gdp_logprob_grad_stats, H.logprob_grad)}


def test_records_with_row_stats_have_the_headers_layout(tmp_path):
    if shutil.which("gcc") is None:
        pytest.skip("no gcc")
    records = [r for r, _ in STATS.values()]
    lines = ['#include "%s"' % H.HEADER, "#include <stdio.h>", "int main(void) {"]
    for r in records:
        lines += ['printf("%%zu %%zu\\n", sizeof(%s), offsetof(%s, row_stats));' % (r.__name__, r.__name__)]
    (tmp_path / "a.c").write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", str(tmp_path / "a.c"), "-o", str(tmp_path / "a")], check=True)
    got = [int(v) for v in subprocess.run([str(tmp_path / "a")], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [v for r in records for v in (ctypes.sizeof(r), r.row_stats.offset)]


@pytest.mark.parametrize("name", STATS)
def test_row_stats_refused_on_the_host(name):
    lib = ops._ops()
    record, given = STATS[name]
    for bad in (record(given(), None), record(given(), H.P + 4), record(given(n=-1), H.P), record(given(vocab=0), H.P), record(given(scale=0.0), H.P)):
        assert getattr(lib, name)(ctypes.byref(bad), None) == _lib.GDP_E_BADARG
        assert lib.gdp_last_error().startswith(b"gdp_")
    assert getattr(lib, name)(ctypes.byref(record(given(n=0), None)), None) == _lib.GDP_OK


# ---- the command that measures a model's ends -------------------------------------------------------------------
def test_a_shards_time_is_not_written_as_the_whole_parts(tmp_path, capsys, monkeypatch):
    """The search divides the profile's entry by the tensor-parallel degree itself: a shard's time would be divided twice."""
    from galvatron_dp import model_ends
    path = tmp_path / "computation_profiling_bf16_small.json"
    path.write_text('{"layertype_other_bsz1_seq64": 3.5}')
    monkeypatch.setattr(model_ends, "ModelEnds", lambda *a, **k: None)
    monkeypatch.setattr(model_ends, "measure", lambda *a, **k: 1.0)
    given = ["--hidden", "128", "--vocab", "2000", "--seq", "64", "--shards", "4"]
    with pytest.raises(SystemExit):
        model_ends.main(given + ["--profile", str(path)])
    assert "--profile" in capsys.readouterr().err
    assert path.read_text() == '{"layertype_other_bsz1_seq64": 3.5}'
    assert model_ends.main(given) == {(1, 64): 1.0}          # measured and printed, not under the entry's name
    assert "layertype_other" not in capsys.readouterr().out
    model_ends.main(given[:-2] + ["--profile", str(path)])
    assert '"layertype_other_bsz1_seq64": 1.0' in path.read_text()


# ---- derivatives that there are none of ----------------------------------------------------------------------------
def test_tangents_are_refused():
    """Forward-mode derivatives would be dropped without a word: the operators say that they have none, whichever tensor carries one."""
    import torch.autograd.forward_ad as fw
    t, w, x, v = torch.zeros(3, dtype=torch.int64), torch.ones(5, 8), torch.zeros(3, 9), torch.zeros(3)
    parts = ops.LogprobParts(torch.zeros(1, 3, 4), torch.zeros(1, 3, 0), torch.zeros(1, 3, 0, dtype=torch.int32))
    norm = ops.Norm("layer", torch.ones(9), torch.zeros(9))
    calls = [lambda d: ops.embedding(t, d(w)), lambda d: ops.embedding_grad(t, d(w[:3]), 5), lambda d: ops.embedding_grad(t, w[:3], 5, into=d(w)),
             lambda d: ops.token_logprobs(d(x), t), lambda d: ops.token_logprobs_grad(d(x), t, v, v), lambda d: ops.token_logprobs_grad(x, t, d(v), v),
             lambda d: ops.token_logprobs_grad(x, t, v, d(v)), lambda d: ops.token_logprobs_grad(x, t, v, grad_lse=d(v)),
             lambda d: ops.token_logprobs_grad(x, t, v, entropy=v, grad_entropy=d(v)), lambda d: ops.logprob_parts(d(x), t, first=0),
             lambda d: ops.join_logprobs(parts._replace(stats=d(parts.stats)), t, 9), lambda d: ops.residual_norm(d(x), x, pre=norm),
             lambda d: ops.residual_norm(x, d(x), pre=norm), lambda d: ops.residual_norm(x, x, pre=norm._replace(weight=d(norm.weight))),
             lambda d: ops.residual_norm(x, x, post=norm._replace(bias=d(norm.bias)), pre=norm), lambda d: ops.residual_norm(x, x, pre=norm, gate=d(norm.weight)),
             lambda d: ops.residual_norm_grad(x, x, torch.zeros(3, 4), d(x), pre=norm), lambda d: ops.residual_norm_grad(d(x), x, torch.zeros(3, 4), x, pre=norm),
             lambda d: ops.residual_norm_grad(x, x, torch.zeros(3, 4), x, x, pre=norm._replace(weight=d(norm.weight)))]
    for leaf in (False, True):
        for call in calls:
            with fw.dual_level():
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    call(lambda p: fw.make_dual(p.clone().requires_grad_(leaf), torch.ones_like(p)))
                with pytest.raises(ValueError, match="HIP device"):      # no tangent: goes on to the other checks
                    call(lambda p: p)
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(lambda p: ops.token_logprobs(p, t).logp, (x,), (x,))


# ---- what is compiled ------------------------------------------------------------------------------------------------
@pytest.mark.skipif(shutil.which("nm") is None, reason="no nm")
def test_every_embedding_kernel_has_calls_that_reach_it():
    """Rows of less than 16 bytes are taken an element at a time, by less than a wave; others 16 bytes of the smaller type at a time: 4 elements
    where both types are float32, 8 otherwise."""
    names = subprocess.run(["nm", "-C", _lib.LIB_PATH], capture_output=True, text=True, check=True).stdout
    got = {(k, *a.replace("ops::", "").split(", ")) for k, a in re.findall(r" (embed_\w+_kernel)<([^>]*)>", names.replace("(anonymous namespace)::", " "))}
    types = ("F32", "F16", "BF16")
    want = {("embed_index_kernel", t) for t in ("int", "long")} | {("embed_join_kernel", o, n) for o in types for n in "14"}
    for t in types:
        for o in types:
            wide = "4" if t == o == "F32" else "8"
            want |= {("embed_rows_kernel", t, o, n) for n in ("1", wide)}
            want |= {("embed_sum_kernel", t, o, "1", "false"), ("embed_sum_kernel", t, o, wide, "false"), ("embed_sum_kernel", t, o, wide, "true")}
    assert got == want
