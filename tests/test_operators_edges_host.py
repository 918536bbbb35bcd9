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
