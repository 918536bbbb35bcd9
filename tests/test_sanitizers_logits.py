"""The host side of the operators on logits under AddressSanitizer + UndefinedBehaviorSanitizer (no GPU involved): sizes of workspaces and checks
of calls, with arguments from the ends of their ranges.  The program is in tests/sanitize/logits_check.cpp."""
import os
import shutil
import subprocess
from concurrent.futures import ThreadPoolExecutor

import pytest

from galvatron_dp import _build
from test_sanitizers import ENV, SRC, _run

HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")


@pytest.mark.skipif(shutil.which(HIPCC) is None, reason="no hipcc")
def test_logits_host_code_under_sanitizers(tmp_path):
    """Instruments the host pass only (each -fsanitize right after -Xarch_host); the sources are compiled side by side."""
    flags = [f for f in _build.HIPCC_FLAGS if f not in ("-O3", "-shared", "-fPIC")]
    checked = ["-Xarch_host", "-fsanitize=address,undefined", "-Xarch_host", "-fno-sanitize-recover=all"]
    sources = [os.path.join(SRC, "logits_check.cpp")] + [os.path.join(_build.CSRC, s) for s in _build.SOURCES if s.startswith("logit_")]
    objects = [str(tmp_path / (os.path.basename(s) + ".o")) for s in sources]
    assert len(sources) == 3
    with ThreadPoolExecutor(max_workers=3) as pool:
        list(pool.map(lambda so: _run([HIPCC, "-O1", "-g"] + flags + checked + ["-c", so[0], "-o", so[1]]), zip(sources, objects)))
    exe = str(tmp_path / "logits_check")
    _run([HIPCC] + flags + checked + ["-static-libsan"] + objects + ["-o", exe])
    symbols = subprocess.run(["nm", exe], stdout=subprocess.PIPE, text=True).stdout
    assert "__asan_init" in symbols and "__ubsan_handle" in symbols, "the host pass was not instrumented"
    out = _run([exe], env=ENV)
    assert any("calls clean" in ln for ln in out), out
