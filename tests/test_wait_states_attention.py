"""The wait states between matrix instructions and the code on their results (tests/test_wait_states.py) in the
attention kernels, those with a relative position bias among them: their near and far tiles lie behind branches."""
import re
import subprocess

import pytest

from mind_amd import _build
from tests import test_wait_states as waits


@pytest.mark.parametrize("source,least", [("esa_attn_dense", 6), ("esa_attn_wide", 40), ("esa_attn", 40)])
def test_no_early_use_in_attention(source, least, tmp_path, monkeypatch):
    monkeypatch.setitem(waits.MFMA, "16x16x16_bf16", (4, 7))
    out = tmp_path / "kernels.txt"
    run = subprocess.run([_build.hipcc(), *_build.HIPFLAGS, "--cuda-device-only", "-S", str(_build.CSRC / f"{source}.hip"),
                          "-o", str(out)], capture_output=True, text=True)
    assert run.returncode == 0, run.stderr[-2000:]
    kernels = [part.split("\n.Lfunc_end")[0].split("\n")[1:] for part in re.split(r"\n(?=_Z\w+:)", out.read_text())[1:]]
    kernels = [k for k in kernels if any("v_mfma" in line for line in k)]
    assert len(kernels) >= least and not any(waits.early_uses(k) for k in kernels)
