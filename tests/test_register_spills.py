"""The attention and log-probability kernels keep every vector register where it is: the sources compiled to assembly hold no access to
scratch memory, and the compiler's resource counts say the same."""
import os
import re
import subprocess

import pytest


@pytest.mark.parametrize("source,kernels", [("attention.hip", 8), ("logprobs.hip", 16)])
def test_no_vector_register_is_spilled(tmp_path, source, kernels):
    from llmq_amd import build as B
    out = tmp_path / "out.s"
    r = subprocess.run([B.HIPCC] + B.FLAGS + ["--cuda-device-only", "-S", os.path.join(B.CSRC, source), "-o", str(out)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]
    text = out.read_text()
    spilled = {m.group(1): int(m.group(2)) for m in re.finditer(r"\.name: +(_Z\w+)\n(?:(?! +- ).*\n)*? +\.vgpr_spill_count: (\d+)", text)}
    ours = {k: n for k, n in spilled.items() if "attention" in k or "logprobs" in k}
    assert len(ours) >= kernels and not any(ours.values()), ours
    assert not re.search(r"^\s+(scratch|buffer)_(load|store)", text, re.M)
