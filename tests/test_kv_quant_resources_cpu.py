"""What the compiler makes of the kernels of the 4- and 8-bit cache, checked without a GPU: registers, scratch
memory and LDS as hipcc reports them with the library's own flags.  The attention's layouts count on two (at
head_dim 64 three) waves on a SIMD, and a change that looks harmless in the source can move accumulators
into scratch memory."""
import os
import re
import shutil
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "ml-recurrent-drafter_amd"))
import build_hip  # noqa: E402

pytestmark = pytest.mark.skipif(shutil.which(build_hip.HIPCC) is None and not os.path.exists(build_hip.HIPCC),
                                reason="needs hipcc")


def _usage(tmp_path_factory, source):
    out = tmp_path_factory.mktemp("ru") / "x.o"
    cmd = [build_hip.HIPCC, "-x", "hip", *build_hip.FLAGS, "-Rpass-analysis=kernel-resource-usage", "-c",
           os.path.join(build_hip.CSRC, source), "-o", str(out)]
    r = subprocess.run(cmd, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]
    kernels, name = {}, None
    for line in r.stderr.splitlines():
        m = re.search(r"remark: (?:Function Name: (\S+)|\s*([A-Za-z ]+?)(?: \[[^\]]*\])?: (\d+))", line)
        if m and m.group(1):
            name = m.group(1)
            kernels[name] = {}
        elif m and name is not None:
            kernels[name][m.group(2).strip()] = int(m.group(3))
    return kernels


def test_attention_layouts(tmp_path_factory):
    usage = _usage(tmp_path_factory, "quant_attention.hip")
    found = 0
    for name, u in usage.items():
        m = re.search(r"attn_quant_kernelI.*?Li(\d+)ELi(\d+)ELi(\d+)ELi(\d+)ELi(\d+)EE", name)
        if not m:
            assert u["ScratchSize"] == 0, (name, u)
            continue
        bits, dim, rb, r, k = map(int, m.groups())
        found += 1
        assert u["VGPRs"] <= 256 and u["LDS Size"] <= 163840, (name, u)
        assert u["Occupancy"] >= (3 if dim == 64 and r == 1 else 2), (name, u)
        # a few words that the second sweep, the one for NaN blocks, keeps there
        limit = 0 if r > 1 or rb == 1 else (64 if dim == 64 else (40 if bits == 8 else 0))
        assert u["ScratchSize"] <= limit, (name, u)
    assert found == 2 * 2 * 2 * 4, found  # types, bits, head sizes, layouts


def test_append_and_read_kernels(tmp_path_factory):
    usage = _usage(tmp_path_factory, "kv_quant.hip")
    kernels = {k: v for k, v in usage.items() if "quant" in k}
    assert len(kernels) == 3 * 3 * 2, sorted(usage)
    for name, u in kernels.items():
        assert u["ScratchSize"] == 0 and u["VGPRs"] <= 128, (name, u)
