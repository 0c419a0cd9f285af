"""Build-time guards (no GPU) of the prediction network's and the decoder's kernels, read from hipcc's own output: registers
spilled to scratch, accesses that lost their address space, and packed fp32 instructions, none of which a test of
results shows."""
import os
import re
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "rnnt_amd", "csrc")
FLAGS = ["-O3", "-std=c++17", "--offload-arch=gfx950", "-ffp-contract=off", "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]
SOURCES = ["embedding_mi355.hip", "state_space_mi355.hip", "rules_mi355.hip"]
MAX_SPILLED_VGPRS = 8


@pytest.mark.parametrize("src", SOURCES)
def test_no_kernel_spills(src, tmp_path):
    out = subprocess.run(["/opt/rocm/bin/hipcc", *FLAGS, "-fPIC", "-Rpass-analysis=kernel-resource-usage", "-c", "-o", str(tmp_path / "o.o"),
                          os.path.join(CSRC, src)], capture_output=True, text=True, timeout=900)
    assert out.returncode == 0, out.stderr[-2000:]
    names = re.findall(r"Function Name: (\S+)", out.stderr)
    spills = [int(x) for x in re.findall(r"VGPRs Spill: (\d+)", out.stderr)]
    assert names and len(names) == len(spills)
    assert not [(n, s) for n, s in zip(names, spills) if s > MAX_SPILLED_VGPRS]


@pytest.mark.parametrize("src", SOURCES)
def test_no_flat_accesses_and_no_packed_arithmetic(src, tmp_path):
    asm = tmp_path / "k.s"
    out = subprocess.run(["/opt/rocm/bin/hipcc", *FLAGS, "--offload-device-only", "-S", "-o", str(asm), os.path.join(CSRC, src)],
                         capture_output=True, text=True, timeout=900)
    assert out.returncode == 0, out.stderr[-2000:]
    text = asm.read_text()
    assert "global_load" in text
    assert not re.findall(r"^\s*flat_(?:load|store|atomic)\S*", text, re.M)[:5]
    assert not re.findall(r"^\s*v_pk_(?:add|mul|fma)_f32", text, re.M)[:5]


def test_the_scan_reads_its_rows_through_the_scalar_cache(tmp_path):
    """B and C of a step are scalar operands of the recurrence: a row that became a vector load (a pointer that hipcc no
    longer sees as the wave's) would cost a register and a load per state and lane."""
    asm = tmp_path / "k.s"
    out = subprocess.run(["/opt/rocm/bin/hipcc", *FLAGS, "--offload-device-only", "-S", "-o", str(asm), os.path.join(CSRC, SOURCES[1])],
                         capture_output=True, text=True, timeout=900)
    assert out.returncode == 0, out.stderr[-2000:]
    kernels = {m.group(1): m.group(2) for m in re.finditer(r"^(_Z\w+):[^\n]*\n(.*?)^\.Lfunc_end\d+:", asm.read_text(), flags=re.S | re.M)}
    walks = {n: b for n, b in kernels.items() if "scan_forward_kernel" in n or "scan_backward_local_kernel" in n}
    assert len(walks) == 27       # {full, local, backward local} x {fp32, bf16, fp16} x {8, 16, 32 states}
    for name, body in walks.items():
        assert len(re.findall(r"s_load_dwordx(?:8|16) ", body)) >= 1, name
