"""Build-time guards (no GPU) on the flags that the library is built with, as the Makefile gives them: the guards of
test_build_resources.py, whose own command lines lack some of these flags, on the code that is shipped, and no packed fp32
arithmetic in any of its sources."""
import os
import re
import shlex
import shutil
import subprocess
from concurrent.futures import ThreadPoolExecutor

import pytest

import test_build_resources as guards
import test_operator_build as operator_guards

CSRC = guards.CSRC
SOURCES = ["rnnt_mi355.hip", "joint_mi355.hip", "fused_mi355.hip", "fused_bwd_mi355.hip"]


def shipped_flags():
    """HIPFLAGS as make itself expands them."""
    out = subprocess.run(["make", "-C", CSRC, "-pn", "-f", "Makefile"], capture_output=True, text=True, timeout=300).stdout
    values = dict(re.findall(r"^(HIPFLAGS|ARCH) [:?]?= (.*)$", out, re.M))
    return shlex.split(values["HIPFLAGS"].replace("$(ARCH)", values["ARCH"]))


@pytest.fixture(scope="module")
def shipped():
    flags = shipped_flags()
    assert "--offload-arch=gfx950" in flags and "-O3" in flags
    return flags


def test_every_source_of_the_library_is_guarded():
    text = open(os.path.join(CSRC, "Makefile")).read()
    listed = re.search(r"^SRCS := (.*)$", text, re.M).group(1).split()
    assert sorted(listed) == sorted(SOURCES + operator_guards.SOURCES)


def test_the_operators_guards_compile_what_is_shipped(shipped):
    ignored = {"-fPIC", "-Wall", "-Wno-unused-const-variable"}       # (of no effect on device code)
    assert [f for f in shipped if f not in ignored] == operator_guards.FLAGS


@pytest.fixture(scope="module")
def compiled(shipped, tmp_path_factory):
    """source -> (hipcc's result with its report of resources, device assembly), compiled once for all guards, several at a time."""
    where, run = tmp_path_factory.mktemp("asm"), subprocess.run

    def one(src):
        path, asm = os.path.join(CSRC, src), where / (src + ".s")
        return path, (run(["/opt/rocm/bin/hipcc", *shipped, "-Rpass-analysis=kernel-resource-usage", "--offload-device-only", "-S",
                           "-o", str(asm), path], capture_output=True, text=True, timeout=900), asm)

    with ThreadPoolExecutor(4) as pool:
        return dict(pool.map(one, SOURCES + operator_guards.SOURCES))


@pytest.fixture()
def with_shipped_flags(compiled, monkeypatch):
    """The guards' own hipcc commands give what the shipped flags give for their source."""
    def shipped_run(command, **kw):
        result, asm = compiled[command[-1]]
        if "-S" in command:
            shutil.copy(asm, command[command.index("-o") + 1])
        return result

    monkeypatch.setattr(guards.subprocess, "run", shipped_run)


@pytest.mark.parametrize("src", SOURCES[:2])
def test_no_reachable_kernel_spills(src, tmp_path, with_shipped_flags):
    guards.test_no_reachable_kernel_spills(src, tmp_path)


@pytest.mark.parametrize("src", SOURCES[:2])
def test_no_flat_memory_instructions(src, tmp_path, with_shipped_flags):
    guards.test_no_flat_memory_instructions(src, tmp_path)


@pytest.mark.parametrize("src", SOURCES[2:])
def test_mfma_kernels_stay_within_their_register_budget(src, tmp_path, with_shipped_flags):
    guards.test_mfma_kernels_stay_within_their_register_budget(src, tmp_path)


def test_fused_forward_isa_guards(tmp_path, with_shipped_flags):
    guards.test_fused_forward_isa_guards(tmp_path)


def test_fused_backward_counts_its_own_vector_memory_waits(tmp_path, with_shipped_flags):
    guards.test_fused_backward_counts_its_own_vector_memory_waits(tmp_path)


@pytest.mark.parametrize("src", SOURCES)
def test_no_packed_arithmetic(src, tmp_path, with_shipped_flags):
    kernels = guards._device_asm(src, tmp_path)
    assert kernels
    for name, body in kernels.items():
        assert not re.findall(r"^\s*v_pk_(?:add|mul|fma)_f32", body, re.M)[:5], name


@pytest.mark.parametrize("src", SOURCES + operator_guards.SOURCES)
def test_which_kernels_spill(src, compiled):
    """Exactly: the scan's backward pass with 8 states (as its comment says) and, outside its vocabulary walk, the fused forward kernel
    of the widest joint."""
    result, _ = compiled[os.path.join(CSRC, src)]
    assert result.returncode == 0, result.stderr[-2000:]
    names = re.findall(r"Function Name: (\S+)", result.stderr)
    spills = [int(x) for x in re.findall(r"VGPRs Spill: (\d+)", result.stderr)]
    assert names and len(names) == len(spills)
    known = {"scan_backward_kernel": ("ELi8EEE", 5), "rnnt_fused_proj_k1": ("ELi512EEE", 7)}
    for name, spilled in zip(names, spills):
        limit = next((most for kernel, (form, most) in known.items() if kernel in name and form in name), 0)
        assert spilled <= limit, (name, spilled)
