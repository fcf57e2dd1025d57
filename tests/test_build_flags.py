"""The library is the one that the Makefile describes: objects of other flags are not kept, and no kernel holds packed fp32
arithmetic, which the build turns off."""
import os
import re
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "pigeon_amd", "csrc")
needs_make = pytest.mark.skipif(shutil.which("make") is None, reason="make not available")


def _sources():
    return re.search(r"^SRCS\s*:=\s*(.*)$", open(os.path.join(CSRC, "Makefile")).read(), re.M).group(1).split()


@needs_make
@pytest.mark.parametrize("target", ["all", "tuning"])
def test_a_change_of_the_flags_compiles_every_source_again(target):
    out = subprocess.run(["make", "-C", CSRC, "-n", "-W", "Makefile", target], capture_output=True, text=True, timeout=60)
    assert out.returncode == 0, out.stderr[-2000:]
    for src in _sources():
        lines = [ln for ln in out.stdout.splitlines() if f"-c {src} " in ln]
        assert len(lines) == 1 and "-packed-fp32-ops" in lines[0], src


def test_every_source_belongs_to_the_library():
    assert sorted(_sources()) == sorted(f for f in os.listdir(CSRC) if f.endswith(".hip"))


@pytest.mark.skipif(not os.path.exists("/opt/rocm/llvm/bin/llvm-objdump"), reason="llvm-objdump not available")
def test_no_kernel_of_the_built_objects_holds_packed_fp32_arithmetic(tmp_path):
    """Of the objects that are built here from the sources beside them."""
    objects = [os.path.join(CSRC, "build", src.replace(".hip", ".o")) for src in _sources()]
    if not all(os.path.exists(o) for o in objects):
        pytest.skip("nothing is built")
    for o in objects:
        copy = shutil.copy(o, tmp_path)                             # the device code is written beside its object
        subprocess.run(["/opt/rocm/llvm/bin/llvm-objdump", "--offloading", copy], capture_output=True, check=True, timeout=120)
    code = [p for p in sorted(os.listdir(tmp_path)) if "gfx950" in p]
    assert code
    kernels = 0
    for p in code:
        text = subprocess.run(["/opt/rocm/llvm/bin/llvm-objdump", "-d", str(tmp_path / p)], capture_output=True, text=True, check=True, timeout=300).stdout
        kernels += text.count("s_endpgm")
        assert not re.search(r"\bv_pk_(add|mul|fma)_f32\b", text), p
    assert kernels > 100
