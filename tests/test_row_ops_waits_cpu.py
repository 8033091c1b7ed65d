"""The order of two stores to one element, read off the assembly of the library's own kernels: where a kernel of
the distillation loss stores elements of the gradient a second time, every wave has waited for its first stores before
the workgroup's last barrier."""
import os
import re
import shutil
import subprocess

import pytest

from motifcl_amd import build


def kernels(text):
    """{name: instructions and labels} of the kernels of an assembly listing."""
    out, name = {}, None
    for line in text.splitlines():
        line = line.split(";")[0].strip()
        if re.match(r"_ZN\w*kernel\w*:$", line):
            name = line[:-1]
            out[name] = []
        elif line.startswith(".Lfunc_end"):
            name = None
        elif name and line and (not line.startswith(".") or line.endswith(":")):
            out[name].append(line)
    return out


def waits_before_last_barrier(code):
    """Whether the instructions of one block end, before the last barrier, with a wait for all stores."""
    last = max(i for i, line in enumerate(code) if line == "s_barrier")
    for line in reversed(code[:last]):
        if line.startswith("s_waitcnt") and "vmcnt(0)" in line:
            return True
        if line.endswith(":") or re.match(r"(global|flat|buffer)_", line):
            return False
    return False


def test_the_check_itself():
    assert waits_before_last_barrier(["global_store_dword v1, v2, off", "s_waitcnt vmcnt(0)", "s_nop 0", "s_barrier", "s_endpgm"])
    assert not waits_before_last_barrier(["s_waitcnt vmcnt(0)", "s_barrier", "global_store_dword v1, v2, off", "s_barrier"])
    assert not waits_before_last_barrier(["s_waitcnt vmcnt(0)", ".LBB0_1:", "s_waitcnt lgkmcnt(0)", "s_barrier"])


def test_the_gradient_is_written_before_it_is_patched(tmp_path):
    hipcc = shutil.which(build._hipcc())
    if hipcc is None:
        pytest.skip("no hipcc")
    listing = str(tmp_path / "distill_top.s")
    subprocess.run([hipcc, *build.FLAGS, "--offload-device-only", "-S", "-o", listing,
                    os.path.join(build.CSRC, "distill_top.hip")], check=True, capture_output=True, text=True)
    with open(listing) as f:
        found = kernels(f.read())
    sweeps = [name for name in found if "distill_sweep_kernel" in name]
    assert len(sweeps) == 3 and len(found) > len(sweeps)  # one for each element type
    checked = 0
    for name, code in found.items():
        if "s_barrier" in code:  # a workgroup of one wave needs none
            assert waits_before_last_barrier(code), name
            checked += 1
    assert checked > len(sweeps)
