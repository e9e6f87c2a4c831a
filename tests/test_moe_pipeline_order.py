"""The order of the loads that the experts' pipelines count, in the assembly that
hipcc makes of them.

A stage's rows are copied to LDS for all waves of a work-group. Before a barrier
each wave waits until at most a given number of its loads are in flight, which
stands for "all but the youngest stage's". That holds only if the youngest loads
are those of one stage: a copy of the stage before that went out among them would
still be in flight where other waves read it.
"""
import os
import re
import shutil
import subprocess

import pytest

PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "qwen-mlx_amd")


def _kind(line):
    """x: 16 bytes a lane to LDS, s: 4 bytes a lane to LDS, r: to registers."""
    if not re.match(r"(global|buffer)_load", line):
        return None
    if not re.search(r"\blds\b", line):
        return "r"
    return "x" if "dwordx4" in line else "s"


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    out = tmp_path_factory.mktemp("asm") / "moe.s"
    line = subprocess.run(["make", "-s", "-n", "-B", "-C", PKG, "_obj/gdn_moe.hip.o"], check=True,
                          capture_output=True, text=True).stdout
    cmd = next(ln for ln in line.splitlines() if "-c -o" in ln).split()
    cmd[cmd.index("-o") + 1] = str(out)
    cmd[cmd.index("-c")] = "-S"
    subprocess.run([*cmd, "--cuda-device-only"], check=True, cwd=PKG, capture_output=True)
    found = {}
    for m in re.finditer(r"^_ZN3gdn\w*?moe_(tile|stream|wide)_kernel(I\w*?E)EvNS\w*:[^\n]*\n(.*?)"
                         r"^\.Lfunc_end", out.read_text(), re.S | re.M):
        code = [ln.split(";")[0].strip() for ln in m.group(3).splitlines()]
        found[m.group(1), m.group(2)] = [ln for ln in code if ln and not ln.startswith(".")]
    return found


@pytest.mark.skipif(shutil.which("make") is None or not os.path.exists("/opt/rocm/bin/hipcc"),
                    reason="needs make and hipcc")
@pytest.mark.parametrize("kernel,args,stage,barriers", [
    # the loads of the youngest stage at a barrier that leaves it in flight, and how
    # many such barriers there are at least: after the first loads and in the loop
    ("tile", "ILi1ELb1EE", "xrrs", 4), ("tile", "ILi1ELb0EE", "xrrs", 4),
    ("tile", "ILi2ELb1EE", "xxrrs", 4), ("tile", "ILi2ELb0EE", "xxrrs", 4),
    ("stream", "ILi1ELb1EE", "xxrrs", 4), ("stream", "ILi1ELb0EE", "xxrrs", 4),
    ("stream", "ILi2ELb1EE", "xxrrs", 4), ("stream", "ILi2ELb0EE", "xxrrs", 4),
    ("wide", "ILb1EE", "rrrrrr", 5), ("wide", "ILb0EE", "rrrrrr", 5)])
def test_loads_in_flight_at_a_barrier_are_one_stage(kernels, kernel, args, stage, barriers):
    code = kernels[kernel, args]
    seen = 0
    for i in (j for j, ln in enumerate(code) if ln.startswith("s_barrier")):
        vm, lgkm, loads = None, False, []
        for ln in reversed(code[:i]):
            if ln.startswith("s_waitcnt") and not loads:
                n = re.search(r"vmcnt\((\d+)\)", ln)
                vm = int(n.group(1)) if n and vm is None else vm
                lgkm = lgkm or "lgkmcnt(0)" in ln
            elif _kind(ln):
                loads.append(_kind(ln))
            if vm is None and loads:
                break
            if vm is not None and len(loads) >= vm:
                break
        if not vm:  # nothing in flight, or a barrier without copies
            continue
        seen += 1
        assert lgkm, "LDS reads are not waited for"
        assert vm == len(stage) and sorted(loads) == sorted(stage), (i, vm, loads)
    assert seen >= barriers
