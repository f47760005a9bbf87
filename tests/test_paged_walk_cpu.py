"""CPU tier of the paged cache: programs that run the kernels' own whole-number code (csrc/fa_paged_index.hpp) on the host."""
import importlib.util
import os
import subprocess

import pytest

from conftest import ROOT

CPP = os.path.join(ROOT, "tests", "cpp")


@pytest.mark.parametrize("program", ["paged_walk_check", "paged_division_check"])
def test_host_program(program):
    subprocess.run(["make", "-s", "-C", CPP, program], check=True)
    r = subprocess.run([os.path.join(CPP, program)], capture_output=True, text=True)
    assert (r.returncode, r.stdout) == (0, "ok\n")


def test_lanes_exchange_tables_behind_a_barrier(tmp_path):
    """The attention kernels' start: tables that lanes of one wave write to LDS and others read, with nothing between but the order
    of the code, need that order held.  On the assembly that the library is built from."""
    spec = importlib.util.spec_from_file_location("check_owned_regs", os.path.join(ROOT, "tools", "check_owned_regs.py"))
    tool = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(tool)
    out = tmp_path / "paged.s"
    subprocess.run(["/opt/rocm/bin/hipcc", "-O3", "-std=c++17", "--offload-arch=gfx950"] + tool.PAGED_FLAGS +
                   ["-S", "--cuda-device-only", "-o", str(out), tool.PAGED_SRC], check=True, stderr=subprocess.DEVNULL)
    text = out.read_text()
    for kernel in tool.PAGED_KERNELS:
        assert "wave barrier" in tool.body_of(text, kernel).group(0).split("s_barrier")[0]
        tool.audit_exchange(text, kernel)
    planted = "k:\n\tds_write_b32 v0, v1\n\t%s\tds_read_b32 v2, v3\n\ts_barrier\n\tds_write_b32 v0, v1\n\tds_read_b32 v2, v3\n.Lfunc_end0:\n"
    tool.audit_exchange(planted % "; wave barrier\n", "k")
    with pytest.raises(SystemExit):
        tool.audit_exchange(planted % "", "k")
