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


def test_workspace_of_long_prompts(fa):
    """Long prompts' row tiles fill the chip by themselves: their rows are not divided, and no room for parts of them is asked for
    beyond 1 GiB, or beyond one part behind the prefix and one of the prefix."""
    for T, B, Hq, Hkv, D in [(65536, 1, 64, 8, 128), (40000, 3, 64, 8, 128), (65536, 4, 32, 8, 256), (200000, 16, 32, 32, 64)]:
        rows, part = T * Hq, (D + 2) * 4
        assert rows * part > 1 << 30
        assert fa.lib().fa_shared_prefix_workspace(T, B, Hq, Hkv, D, 0, 1 << 20) == 4 * rows
        assert fa.lib().fa_shared_prefix_workspace(T, B, Hq, Hkv, D, 5000, 1 << 20) == rows * (2 * part + 4)
    rows, part = 33000 * 64, 66 * 4
    assert fa.lib().fa_shared_prefix_workspace(33000, 2, 64, 4, 64, 0, 1 << 20) == rows * (part + 4)
