"""CPU tier of the paged cache: programs that run the kernels' own whole-number code (csrc/fa_paged_index.hpp) on the host."""
import os
import subprocess

import pytest

from conftest import ROOT

CPP = os.path.join(ROOT, "tests", "cpp")


@pytest.mark.parametrize("program", ["paged_walk_check"])
def test_host_program(program):
    subprocess.run(["make", "-s", "-C", CPP, program], check=True)
    r = subprocess.run([os.path.join(CPP, program)], capture_output=True, text=True)
    assert (r.returncode, r.stdout) == (0, "ok\n")
