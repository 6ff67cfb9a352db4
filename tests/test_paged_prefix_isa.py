"""The attention behind shared prefixes as compiled: its instances of the paged attention's matrix-core kernels under the
same checks as test_paged_isa_flow.py's, that no product reads as an operand what a product may have written last."""
import shlex
import subprocess

import pytest

import chpe_amd as ca
from test_paged_isa_flow import clashes, kernels


@pytest.mark.timeout(600)
def test_products_leave_operands_alone_on_every_path(tmp_path):
    out = subprocess.run(["make", "-n", "-B", "_build/paged_prefix.o"], cwd=ca.PKG_DIR, capture_output=True, text=True,
                         check=True).stdout
    cmd = shlex.split(next(ln for ln in out.splitlines() if "paged_prefix.hip" in ln and "-c" in ln))
    asm = tmp_path / "prefix.s"
    cmd[cmd.index("-o") + 1] = str(asm)
    cmd[cmd.index("-c")] = "-S"
    subprocess.run(cmd + ["--cuda-device-only", "-w"], cwd=ca.PKG_DIR, check=True)
    code = kernels(asm.read_text())
    assert sum("k_paged_16" in n for n in code) == 10 and sum("k_paged_32" in n for n in code) == 3
    for name, c in code.items():
        found = clashes(c, last_turn_skips_loads="ILi256E" not in name)
        assert not found, (name, found[:3])
