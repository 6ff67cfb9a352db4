"""The paged attention's matrix-core kernels as compiled (the assembly of csrc/paged_attention.hip with the
Makefile's flags): no product takes as its first or second operand a register that another product wrote last.
The operands come from loads, from LDS and from the vector ALU, never from a product; where one seems to, the
compiler has put a product's result over an operand that is still to be read, as it did with another order
of the same products."""
import re
import shlex
import subprocess

import pytest

import chpe_amd as ca


@pytest.mark.timeout(600)
def test_products_leave_operands_alone(tmp_path):
    out = subprocess.run(["make", "-n", "-B", "_build/paged_attention.o"], cwd=ca.PKG_DIR, capture_output=True, text=True,
                         check=True).stdout
    cmd = shlex.split(next(ln for ln in out.splitlines() if "paged_attention.hip" in ln and "-c" in ln))
    asm = tmp_path / "paged.s"
    cmd[cmd.index("-o") + 1] = str(asm)
    cmd[cmd.index("-c")] = "-S"
    subprocess.run(cmd + ["--cuda-device-only", "-w"], cwd=ca.PKG_DIR, check=True)

    def regs(t):
        m = re.match(r"([va])(?:(\d+)|\[(\d+):(\d+)\])$", t)
        return [] if not m else [f"{m[1]}{i}" for i in range(int(m[2] or m[3]), int(m[2] or m[4]) + 1)]

    name, by_product, products = None, set(), {}
    for line in asm.read_text().splitlines():
        m = re.match(r"(_ZN\S+):", line)
        if m:
            name, by_product = m.group(1), set()
            continue
        t = line.split(";")[0].strip()
        if not name or not t or t.startswith(".") or t.endswith(":"):
            continue
        op, _, rest = t.partition(" ")
        args = [a.strip() for a in rest.split(",")]
        if op.startswith("v_mfma"):
            products[name] = products.get(name, 0) + 1
            for a in args[1:3]:
                clash = by_product & set(regs(a))
                assert not clash, (name, t, sorted(clash))
            by_product |= set(regs(args[0]))
        elif not op.startswith(("global_store", "ds_write", "s_", "scratch_store", "buffer_store")):
            by_product -= set(regs(args[0]))
            if "swap" in op:  # (both registers are written)
                by_product -= set(regs(args[1]))
    assert sum("k_paged_16" in n for n in products) == 13 and sum("k_paged_32" in n for n in products) == 3, products
