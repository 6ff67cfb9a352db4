"""The paged attention's matrix-core kernels as compiled, along every path: no product takes as its first or second
operand a register that, on any way there (round a loop's back edge too), a product may have written last.  The operands
come from loads, from LDS and from the vector ALU alone."""
import re
import shlex
import subprocess

import pytest

import chpe_amd as ca

# (what ends at the first comma or blank: the op; registers as v12 or v[12:15], a for accumulation registers)
STORES = ("global_store", "ds_write", "s_", "scratch_store", "buffer_store")


def regs(t):
    m = re.match(r"([va])(?:(\d+)|\[(\d+):(\d+)\])$", t)
    return [] if not m else [f"{m[1]}{i}" for i in range(int(m[2] or m[3]), int(m[2] or m[4]) + 1)]


def kernels(asm):
    """name -> list of (op, args, line without comment), labels as (None, [], label)."""
    out, name = {}, None
    for line in asm.splitlines():
        m = re.match(r"(_ZN\S+):", line)
        if m:
            name = m.group(1)
            out[name] = []
            continue
        t = line.split(";")[0].strip()
        if name is None or not t:
            continue
        if re.match(r"\.L\S+:$", t):
            if t.startswith(".Lfunc_end"):
                name = None
            else:
                out[name].append((None, [], t[:-1]))
        elif not t.startswith("."):
            op, _, rest = t.partition(" ")
            out[name].append((op, [a.strip() for a in rest.split(",")], t))
    return {k: v for k, v in out.items() if any(op and op.startswith("v_mfma") for op, _, _ in v)}


def clashes(code, last_turn_skips_loads=False):
    """What reads a register that a product may have written last, as a product's operand or in a byte permutation (which
    brings V into operands).  last_turn_skips_loads: a turn of the loop that skips the loads of the next tile's V is
    the last one (the source's `more` is then the loop's condition, which the branches alone do not say)."""
    blocks, at = [[]], {}
    for op, args, t in code:
        if op is None:
            blocks.append([])
            at[t] = len(blocks) - 1
            continue
        assert not op.startswith(("s_setpc", "s_swappc", "s_call")), t
        blocks[-1].append((op, args, t))
        if op.startswith(("s_branch", "s_cbranch", "s_endpgm")):
            blocks.append([])
    loads_v = [any(op.startswith("global_load") and t.endswith(" nt") for op, _, t in b) for b in blocks]

    def after(i, skipped):
        op, args = (blocks[i][-1][0], blocks[i][-1][1]) if blocks[i] else ("", [])
        if loads_v[i]:
            skipped = False
        if not op.startswith(("s_branch", "s_cbranch")):
            return [] if op.startswith("s_endpgm") or i + 1 == len(blocks) else [(i + 1, skipped)]
        to, out = at[args[0]], []
        if to > i or not (last_turn_skips_loads and skipped):
            out.append((to, skipped or any(loads_v[i + 1:to]) if to > i else False))
        return out + ([(i + 1, skipped)] if op.startswith("s_cbranch") else [])

    def walk(block, live, found=None):
        for op, args, t in block:
            if op.startswith(("v_mfma", "v_perm_b32")):
                clash = live & {r for a in args[1:3] for r in regs(a)}
                if found is not None and clash:
                    found.append((t, sorted(clash)))
            if op.startswith("v_mfma"):
                live = live | set(regs(args[0]))
            elif not op.startswith(STORES):
                live = live - set(regs(args[0])) - (set(regs(args[1])) if "swap" in op else set())
        return live

    before, todo = {(0, False): set()}, [(0, False)]
    while todo:
        i, skipped = todo.pop()
        live = walk(blocks[i], before[i, skipped])
        for n in after(i, skipped):
            if n not in before or not live <= before[n]:
                before[n] = before.get(n, set()) | live
                todo.append(n)
    found = []
    for (i, _), live in before.items():
        walk(blocks[i], live, found)
    return found


@pytest.mark.timeout(600)
def test_products_leave_operands_alone_on_every_path(tmp_path):
    out = subprocess.run(["make", "-n", "-B", "_build/paged_attention.o"], cwd=ca.PKG_DIR, capture_output=True, text=True,
                         check=True).stdout
    cmd = shlex.split(next(ln for ln in out.splitlines() if "paged_attention.hip" in ln and "-c" in ln))
    asm = tmp_path / "paged.s"
    cmd[cmd.index("-o") + 1] = str(asm)
    cmd[cmd.index("-c")] = "-S"
    subprocess.run(cmd + ["--cuda-device-only", "-w"], cwd=ca.PKG_DIR, check=True)
    code = kernels(asm.read_text())
    assert sum("k_paged_16" in n for n in code) == 13 and sum("k_paged_32" in n for n in code) == 3
    for name, c in code.items():
        # (at head dim 256 two waves share a tile, and one of them may turn once more without a tile of its own)
        found = clashes(c, last_turn_skips_loads="ILi256E" not in name)
        assert not found, (name, found[:3])


LOOP = """_ZN4loop:
\tglobal_load_dword v1, v[20:21], off
\tv_mov_b32_e32 v2, 0
.LBB0_1:
\tv_mfma_f32_16x16x4_f32 v[4:7], v1, v2, v[4:7]
{0}
\ts_cbranch_scc1 .LBB0_1
\ts_endpgm
"""


def test_a_clash_round_the_back_edge_is_found():
    """The check itself: a product's result that only the next turn of the loop reads as an operand."""
    clean = LOOP.format("\tv_mfma_f32_16x16x4_f32 v[8:11], v2, v1, v[8:11]")
    late = LOOP.format("\tv_mfma_f32_16x16x4_f32 v[0:3], v2, v1, v[8:11]")
    mended = LOOP.format("\tv_mfma_f32_16x16x4_f32 v[0:3], v2, v1, v[8:11]\n\tv_mov_b32_e32 v2, v9\n"
                         "\tglobal_load_dword v1, v[20:21], off")
    assert [bool(clashes(kernels(t)["_ZN4loop"])) for t in (clean, late, mended)] == [False, True, False]
    # loads that are skipped on the last turn only: nothing reads the result that stands in their place
    skips = LOOP.format("\tv_mfma_f32_16x16x4_f32 v[0:3], v2, v1, v[8:11]\n\ts_cbranch_vccnz .LBB0_2\n"
                        "\tglobal_load_dwordx2 v[1:2], v[20:21], off nt\n.LBB0_2:")
    assert clashes(kernels(skips)["_ZN4loop"]) and not clashes(kernels(skips)["_ZN4loop"], True)
    assert clashes(kernels(late)["_ZN4loop"], True)
    perm = LOOP.format("\tv_perm_b32 v30, v4, v1, s2")
    assert clashes(kernels(perm)["_ZN4loop"])
