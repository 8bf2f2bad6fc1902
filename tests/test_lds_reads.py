"""No kernel of the library touches a register that an LDS read is still to fill (tests/lds_reads.py), whatever compiler
and flags built it."""
import pytest

from lds_reads import code_objects, compiled, kernels, touched_in_flight


def code(*lines):
    """Instructions four bytes apart; `target: line` is where `branch target` goes."""
    at = {line.split(": ")[0]: 4 * i for i, line in enumerate(lines) if ": " in line}
    out = []
    for i, line in enumerate(lines):
        text = line.split(": ")[-1]
        name = text.split()[-1] if text.startswith(("s_branch", "s_cbranch")) else None
        out.append((4 * i, text, at[name] if name else None))
    return out


READ = "ds_read_b128 v[0:3], v8 offset:16"


@pytest.mark.parametrize("lines,bad", [
    ([READ, "s_waitcnt lgkmcnt(0)", "v_add_f32_e32 v4, v0, v1"], []),
    ([READ, "v_add_f32_e32 v4, v4, v2"], [1]),
    ([READ, "v_mov_b32_e32 v3, 0"], [1]),
    ([READ, "v_mov_b32_e32 v4, v5", "s_waitcnt vmcnt(0)", "v_mov_b32_e32 v5, v3"], [3]),
    ([READ, "ds_read_b32 v9, v4", "s_waitcnt lgkmcnt(1)", "v_mov_b32_e32 v5, v3", "v_mov_b32_e32 v5, v9"], [4]),
    ([READ, "ds_write_b32 v7, v6", "s_waitcnt lgkmcnt(2)", "v_mov_b32_e32 v5, v3"], [3]),
    ([READ, "ds_write_b32 v7, v2"], [1]),
    ([READ, "ds_read_b32 v9, v1"], [1]),
    ([READ, "v_mfma_f32_16x16x32_bf16 a[0:3], v[2:5], v[12:15], a[0:3]"], [1]),
    (["ds_read_b128 a[4:7], v8", "v_accvgpr_read_b32 v0, a5"], [1]),
    # around a loop: the read at its end is waited for at its start, and then not
    (["top: s_waitcnt lgkmcnt(0)", "v_mov_b32_e32 v5, v0", READ, "s_cbranch_scc1 top", "s_endpgm"], []),
    (["top: v_mov_b32_e32 v6, v5", "v_mov_b32_e32 v5, v0", READ, "s_cbranch_scc1 top", "s_endpgm"], [1]),
    # one way to a place waits, the other does not
    ([READ, "s_cbranch_vccz there", "s_waitcnt lgkmcnt(0)", "there: v_mov_b32_e32 v5, v0", "s_endpgm"], [3]),
    ([READ, "s_cbranch_vccz there", "ds_read_b32 v9, v8", "there: s_waitcnt lgkmcnt(1)", "v_mov_b32_e32 v5, v0", "s_endpgm"], [4]),
    ([READ, "s_branch there", "v_mov_b32_e32 v5, v0", "there: s_waitcnt lgkmcnt(0)", "v_mov_b32_e32 v5, v0", "s_endpgm"], []),
])
def test_the_check_itself(lines, bad):
    assert touched_in_flight(code(*lines)) == [(4 * i, lines[i].split(": ")[-1]) for i in bad]


def test_no_register_is_touched_in_flight(cev):
    reads = waits = 0
    for obj in code_objects(cev._abi.LIB_PATH):
        for name, instructions in kernels(obj).items():
            found = touched_in_flight(instructions)
            assert not found, (name, found[:4])
            if "fp8_tile" in name:
                steps = compiled(instructions)
                reads += sum(what == "lds" and bool(fills) for what, fills, _ in steps)
                waits += sum(what == "wait" and bool(arg) for what, arg, _ in steps)
    assert reads > 500 and waits > 200, (reads, waits)  # (counted waits: the code that this is about was looked at)
