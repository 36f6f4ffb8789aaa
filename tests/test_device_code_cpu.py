"""The assembly of this build's own kernels (kernel.h_amd/build/co/*.isa, written
by build.py beside the code objects): rules that the compiler cannot keep for
inline assembly."""
import glob
import json
import os
import re

import pytest

CO = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "kernel.h_amd", "build", "co")


def instructions(path):
    """(mnemonic, operands) in order."""
    out = []
    with open(path) as f:
        for line in f:
            m = re.match(r"\t(\S+)\s*(.*?)\s*//", line)
            if m:
                out.append((m[1], [x.strip() for x in m[2].split(",")]))
    return out


def scalars(operand):
    m = re.fullmatch(r"s\[(\d+):(\d+)\]", operand)
    if m:
        return set(range(int(m[1]), int(m[2]) + 1))
    m = re.fullmatch(r"s(\d+)", operand)
    return {int(m[1])} if m else set()


FILES = sorted(glob.glob(os.path.join(CO, "*.isa")))


def test_there_is_assembly():
    if not FILES:
        pytest.skip("not built here")
    assert any("paged_weights" in f for f in FILES)


def test_the_build_says_nothing():
    path = os.path.join(os.path.dirname(CO), "warnings.txt")
    if not FILES:
        pytest.skip("not built here")
    with open(path) as f:
        assert f.read() == ""


@pytest.mark.parametrize("path", FILES, ids=os.path.basename)
def test_vector_writes_of_scalars_settle_before_loads_read_them(path):
    """Five wait states between a vector instruction that writes a scalar
    register and a buffer instruction that reads it."""
    code = instructions(path)
    for i, (op, operands) in enumerate(code):
        if not op.startswith("buffer_"):
            continue
        read = set().union(*(scalars(x) for o in operands for x in o.split()))
        states = 0
        for before, args in reversed(code[max(0, i - 5):i]):
            if states >= 5:
                break
            assert not (before.startswith("v_") and scalars(args[0]) & read), (op, operands, before, args, states)
            states += 1 + int(args[0]) if before == "s_nop" else 1


@pytest.mark.parametrize("path", [f for f in FILES if os.path.basename(f).startswith("paged_")], ids=os.path.basename)
def test_loads_to_lds_bring_their_own_wait_states_and_keep_m0(path):
    """Whatever stands before it, a load straight to LDS has five wait states
    of its own, and M0 is afterwards what it was."""
    code = instructions(path)
    for i, (op, operands) in enumerate(code):
        if not (op.startswith("buffer_load") and "lds" in operands[-1].split()):
            continue
        save, set_m0, nop, restore = code[i - 3], code[i - 2], code[i - 1], code[i + 1]
        assert save[0] == set_m0[0] == restore[0] == "s_mov_b32" and nop[0] == "s_nop", code[i - 3:i + 2]
        assert save[1][1] == "m0" and set_m0[1][0] == "m0" and restore[1] == ["m0", save[1][0]], code[i - 3:i + 2]
        assert int(nop[1][0]) + 3 >= 5, code[i - 3:i + 2]


# Symbols that spill, and how much at the most: registers and bytes of scratch of a lane.
SPILLS = {"paged_attention_wide_256_f32": (34, 140), "paged_attention_wide_256_f16": (8, 36), "paged_attention_wide_256_bf16": (8, 36)}


@pytest.mark.parametrize("path", [f[:-len("isa")] + "notes.json" for f in FILES if os.path.basename(f).startswith(("paged_", "qk_"))],
                         ids=os.path.basename)
def test_what_the_sequence_cache_kernels_spill(path):
    with open(path) as f:
        for k in json.load(f):
            registers, scratch = SPILLS.get(k["name"], (0, 0))
            assert k["vgpr_spill_count"] <= registers and k["private_segment_bytes"] <= scratch, k["name"]
