"""Matrix instructions and LDS reads written in assembly, of which the compiler knows
neither what they read nor when it is there: checked in the machine code that was built.
No device is needed."""

import re

import pytest

from device_code import kernels, registers

WANTED = ("mx4_tile_kernel", "mx4_dx_kernel")


@pytest.fixture(scope="module")
def code(tmp_path_factory):
    k = kernels(str(tmp_path_factory.mktemp("code")), WANTED)
    assert sum("mx4_tile_kernel" in n for n in k) == 4 and sum("mx4_dx_kernel" in n for n in k) == 3
    return k


def vector_writes(op, args):
    """The VGPRs that a vector ALU instruction writes."""
    if not op.startswith("v_") or op.startswith(("v_mfma", "v_cmp", "v_readfirstlane", "v_readlane",
                                                 "v_accvgpr_write", "v_nop")):
        return set()
    writes = registers(args[0], "v")
    return writes | registers(args[1], "v") if "swap" in op else writes


def test_mfma_operands_two_wait_states_after_their_writes(code):
    """An MFMA reads a VGPR at the earliest two wait states after a vector ALU
    instruction wrote it."""
    for name, body in code.items():
        last, now, count = {}, 0, 0                       # the state after which a register was written
        for op, args in body:
            if op.startswith("v_mfma"):
                count += 1
                for a in args[1:]:
                    for r in registers(a.split()[0], "v"):
                        gap = now - last.get(r, -8)
                        assert gap >= 2, f"{name}: {op} {', '.join(args)} reads v{r} {gap} states after its write"
            for r in vector_writes(op, args):
                last[r] = now + 1
            now += 1 + (int(args[0], 0) if op == "s_nop" else 0)
        assert count >= 16, name


def accumulators(op, args):
    """The AGPRs that an instruction names, as (written, read)."""
    named = [registers(a.split()[0], "a") for a in args if a]
    if op.startswith(("ds_write", "global_store", "buffer_store", "scratch_store", "flat_store")):
        return set(), set().union(*named)
    return (named[0] if named else set()), set().union(*named[1:])


def test_accumulators_are_the_matrix_instructions_until_they_are_read(code):
    """From the first MFMA to the last read, in the order of the code, nothing but an MFMA
    writes an accumulator; the first read is eighteen wait states after the last MFMA."""
    for name, body in code.items():
        mfma = [i for i, (op, _) in enumerate(body) if op.startswith("v_mfma")]
        mine = set().union(*(accumulators(*body[i])[0] for i in mfma))
        assert mine == set(range(len(mine))), name         # a0 up
        reads = [i for i, b in enumerate(body) if b[0] == "v_accvgpr_read_b32" and accumulators(*b)[1] & mine]
        # each is read: by every one of the three ways out (bf16, fp16, and through LDS)
        assert len(reads) == 3 * len(mine), name
        assert reads[0] > mfma[-1], name
        states = sum(1 + (int(args[0], 0) if op == "s_nop" else 0) for op, args in body[mfma[-1] + 1:reads[0]])
        assert states >= 18, f"{name}: read {states} states after the last MFMA"
        for i in range(mfma[0] + 1, len(body)):
            op, args = body[i]
            if not op.startswith("v_mfma") and (i < reads[-1]):
                written = accumulators(op, args)[0] & mine
                assert not written, f"{name}: {op} {', '.join(args)} writes an accumulator"


def after_wait(state, args):
    """The LDS operations still in flight after an s_waitcnt."""
    text = " ".join(args)
    left = re.search(r"lgkmcnt\((\d+)\)", text)
    if left:
        return state[max(0, len(state) - int(left[1])):]
    return state if re.search("vmcnt|expcnt", text) else ()


def test_nothing_touches_a_register_that_an_lds_read_has_still_to_write(code):
    """Along every path: an instruction that names the target of an LDS read comes after
    a wait for that read."""
    for name, body in code.items():
        index = {op.at: i for i, op in enumerate(body)}
        seen, open_ = set(), [(0, ())]
        while open_:
            i, state = open_.pop()
            while i < len(body) and (i, state) not in seen:
                seen.add((i, state))
                assert len(seen) < 40 * len(body), f"{name}: too many paths"
                op, args = body[i]
                named = set().union(*(registers(w, "v") for a in args for w in a.split()))
                for target in state:
                    assert not named & target, f"{name}: {op} {', '.join(args)} before its LDS read's wait"
                if op == "s_waitcnt":
                    state = after_wait(state, args)
                elif op.startswith("ds_read"):
                    state += (frozenset(registers(args[0], "v")),)
                elif op.startswith(("ds_", "s_load")):
                    state += (frozenset(),)
                if body[i].target is not None and op != "s_branch":
                    open_.append((index[body[i].target], state))
                if op == "s_endpgm":
                    break
                i = index[body[i].target] if op == "s_branch" else i + 1
