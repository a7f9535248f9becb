"""Matrix instructions written in assembly, of which the compiler knows neither what they
read nor when: checked in the machine code that was built.  No device is needed."""

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
