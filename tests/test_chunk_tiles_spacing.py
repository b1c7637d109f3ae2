"""The kernel of chunk attention for many rows spells its matrix instructions out (chunk_tiles.hip), where the compiler inserts no wait states: in the built
code nothing else may touch a result, and no vector instruction may write an operand, closer than the hardware allows."""
import re
import shutil
import subprocess

import pytest

from tests.test_matrix_instruction_spacing import TOOLS, _code_object, _functions

PASSES = 8           # of 4 cycles, of an instruction of 32 x 32 x 16: the next one that the matrix unit takes starts that much later
RESULT = 12          # wait states from one to a read or write of its result by another kind of instruction, or as a first or second factor
SAME = 2             # ... to the next one that accumulates into the same registers
OPERAND = 2          # ... from a vector instruction that writes an operand


def _registers(text):
    """Vector registers and accumulation registers (numbered from 1000) in an operand text."""
    found = set()
    for kind, one, low, high in re.findall(r"\b([av])(?:(\d+)|\[(\d+):(\d+)\])", text):
        base = 1000 if kind == "a" else 0
        found |= {base + int(one)} if one else set(range(base + int(low), base + int(high) + 1))
    return found


def _following(function, places, index, states):
    """Instructions that can follow `index` with fewer than so many wait states between, over branches."""
    todo, best = [(index, 0)], {}
    while todo:
        at, passed = todo.pop()
        _, name, operands, target = function[at]
        if at != index:
            passed += 1 + int(operands, 0) if name == "s_nop" else PASSES if name.startswith("v_mfma") else 1
        if passed >= states or (at != index and best.get(at, states) <= passed):
            continue
        best[at] = passed
        follow = [] if name in ("s_branch", "s_endpgm") or at + 1 == len(function) else [at + 1]
        for following in follow + ([] if target is None else [places[target]]):
            # (a matrix instruction that follows one starts only when the first one's passes are over)
            ahead = PASSES - 1 if function[following][1].startswith("v_mfma") and function[index][1].startswith("v_mfma") else 0
            yield following, max(passed, ahead)
            todo.append((following, passed))


@pytest.mark.skipif(not shutil.which("llvm-objdump", path=str(TOOLS)), reason="needs the ROCm LLVM tools")
def test_spelled_out_matrix_instructions_keep_their_distance(tmp_path):
    elf = _code_object(b"chunk_tiles_kernel", tmp_path)
    listing = subprocess.run([TOOLS / "llvm-objdump", "-d", "--mcpu=gfx950", elf], check=True, capture_output=True, text=True).stdout
    seen = 0
    for name, function in _functions(listing).items():
        if "chunk_tiles_kernel" not in name or ".kd" in name:
            continue
        places = {entry[0]: i for i, entry in enumerate(function)}
        inline = 0
        for i, (_, op, operands, _) in enumerate(function):
            if op.startswith("v_mfma"):
                inline += 1
                assert op in ("v_mfma_f32_32x32x16_f16", "v_mfma_f32_32x32x16_bf16"), op
                result = _registers(operands.split(", ")[0])
                assert len(result) == 16, operands
                for j, passed in _following(function, places, i, RESULT):
                    other, parts = function[j], function[j][2].split(", ")
                    if other[1].startswith("v_mfma"):
                        again = _registers(parts[0])
                        assert not result & _registers(", ".join(parts[1:3])), (name, operands, other)
                        assert again == result or not again & result, (name, operands, other)
                        assert again != result or passed >= SAME, (name, operands, other)
                    else:
                        assert not result & _registers(other[2]), (name, hex(function[i][0]), operands, other)
            elif op.startswith("v_") and not op.startswith(("v_cmp", "v_readfirstlane", "v_readlane")):
                written = _registers(", ".join(operands.split(", ")[:2]) if "swap" in op else operands.split(", ")[0])
                for j, _ in _following(function, places, i, OPERAND):
                    if function[j][1].startswith("v_mfma"):
                        assert not written & _registers(function[j][2]), (name, function[i], function[j])
        assert inline > 0, name
        seen += 1
    assert seen == 4
