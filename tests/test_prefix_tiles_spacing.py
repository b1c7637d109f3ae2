"""The kernel of a shared prefix's tiles spells its matrix instructions out like that of attention of new tokens (test_chunk_tiles_spacing.py): the same distances hold in
the built code."""
import shutil
import subprocess

import pytest

from tests.test_chunk_tiles_spacing import OPERAND, RESULT, SAME, _following, _registers
from tests.test_matrix_instruction_spacing import TOOLS, _code_object, _functions


@pytest.mark.skipif(not shutil.which("llvm-objdump", path=str(TOOLS)), reason="needs the ROCm LLVM tools")
def test_spelled_out_matrix_instructions_keep_their_distance(tmp_path):
    elf = _code_object(b"prefix_tiles_kernel", tmp_path)
    listing = subprocess.run([TOOLS / "llvm-objdump", "-d", "--mcpu=gfx950", elf], check=True, capture_output=True, text=True).stdout
    seen = 0
    for name, function in _functions(listing).items():
        if "prefix_tiles_kernel" not in name or ".kd" in name:
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
