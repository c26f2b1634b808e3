"""Writes of the vector units to registers that a matrix product still has in hand, in the built library's gfx950 code (no GPU).

A product writes its result some cycles after it was issued, and reads the sum that it adds to while it goes on.  An ordinary
vector instruction that writes a register of the result before then is overtaken by it, and one that writes a register of the sum
changes it: both need wait states between, as reads of the result do (test_compiled_products_cpu.py), and where branches
lead around products the compiler can miss them in the same way."""
import os

import pytest

from test_compiled_products_cpu import OBJDUMP, _code, _registers, _successors, _uses

# Wait states between a product and a vector instruction that writes its result (4 passes and 3 more, 8 and 2) or its sum
# (float32 products have read that when they are issued).
RESULT = {"v_mfma_f32_16x16x32_bf16": 7, "v_mfma_f32_16x16x4_f32": 10}
SUM = {"v_mfma_f32_16x16x32_bf16": 3, "v_mfma_f32_16x16x4_f32": 0}


def _overtaken(code):
    """(products, vector writes that come too soon after one on some way)."""
    index = {at: i for i, (at, _) in enumerate(code)}
    uses = [_uses(op) for _, op in code]
    products, bad = 0, []
    for i, (_, op) in enumerate(code):
        if not op.startswith("v_mfma"):
            continue
        products += 1
        name = op.split()[0]
        for registers, need in ((uses[i][2], RESULT[name]), (_registers(op.split(", ")[3]) - uses[i][2], SUM[name])):
            ways, seen = [(j, 0, frozenset(registers)) for j in _successors(code, index, i)], {}
            while ways:
                j, waited, live = ways.pop()
                if not live or waited >= need or seen.get((j, live), need) <= waited:
                    continue
                seen[j, live] = waited
                words = code[j][1].split()
                writes = uses[j][2]
                if words[0].startswith("v_mfma"):
                    live = live - writes  # (products wait for each other)
                elif words[0].startswith("v_") and writes & live:
                    bad.append((op, code[j][1], waited))
                    continue
                waited += 1 + (int(words[1]) if words[0] == "s_nop" else 0)
                ways += [(k, waited, live) for k in _successors(code, index, j)]
    return products, bad


@pytest.mark.skipif(not os.path.exists(OBJDUMP), reason="no llvm-objdump")
def test_no_register_of_a_product_is_written_while_it_has_it(tmp_path):
    total = 0
    for kernel, code in _code(tmp_path):
        products, bad = _overtaken(code)
        total += products
        assert not bad, (kernel, bad[:4])
    assert total > 0


def test_the_search_itself():
    def code(*ops):
        return [(4 * i, op) for i, op in enumerate(ops)]
    mul, write = "v_mfma_f32_16x16x32_bf16 v[0:3], v[8:11], v[12:15], v[4:7]", "v_mov_b32_e32 v3, 0"
    assert _overtaken(code(mul, "s_nop 6", write, "s_endpgm"))[1] == []
    assert len(_overtaken(code(mul, "s_nop 5", write, "s_endpgm"))[1]) == 1
    assert len(_overtaken(code(mul, write, "s_endpgm"))[1]) == 1
    assert len(_overtaken(code(mul, "s_cbranch_vccnz 1", "s_nop 7", write, "s_endpgm"))[1]) == 1  # around the wait
    assert _overtaken(code(mul, "v_mov_b32_e32 v9, 0", "s_endpgm"))[1] == []  # a factor: read when it was issued
    assert len(_overtaken(code(mul, "s_nop 1", "v_mov_b32_e32 v5, 0", "s_endpgm"))[1]) == 1  # the sum
    assert _overtaken(code(mul, "s_nop 2", "v_mov_b32_e32 v5, 0", "s_endpgm"))[1] == []
    again = "v_mfma_f32_16x16x32_bf16 v[0:3], v[8:11], v[12:15], v[0:3]"
    assert len(_overtaken(code(again, again, "s_nop 5", write, "s_endpgm"))[1]) == 1  # of the second
