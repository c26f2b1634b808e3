"""Waits between matrix products and what reads their results, in the built library's gfx950 code (no GPU).

A result of a v_mfma instruction may not be read by another kind of instruction, nor as a factor of another product, for some
cycles, and the compiler counts them.  Where branches lead around products it has missed the shortest way: a state's
copies were emitted two instructions after the product, and read the sums of before.  So every way through the code, from
each product to each use, is followed here."""
import os
import re
import shutil
import subprocess

import pytest

from rl_triton import _native

OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"
# The waits that the compiler itself leaves in code without branches: 4 passes and 4 more, 8 passes and 2 more.
WAITS = {"v_mfma_f32_16x16x32_bf16": 8, "v_mfma_f32_16x16x4_f32": 10}


def _code(tmp_path):
    """(kernel, [(address, instruction)]) of every kernel with a product in it."""
    lib = shutil.copy(_native.library_path(), tmp_path / "lib.so")
    subprocess.run([OBJDUMP, "--offloading", str(lib)], check=True, stdout=subprocess.DEVNULL)
    for part in sorted(tmp_path.glob("lib.so.*gfx950")):
        out = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", str(part)], check=True, capture_output=True, text=True).stdout
        if "v_mfma" not in out:
            continue
        for m in re.finditer(r"^[0-9a-f]+ <(_ZN\S+)>:\n((?:(?!^[0-9a-f]+ <_ZN).*\n)*)", out, re.M):
            if "v_mfma" in m[2]:
                lines = re.findall(r"^\s+(\S.*?)\s*// ([0-9A-F]+):", m[2], re.M)
                yield m[1], [(int(at, 16), op) for op, at in lines]


def _registers(text):
    found = set()
    for kind, lo, hi, one, n in re.findall(r"\b([va])\[(\d+):(\d+)\]|\b([va])(\d+)\b", text):
        found |= {(kind, i) for i in range(int(lo), int(hi) + 1)} if kind else {(one, int(n))}
    return found


def _uses(op):
    """(registers read other than as the sum of a product, registers read as one, registers written)."""
    name, _, rest = op.partition(" ")
    args = rest.split(", ")
    if name.startswith("v_mfma"):
        return _registers(args[1]) | _registers(args[2]), _registers(args[3]), _registers(args[0])
    if name.startswith(("global_store", "ds_write", "buffer_store", "scratch_store", "global_atomic")):
        return _registers(rest), set(), set()
    if name.startswith(("v_", "global_load", "ds_", "buffer_load", "scratch_load")):
        reads = _registers(", ".join(args[1:]))
        if name.startswith(("v_fmac", "v_dot2c", "v_swap")):
            reads |= _registers(args[0])
        return reads, set(), _registers(args[0])
    return set(), set(), set()


def _successors(code, index, i):
    at, op = code[i]
    name = op.split()[0]
    if name == "s_endpgm":
        return []
    out = []
    if name.startswith(("s_branch", "s_cbranch")):
        offset = int(op.split()[1])
        out.append(index[at + 4 + 4 * (offset - 65536 if offset >= 32768 else offset)])
    if not name.startswith("s_branch") and i + 1 < len(code):
        out.append(i + 1)
    return out


def _early(code):
    """Reads of a product's result that come too soon after it on some way."""
    index = {at: i for i, (at, _) in enumerate(code)}
    products, bad = 0, []
    uses = [_uses(op) for _, op in code]
    for i, (_, op) in enumerate(code):
        if not op.startswith("v_mfma"):
            continue
        products += 1
        need = WAITS[op.split()[0]]
        ways, seen = [(j, 0, frozenset(uses[i][2])) for j in _successors(code, index, i)], {}
        while ways:
            j, waited, live = ways.pop()
            if waited >= need or seen.get((j, live), need) <= waited:
                continue
            seen[j, live] = waited
            reads, sums, writes = uses[j]
            if reads & live or (sums & live and not live <= sums):  # (a sum that goes on is forwarded)
                bad.append((op, code[j][1], waited))
                continue
            live = live - writes
            name = code[j][1].split()
            waited += 1 + (int(name[1]) if name[0] == "s_nop" else 0)
            if live:
                ways += [(k, waited, live) for k in _successors(code, index, j)]
    return products, bad


@pytest.mark.skipif(not os.path.exists(OBJDUMP), reason="no llvm-objdump")
def test_no_result_is_read_before_it_is_there(tmp_path):
    total = 0
    for kernel, code in _code(tmp_path):
        products, bad = _early(code)
        total += products
        assert not bad, (kernel, bad[:4])
    assert total > 0


def test_the_search_itself():
    def code(*ops):
        return [(4 * i, op) for i, op in enumerate(ops)]
    mul, read = "v_mfma_f32_16x16x32_bf16 v[0:3], v[8:11], v[12:15], v[0:3]", "v_mul_f32_e32 v5, v6, v3"
    assert _early(code(mul, "s_nop 7", read, "s_endpgm"))[1] == []
    assert len(_early(code(mul, "s_nop 6", read, "s_endpgm"))[1]) == 1
    assert len(_early(code(mul, "s_cbranch_vccnz 1", "s_nop 7", read, "s_endpgm"))[1]) == 1  # around the wait
    assert len(_early(code(read, "s_nop 0", mul, "s_branch 65532", "s_endpgm"))[1]) == 1  # back to an earlier use
    assert _early(code(mul, "v_mov_b32_e32 v3, 0", read, "s_endpgm"))[1] == []  # written anew
    assert _early(code(mul, mul, "s_nop 7", read, "s_endpgm"))[1] == []  # a sum that goes on
    assert len(_early(code(mul, "v_mfma_f32_16x16x32_bf16 v[4:7], v[0:3], v[12:15], v[4:7]", "s_endpgm"))[1]) == 1
