"""What the compiler made of the matrix products' loops, once round: from each loop's last
instructions to its first, where the text of the generated code has them apart.

The same holds there as inside: the matrix instructions are written in assembly, and so are the
loads into LDS, so nothing adds wait states to either.  A matrix instruction reads no
register that a vector instruction wrote fewer than two wait states before; sums are
touched by nothing else in the loop; and a load reads no scalar register that a vector
instruction wrote fewer than five wait states before."""
from __future__ import annotations

import os
import re
import subprocess

import pytest

from slideformer_amd import build
from test_ops_code import KERNEL, _operands, _registers


@pytest.fixture(scope="module")
def loops(tmp_path_factory):
    """{kernel: the instructions of its loop of matrix instructions}"""
    out = tmp_path_factory.mktemp("code") / "linear_loss.s"
    flags = [f for f in build.BASE_FLAGS if f not in ("-shared", "-fPIC", "-Wall")]
    subprocess.run([build.hipcc(), *flags, "--cuda-device-only", "-S", "-I",
                    os.path.join(build.REPO_DIR, "include"), "-o", str(out),
                    os.path.join(build.CSRC, "linear_loss.hip")], check=True, capture_output=True)
    text = out.read_text()
    found = {}
    for m in KERNEL.finditer(text):
        lines = [x.split(";")[0].strip() for x in text[m.end():text.index(".Lfunc_end", m.end())].splitlines()]
        lines = [x for x in lines if x and (not x.startswith(".") or x.endswith(":"))]
        labels = {x[:-1]: k for k, x in enumerate(lines) if x.endswith(":")}
        for k, x in enumerate(lines):
            if not x.startswith(("s_cbranch", "s_branch")):
                continue
            body = lines[labels[_operands(x)[-1]] + 1:k + 1]
            # the loop is one block without another label; blocks that lie elsewhere branch back over it
            if any(y.startswith("v_mfma") for y in body) and not any(y.endswith(":") for y in body):
                assert m[1] not in found, m[1]
                found[m[1]] = body
    return found


def _scalars(operand):
    m = re.fullmatch(r"s\[(\d+):(\d+)\]", operand)
    if m:
        return set(range(int(m[1]), int(m[2]) + 1))
    m = re.fullmatch(r"s(\d+)", operand)
    return {int(m[1])} if m else set()


def _states(line):
    return int(line.split()[1], 0) + 1 if line.startswith("s_nop") else 1


def _hazards(body):
    """What is wrong in a loop's instructions, taken twice in a row."""
    wrong = []
    sums = set().union(*(_registers(_operands(x)[0]) for x in body if x.startswith("v_mfma")))
    code = body + body[:12]
    for k, line in enumerate(body):
        if line.startswith("scratch"):
            wrong.append((line, "scratch memory"))
        if not line.startswith("v_") or line.startswith("v_mfma"):
            continue
        operands = _operands(line)
        if sums & set().union(*map(_registers, operands)):
            wrong.append((line, "a sum"))
        vector, scalar, states = _registers(operands[0]), _scalars(operands[0]), 0
        for after in code[k + 1:k + 8]:
            if after.startswith("v_mfma") and states < 2 and vector & set().union(*map(_registers, _operands(after)[1:4])):
                wrong.append((line, after))
            if after.startswith("buffer_load") and states < 5 and \
                    scalar & set().union(*(_scalars(x.split()[0]) for x in _operands(after))):
                wrong.append((line, after))
            states += _states(after)
    return wrong


@pytest.mark.slow
def test_matrix_loops_need_no_wait_states_once_round(loops):
    assert len(loops) == 16, sorted(loops)                   # 2 types, 2 sides; two types of the matrix's gradient
    for name, body in loops.items():
        assert body[-1].startswith(("s_cbranch", "s_branch")), name
        assert sum(x.startswith("v_mfma") for x in body) in (32, 128), name
        assert not _hazards(body), name


def test_hazards_are_seen():
    """The check itself, on code that has each of them."""
    product, load = "v_mfma_f32_16x16x32_bf16 a[0:3], v[4:7], v[8:11], a[0:3]", "buffer_load_dwordx4 v1, s[4:7], 0 offen lds"
    assert not _hazards([product, "v_add_u32 v4, v1, v2", "s_nop 0", "s_nop 0", "s_cbranch_scc1 x"])
    assert _hazards([product, "s_nop 0", "v_add_u32 v5, v1, v2"])           # only once round
    assert _hazards(["v_add_u32 v5, v1, v2", product])
    assert _hazards([product, "v_accvgpr_write_b32 a2, v1"])
    assert _hazards([product, load, "s_nop 2", "v_readfirstlane_b32 s5, v1"])
    assert not _hazards([product, load, "v_readfirstlane_b32 s5, v1", "s_nop 4"])
