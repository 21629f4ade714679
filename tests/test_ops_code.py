"""What the compiler made of the matrix products' loops.

Their matrix instructions are written in assembly, so the compiler adds no wait
states between them and what it schedules around them.  The source leaves it no
reason to: fragments come from LDS, and sums stay in their registers.  This compiles
the kernels and holds the generated code to that: no vector ALU instruction writes a
register that a matrix instruction reads fewer than two instructions later, none
touches a sum inside the loop, and nothing there goes through scratch memory."""
from __future__ import annotations

import os
import re
import subprocess

import pytest

from slideformer_amd import build

KERNEL = re.compile(r"^(_ZN12_GLOBAL__N_1\S*(?:13scores_kernel|13grad_x_kernel|18grad_weight_kernel)\S*):", re.M)


def _registers(operand):
    m = re.fullmatch(r"([va])\[(\d+):(\d+)\]", operand)
    if m:
        return {(m[1], k) for k in range(int(m[2]), int(m[3]) + 1)}
    m = re.fullmatch(r"([va])(\d+)", operand)
    return {(m[1], int(m[2]))} if m else set()


def _operands(line):
    parts = line.split(None, 1)
    return [x.strip() for x in parts[1].split(",")] if len(parts) > 1 else []


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    out = tmp_path_factory.mktemp("code") / "linear_loss.s"
    flags = [f for f in build.BASE_FLAGS if f not in ("-shared", "-fPIC", "-Wall")]
    subprocess.run([build.hipcc(), *flags, "--cuda-device-only", "-S", "-I",
                    os.path.join(build.REPO_DIR, "include"), "-o", str(out),
                    os.path.join(build.CSRC, "linear_loss.hip")], check=True, capture_output=True)
    text = out.read_text()
    found = {}
    for m in KERNEL.finditer(text):
        lines = [x.split(";")[0].strip() for x in text[m.end():text.index("s_endpgm", m.end())].splitlines()]
        found[m[1]] = [x for x in lines if x and not x.startswith(".") and not x.endswith(":")]
    return found


@pytest.mark.slow
def test_matrix_loops_need_no_wait_states(kernels):
    assert len(kernels) == 16, sorted(kernels)      # 2 types, 2 sides; two types of the matrix's gradient
    for name, code in kernels.items():
        products = [k for k, x in enumerate(code) if x.startswith("v_mfma")]
        assert len(products) in (32, 128), (name, len(products))
        sums = set().union(*(_registers(_operands(code[k])[0]) for k in products))
        assert {kind for kind, _ in sums} == {"a"}, name
        for k in range(products[0] - 8, products[-1]):
            line = code[k]
            assert not line.startswith("scratch"), (name, line)
            if not line.startswith("v_") or line.startswith(("v_mfma", "v_cmp", "v_readfirstlane")):
                continue
            written = _registers(_operands(line)[0])
            if k > products[0]:
                assert not sums & set().union(*map(_registers, _operands(line))), (name, line)
            states = 0
            for after in code[k + 1:k + 4]:
                if after.startswith("v_mfma"):
                    read = set().union(*map(_registers, _operands(after)[1:4]))
                    assert states >= 2 or not written & read, (name, line, after)
                states += int(after.split()[1], 0) + 1 if after.startswith("s_nop") else 1
