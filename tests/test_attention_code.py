"""What the compiler made of the loop of attention's gradient by keys.

Its matrix instructions are written in assembly, so the compiler adds no wait states between them and what
it schedules around them.  Taken as it lies and once round, and with its forward branches taken or not: a
matrix instruction reads no register that a vector instruction wrote fewer than two wait states before; nothing
but a matrix instruction that adds to it touches a result sooner than 11 wait states after the instruction that
wrote it (eight passes); nothing goes through scratch memory; and a load reads no scalar register that a vector
instruction wrote fewer than five wait states before."""
from __future__ import annotations

import os
import re
import subprocess

import pytest

from slideformer_amd import build
from test_ops_code import _operands, _registers
from test_ops_code_loops import _scalars, _states

KERNEL = re.compile(r"^(_ZN12_GLOBAL__N_1\S*14grad_kv_kernel\S*):", re.M)


def _paths(lines):
    """The loop's instructions with every forward branch falling through, and with every one taken."""
    labels = {x[:-1]: k for k, x in enumerate(lines) if x.endswith(":")}
    through, k = [], 0
    while k < len(lines):
        x = lines[k]
        through.append(x)
        if x.startswith(("s_cbranch", "s_branch")) and labels.get(_operands(x)[-1], -1) > k:
            k = labels[_operands(x)[-1]]
        else:
            k += 1
    return [[x for x in path if not x.endswith(":")] for path in (lines, through)]


@pytest.fixture(scope="module")
def loops(tmp_path_factory):
    """{kernel: the lines of its loop, labels among them}"""
    out = tmp_path_factory.mktemp("code") / "attention_grad.s"
    flags = [f for f in build.BASE_FLAGS if f not in ("-shared", "-fPIC", "-Wall")]
    subprocess.run([build.hipcc(), *flags, "--cuda-device-only", "-S", "-I",
                    os.path.join(build.REPO_DIR, "include"), "-o", str(out),
                    os.path.join(build.CSRC, "attention_grad.hip")], check=True, capture_output=True)
    text = out.read_text()
    found = {}
    for m in KERNEL.finditer(text):
        lines = [x.split(";")[0].strip() for x in text[m.end():text.index(".Lfunc_end", m.end())].splitlines()]
        lines = [x for x in lines if x and (not x.startswith(".") or x.endswith(":"))]
        labels = {x[:-1]: k for k, x in enumerate(lines) if x.endswith(":")}
        best = None
        for k, x in enumerate(lines):
            if x.startswith(("s_cbranch", "s_branch")) and labels.get(_operands(x)[-1], k) < k:
                at = labels[_operands(x)[-1]]
                if sum(y.startswith("v_mfma") for y in lines[at:k]) >= 60 and (best is None or k - at < len(best)):
                    best = lines[at:k + 1]
        found[m[1]] = best
    return found


def _hazards(body):
    wrong, code = [], body + body[:40]
    for k, line in enumerate(body):
        if line.startswith("scratch"):
            wrong.append((line, "scratch memory"))
        if not line.startswith("v_"):
            continue
        operands = _operands(line)
        written = _registers(operands[0])
        states = 0
        for after in code[k + 1:k + 30]:
            if states >= 11:
                break
            touched = [_registers(x) for x in _operands(after)] if after.startswith(("v_", "ds_", "buffer_", "global_")) else []
            if line.startswith("v_mfma"):
                if after.startswith("v_mfma"):
                    # it may add to the same sums, all of them, and nothing else
                    if written & (touched[1] | touched[2]) or written & (touched[0] | touched[3]) and \
                            not (touched[0] == written and touched[3] in (written, set())):
                        wrong.append((line, after))
                elif any(written & t for t in touched):
                    wrong.append((line, after))
            elif states < 2 and after.startswith("v_mfma") and written & set().union(*touched[1:]):
                wrong.append((line, after))
            elif states < 5 and after.startswith("buffer_load") and _scalars(operands[0]) & \
                    set().union(*(_scalars(x.split()[0]) for x in _operands(after))):
                wrong.append((line, after))
            states += _states(after)
    return wrong


@pytest.mark.slow
def test_the_loop_needs_no_wait_states_that_it_has_not(loops):
    assert len(loops) == 4, sorted(loops)                    # two types, heads of 64 and of 128
    for name, body in loops.items():
        assert body, name
        for path in _paths(body):
            assert sum(x.startswith("v_mfma") for x in path) in (64, 128), name
            assert not _hazards(path), (name, _hazards(path)[:5])


def test_the_checks_find_what_they_look_for():
    product = "v_mfma_f32_32x32x16_bf16 a[0:15], v[0:3], v[4:7], a[0:15]"
    score = "v_mfma_f32_32x32x16_bf16 v[16:31], v[0:3], a[32:35], 0"
    more = "v_mfma_f32_32x32x16_bf16 v[16:31], v[8:11], a[36:39], v[16:31]"
    quiet = ["s_nop 15", "s_nop 15"]
    assert not _hazards([score, more, product, *quiet])
    assert not _hazards(["v_mov_b32_e32 v4, v40", "s_nop 1", product, *quiet])
    assert _hazards(["v_mov_b32_e32 v4, v40", "s_nop 0", product, *quiet])
    assert not _hazards([score, "s_nop 10", "v_exp_f32_e32 v16, v16", *quiet])
    assert _hazards([score, "s_nop 9", "v_exp_f32_e32 v50, v16", *quiet])
    assert _hazards([product, "v_accvgpr_read_b32 v50, a3", *quiet])
    assert _hazards([score, "ds_read_b128 v[16:19], v60", *quiet])
    assert _hazards([score, "v_mfma_f32_32x32x16_bf16 a[0:15], v[16:19], v[4:7], a[0:15]", *quiet])
    assert _hazards(["scratch_load_dword v1, off, off", *quiet])
    assert _hazards(["v_readfirstlane_b32 s4, v1", "s_nop 3", "buffer_load_dwordx4 v1, s[4:7], 0 offen lds", *quiet])
    assert not _hazards(["v_readfirstlane_b32 s4, v1", "s_nop 4", "buffer_load_dwordx4 v1, s[4:7], 0 offen lds", *quiet])
    loop = [".L0:", "a", "s_cbranch_vccz .L1", "b", ".L1:", "c", "s_branch .L0"]
    assert _paths(loop) == [["a", "s_cbranch_vccz .L1", "b", "c", "s_branch .L0"], ["a", "s_cbranch_vccz .L1", "c", "s_branch .L0"]]


@pytest.mark.slow
def test_attention_keeps_its_rows_in_registers(tmp_path):
    """No kernel of the forward pass has scratch memory, and those of heads of 64 let three waves on a SIMD."""
    out = tmp_path / "attention.s"
    flags = [f for f in build.BASE_FLAGS if f not in ("-shared", "-fPIC", "-Wall")]
    subprocess.run([build.hipcc(), *flags, "--cuda-device-only", "-S", "-I",
                    os.path.join(build.REPO_DIR, "include"), "-o", str(out),
                    os.path.join(build.CSRC, "attention.hip")], check=True, capture_output=True)
    text = out.read_text()
    kernels = re.findall(r"\.amdhsa_kernel (\S+)(.*?)\.end_amdhsa_kernel", text, re.S)
    assert len(kernels) == 13, [name for name, _ in kernels]     # two types, two sizes, three kernels; the copy into chunks
    for name, fields in kernels:
        got = {k: int(v) for k, v in re.findall(r"\.amdhsa_(private_segment_fixed_size|next_free_vgpr) (\d+)", fields)}
        assert got["private_segment_fixed_size"] == 0, name
        if "16attention_kernel" in name and "Li64" in name:
            assert got["next_free_vgpr"] <= 168, name            # 512 for three, in eights
