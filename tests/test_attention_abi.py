"""CPU checks of the attention's and rotation's entry points: their structs are laid out as the header's, and bad
arguments are refused before any launch.  No kernel is launched here."""
from __future__ import annotations

import ctypes
import os
import shutil
import subprocess

import numpy as np
import pytest
import torch

from slideformer_amd import _lib, _ops_lib, ops

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HOST = np.zeros(1 << 12, np.uint8)
HP = HOST.ctypes.data + (-HOST.ctypes.data) % 256
BF16, F16, F32, I32, I64, I8 = _lib.LA_BF16, _lib.LA_F16, _lib.LA_F32, _ops_lib.LA_I32, _ops_lib.LA_I64, _ops_lib.LA_I8
OK, EINVAL, EDTYPE, EFAULT = _lib.LA_OK, _lib.LA_EINVAL, _lib.LA_EDTYPE, _lib.LA_EFAULT


@pytest.mark.parametrize("mirror,name", [(_ops_lib.LaHeads, "la_heads_t"), (_ops_lib.LaAttention, "la_attention_t"),
                                         (_ops_lib.LaRotary, "la_rotary_t")])
def test_structs_match_the_header(tmp_path, mirror, name):
    """Field offsets of the ctypes mirrors against a C compiler's."""
    gcc = shutil.which("gcc")
    assert gcc, "gcc not found"
    names = [f[0] for f in mirror._fields_]
    src = tmp_path / "s.c"
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "model_ops.h"\nint main(void) {\n' +
                   "".join(f'    printf("%zu ", offsetof({name}, {n}));\n' for n in names) +
                   f'    printf("%zu", sizeof({name}));\n    return 0;\n}}\n')
    exe = tmp_path / "s"
    subprocess.run([gcc, "-std=c11", "-Wall", "-Werror", "-pedantic", "-I", os.path.join(REPO, "include"), str(src),
                    "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [getattr(mirror, n).offset for n in names] + [ctypes.sizeof(mirror)]


def _heads(data=HP, **strides):
    return _ops_lib.LaHeads(data=data, batch_stride=strides.get("batch", 256), row_stride=strides.get("row", 128),
                            head_stride=strides.get("head", 64))


def _attention(**changed):
    fields = dict(dtype=BF16, batch=2, rows=4, key_rows=4, heads=2, kv_heads=1, dim=64, causal=1, scale=0.125,
                  index_dtype=I32)
    fields.update({name: _heads() for name in ("q", "k", "v", "out", "lse", "grad_out", "grad_q", "grad_k", "grad_v")})
    fields.update(changed)
    return _ops_lib.LaAttention(**fields)


@pytest.mark.parametrize("changed,code", [
    (dict(dtype=F32), EDTYPE),
    (dict(dtype=I8), EDTYPE),
    (dict(lengths=HP, index_dtype=BF16), EDTYPE),
    (dict(batch=0), EINVAL),
    (dict(heads=3, kv_heads=2), EINVAL),
    (dict(kv_heads=0), EINVAL),
    (dict(heads=0), EINVAL),
    (dict(dim=0), EINVAL),
    (dict(dim=129), EINVAL),
    (dict(rows=(1 << 30) + 1), EINVAL),
    (dict(rows=1 << 29), EINVAL),                            # times batch and heads
    (dict(key_rows=1 << 30), EINVAL),
    (dict(scale=0.0), EINVAL),
    (dict(scale=-1.0), EINVAL),
    (dict(scale=float("inf")), EINVAL),
    (dict(scale=float("nan")), EINVAL),
    (dict(causal=0, window=4), EINVAL),
    (dict(starts=HP, lengths=HP), EINVAL),
    (dict(key_starts=HP), EINVAL),
    (dict(starts=HP, key_rows=5), EINVAL),                   # without key_starts they have the queries'
    (dict(lengths=HP + 2), EINVAL),
    (dict(lengths=HP + 4, index_dtype=I64), EINVAL),
    (dict(q=_heads(None)), EINVAL),
    (dict(q=_heads(HP + 1)), EINVAL),
    (dict(k=_heads(None)), EINVAL),
    (dict(out=_heads(HP + 1)), EINVAL),
    (dict(lse=_heads(None)), EINVAL),
    (dict(lse=_heads(HP + 2)), EINVAL),
    (dict(), EFAULT),                                        # host memory
    (dict(starts=HP, key_starts=HP, key_rows=9), EFAULT),
])
@pytest.mark.parametrize("name", ["la_attention", "la_attention_grad"])
def test_attention_refusals(name, changed, code):
    L = _ops_lib.load()
    assert getattr(L, name)(ctypes.byref(_attention(**changed)), HP, 1 << 40, None) == code
    assert getattr(L, name)(None, HP, 1 << 40, None) == EINVAL


def test_attention_grad_refusals():
    L = _ops_lib.load()
    for field in ("grad_out", "grad_q", "grad_k", "grad_v"):
        for pointer in (None, HP + 1):
            assert L.la_attention_grad(ctypes.byref(_attention(**{field: _heads(pointer)})), HP, 1 << 40, None) == EINVAL
    good = _attention()
    need = L.la_attention_grad_workspace(ctypes.byref(good))
    assert need > 0
    assert L.la_attention_grad(ctypes.byref(good), HP, need - 1, None) == EINVAL
    assert L.la_attention_grad(ctypes.byref(good), None, need, None) == EINVAL
    assert L.la_attention_grad(ctypes.byref(good), HP + 16, 1 << 40, None) == EINVAL


def test_attention_workspaces():
    """Nothing where rows lie in whole chunks and fill the card; copies of what does not; partial results of few rows."""
    L = _ops_lib.load()

    def size(**changed):
        return L.la_attention_workspace(ctypes.byref(_attention(**changed)))

    assert size() == 0
    assert size(v=_heads(HP + 2)) == 2 * 4 * 64 * 2          # one head of keys
    assert size(q=_heads(head=65)) == 2 * 4 * 2 * 64 * 2
    assert size(dim=60) == 2 * 4 * (2 + 1 + 1) * 64 * 2      # rounded up to a multiple of eight
    parts = size(rows=1, key_rows=8192)
    assert parts % (2 * 2 * 65 * 4) < 256 and 2 <= parts // (2 * 2 * 65 * 4) <= 64
    assert size(rows=1, key_rows=300) == 0
    assert size(dtype=F32) == 0
    assert L.la_attention_workspace(None) == 0
    call = _attention(rows=1, key_rows=8192)
    assert L.la_attention(ctypes.byref(call), HP, parts - 1, None) == EINVAL


@pytest.mark.parametrize("causal", [0, 1])
@pytest.mark.parametrize("rows,key_rows", [(4096, 0), (0, 4096), (4096, 1), (1, 4096), (4096, 4096)])
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_workspaces_of_any_lengths(causal, rows, key_rows, dim):
    """The rows' statistics, and partial results of keys; packed sequences that may all be empty among them."""
    L = _ops_lib.load()
    for packed in (dict(), dict(starts=HP, key_starts=HP, batch=1 << 20)):
        call = _attention(causal=causal, rows=rows, key_rows=key_rows, dim=dim, **packed)
        L.la_attention_workspace(ctypes.byref(call))
        flat = rows * (1 if packed else 2)
        assert L.la_attention_grad_workspace(ctypes.byref(call)) >= 2 * flat * 2 * 4


def test_attention_of_nothing():
    L = _ops_lib.load()
    none = _heads(None)
    call = _attention(rows=0, q=none, out=none, lse=none)
    assert L.la_attention(ctypes.byref(call), None, 0, None) == OK


def _rotary(**changed):
    fields = dict(dtype=BF16, n=3, heads=2, kv_heads=1, dim=64, rotated=64, q_weight=HP, k_weight=HP, eps=1e-6, cos=HP,
                  sin=HP, positions=8, at_dtype=I64, at=HP, weight_grad_dtype=BF16, grad_q_weight=HP, grad_k_weight=HP)
    fields.update({name: _heads() for name in ("q", "k", "q_out", "k_out", "grad_q", "grad_k")})
    fields.update(changed)
    return _ops_lib.LaRotary(**fields)


@pytest.mark.parametrize("changed,code", [
    (dict(dtype=I8), EDTYPE),
    (dict(at_dtype=BF16), EDTYPE),
    (dict(dim=0), EINVAL),
    (dict(dim=257), EINVAL),
    (dict(rotated=66), EINVAL),
    (dict(rotated=31), EINVAL),
    (dict(n=1 << 30), EINVAL),                               # times heads
    (dict(q=_heads(None)), EINVAL),
    (dict(q=_heads(HP + 1)), EINVAL),
    (dict(k_out=_heads(None)), EINVAL),
    (dict(q_weight=HP + 1), EINVAL),
    (dict(cos=None), EINVAL),
    (dict(sin=HP + 2), EINVAL),
    (dict(at=HP + 4), EINVAL),
    (dict(), EFAULT),
])
def test_rotary_refusals(changed, code):
    L = _ops_lib.load()
    call = _rotary(**changed)
    assert L.la_qk_norm_rotary(ctypes.byref(call), None) == code
    assert L.la_qk_norm_rotary_grad(ctypes.byref(call), HP, 1 << 40, None) == code
    assert L.la_qk_norm_rotary(None, None) == EINVAL
    assert L.la_qk_norm_rotary_grad(None, HP, 1 << 40, None) == EINVAL


def test_rotary_grad_refusals():
    L = _ops_lib.load()

    def code(work=HP, size=1 << 40, **changed):
        return L.la_qk_norm_rotary_grad(ctypes.byref(_rotary(**changed)), work, size, None)

    need = L.la_qk_norm_rotary_grad_workspace(ctypes.byref(_rotary()))
    assert need > 0
    assert L.la_qk_norm_rotary_grad_workspace(ctypes.byref(_rotary(q_weight=None, k_weight=None))) == 0
    assert code(weight_grad_dtype=F16) == EDTYPE
    assert code(grad_q_weight=None) == EINVAL
    assert code(grad_k_weight=HP + 1) == EINVAL
    assert code(grad_q=_heads(None)) == EINVAL
    assert code(size=need - 1) == EINVAL
    assert code(work=None) == EINVAL
    assert code(q=_heads(None), k=_heads(None), q_weight=None, k_weight=None) == EFAULT   # its inputs are not needed then
    none = _heads(None)
    assert L.la_qk_norm_rotary(ctypes.byref(_rotary(n=0, q=none, k=none, q_out=none, k_out=none)), None) == OK


def test_python_refusals():
    x = torch.zeros(3, 2, 64, dtype=torch.bfloat16)
    table, starts = torch.zeros(8, 32), torch.tensor([0, 3])
    lse = torch.zeros(3, 2)
    for call in (lambda: ops.qk_norm_rotary(x, x, table, table),
                 lambda: ops.qk_norm_rotary_grad(x, x, x, x, table, table),
                 lambda: ops.attention(x, x, x, starts=starts), lambda: ops.attention(x[None], x[None], x[None]),
                 lambda: ops.attention_grad(x, x, x, x, x, lse, starts=starts)):
        with pytest.raises(RuntimeError, match="expected a HIP device"):
            call()
    with pytest.raises(RuntimeError, match="three dimensions"):
        ops.attention(x[0], x[0], x[0], starts=starts)
    with pytest.raises(RuntimeError, match="needs q, which was normed"):
        ops.qk_norm_rotary_grad(x, x, None, x, table, table, q_weight=torch.zeros(64, dtype=torch.bfloat16))
