"""CPU checks of the model operators' library: it exports what its header declares,
and refuses bad arguments before any launch.  No kernel is launched here."""
from __future__ import annotations

import ctypes
import os
import re

import numpy as np
import pytest
import torch

from slideformer_amd import _lib, _ops_lib, ops

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(REPO, "include", "model_ops.h")


def _header():
    with open(HEADER) as f:
        return f.read()


def test_header_binding_and_library_agree():
    declared = sorted(set(re.findall(r"^\s*(?:int|uint64_t)\s+(la_\w+)\s*\(", _header(), re.M)))
    assert declared == sorted(_ops_lib.EXPORTED)
    L = _ops_lib.load()
    for name in declared:
        assert hasattr(L, name), name
    assert L.la_ops_abi_version() == _ops_lib.ABI_VERSION
    for name in ("LA_OPS_ABI_VERSION", "LA_I32", "LA_I64", "LA_I8", "LA_F8E4M3"):
        value = int(re.search(rf"#define {name} (\d+)", _header()).group(1))
        assert value == (_ops_lib.ABI_VERSION if name == "LA_OPS_ABI_VERSION" else getattr(_ops_lib, name))


def test_loss_struct_matches_the_header(tmp_path):
    """Field offsets of the ctypes mirror against a C compiler's."""
    import shutil
    import subprocess
    gcc = shutil.which("gcc")
    assert gcc, "gcc not found"
    names = [f[0] for f in _ops_lib.LaLinearLoss._fields_]
    src = tmp_path / "s.c"
    src.write_text('#include <stdio.h>\n#include "model_ops.h"\nint main(void) {\n' +
                   "".join(f'    printf("%zu ", offsetof(la_linear_loss_t, {n}));\n' for n in names) +
                   '    printf("%zu", sizeof(la_linear_loss_t));\n    return 0;\n}\n')
    exe = tmp_path / "s"
    subprocess.run([gcc, "-std=c11", "-Wall", "-Werror", "-pedantic", "-I", os.path.join(REPO, "include"), str(src),
                    "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [getattr(_ops_lib.LaLinearLoss, n).offset for n in names] + [ctypes.sizeof(_ops_lib.LaLinearLoss)]


HOST = np.zeros(1 << 14, np.uint8)
HP = HOST.ctypes.data + (-HOST.ctypes.data) % 256


def test_embedding_refusals():
    L = _ops_lib.load()
    I64, F32, BF16 = _ops_lib.LA_I64, _lib.LA_F32, _lib.LA_BF16
    f = L.la_embedding
    assert f(_lib.LA_F32, HP, 4, F32, HP, 4, 8, 8, 1.0, HP, 8, None) == _lib.LA_EDTYPE
    assert f(I64, HP, 4, _ops_lib.LA_I8, HP, 4, 8, 8, 1.0, HP, 8, None) == _lib.LA_EDTYPE
    assert f(I64, None, 4, F32, HP, 4, 8, 8, 1.0, HP, 8, None) == _lib.LA_EINVAL
    assert f(I64, HP + 4, 4, F32, HP, 4, 8, 8, 1.0, HP, 8, None) == _lib.LA_EINVAL      # int64 at 4 bytes
    assert f(I64, HP, 4, F32, HP + 2, 4, 8, 8, 1.0, HP, 8, None) == _lib.LA_EINVAL
    assert f(I64, HP, 4, F32, HP, 4, 8, 7, 1.0, HP, 8, None) == _lib.LA_EINVAL          # rows overlap
    assert f(I64, HP, 4, F32, HP, 1 << 31, 8, 8, 1.0, HP, 8, None) == _lib.LA_EINVAL
    assert f(I64, HP, 4, F32, HP, 4, 8, 8, 1.0, HP, 8, None) == _lib.LA_EFAULT          # host memory
    assert f(I64, None, 0, F32, None, 4, 8, 8, 1.0, None, 8, None) == _lib.LA_OK        # nothing to do
    g = L.la_embedding_grad
    need = L.la_embedding_grad_workspace(4, 4, 8)
    assert need > 0
    assert g(I64, HP, 4, F32, HP, 8, BF16, HP, 4, 8, 8, 1.0, -1, 0, HP, need, None) == _lib.LA_EDTYPE
    assert g(I64, HP, 4, F32, HP, 8, F32, HP, 4, 8, 8, 1.0, -1, 0, HP, need - 1, None) == _lib.LA_EINVAL
    assert g(I64, HP, 4, F32, HP, 8, F32, HP, 4, 8, 8, 1.0, -1, 0, None, need, None) == _lib.LA_EINVAL
    assert g(I64, HP, 4, F32, HP, 8, F32, None, 4, 8, 8, 1.0, -1, 0, HP, need, None) == _lib.LA_EINVAL
    assert g(I64, HP, 4, F32, HP, 8, F32, HP, 4, 8, 8, 1.0, -1, 0, HP, need, None) == _lib.LA_EFAULT
    assert g(I64, None, 0, F32, None, 8, F32, None, 0, 8, 8, 1.0, -1, 0, None, 0, None) == _lib.LA_OK


def test_rms_norm_refusals():
    L = _ops_lib.load()
    F32, BF16, I8 = _lib.LA_F32, _lib.LA_BF16, _ops_lib.LA_I8
    f = L.la_rms_norm
    assert f(I8, HP, 8, None, 8, HP, 2, 8, 1e-6, None, 8, I8, HP, 8, HP, None, None) == _lib.LA_EDTYPE
    assert f(F32, HP, 8, None, 8, HP, 2, 8, 1e-6, None, 8, BF16, HP, 8, None, None, None) == _lib.LA_EDTYPE
    assert f(F32, None, 8, None, 8, HP, 2, 8, 1e-6, None, 8, F32, HP, 8, None, None, None) == _lib.LA_EINVAL
    assert f(F32, HP, 7, None, 8, HP, 2, 8, 1e-6, None, 8, F32, HP, 8, None, None, None) == _lib.LA_EINVAL
    assert f(F32, HP, 8, None, 8, HP, 2, 8, 1e-6, None, 8, I8, HP, 8, None, None, None) == _lib.LA_EINVAL  # no scales
    assert f(F32, HP, 8, None, 8, HP, 1 << 25, 8, 1e-6, None, 8, F32, HP, 8, None, None, None) == _lib.LA_EINVAL
    assert f(F32, HP, 8, None, 8, HP, 2, 8, 1e-6, None, 8, F32, HP, 8, None, None, None) == _lib.LA_EFAULT
    assert f(F32, None, 8, None, 8, None, 0, 8, 1e-6, None, 8, F32, None, 8, None, None, None) == _lib.LA_OK
    g = L.la_rms_norm_grad
    need = L.la_rms_norm_grad_workspace(2, 8)
    assert need > 0
    assert g(F32, HP, 8, HP, 8, HP, HP, None, 8, 2, 8, HP, 8, BF16, HP, 0, HP, need, None) == _lib.LA_EDTYPE
    assert g(F32, HP, 8, HP, 8, HP, HP, None, 8, 2, 8, HP, 8, F32, HP, 0, HP, need - 1, None) == _lib.LA_EINVAL
    assert g(F32, HP, 8, HP, 8, None, HP, None, 8, 2, 8, HP, 8, F32, HP, 0, HP, need, None) == _lib.LA_EINVAL
    assert g(F32, HP, 8, HP, 8, HP, HP, None, 8, 2, 8, HP, 8, F32, HP, 0, HP, need, None) == _lib.LA_EFAULT
    assert g(F32, HP, 8, HP, 8, HP, HP, None, 8, 2, 0, HP, 8, F32, None, 0, None, 0, None) == _lib.LA_OK


def _loss_call(**changed):
    fields = dict(dtype=_lib.LA_BF16, x=HP, n=4, hidden=8, x_stride=8, weight=HP, vocab=16, weight_stride=8, targets=HP,
                  ignore_index=-100, mean=1, loss=HP, row_loss=None, grads=1, grad_scale=None, grad_x=HP,
                  grad_x_stride=8, grad_weight_dtype=_lib.LA_BF16, grad_weight=HP, grad_weight_stride=8, accumulate=0,
                  piece_rows=256)
    fields.update(changed)
    return _ops_lib.LaLinearLoss(**fields)


@pytest.mark.parametrize("changed,code", [
    (dict(dtype=_lib.LA_F32), _lib.LA_EDTYPE),
    (dict(grad_weight_dtype=_lib.LA_F16), _lib.LA_EDTYPE),
    (dict(vocab=0), _lib.LA_EINVAL),
    (dict(hidden=0), _lib.LA_EINVAL),
    (dict(vocab=(1 << 21) + 1), _lib.LA_EINVAL),
    (dict(n=(1 << 22) + 1), _lib.LA_EINVAL),
    (dict(weight=None), _lib.LA_EINVAL),
    (dict(weight=HP + 1), _lib.LA_EINVAL),
    (dict(x_stride=7), _lib.LA_EINVAL),
    (dict(targets=HP + 4), _lib.LA_EINVAL),
    (dict(grad_x=None), _lib.LA_EINVAL),
    (dict(grad_weight=None), _lib.LA_EINVAL),
    (dict(grad_weight_stride=7), _lib.LA_EINVAL),
    (dict(), _lib.LA_EFAULT),
])
def test_linear_loss_refusals(changed, code):
    L = _ops_lib.load()
    call = _loss_call(**changed)
    assert L.la_linear_loss(ctypes.byref(call), HP, 1 << 40, None) == code
    assert L.la_linear_loss(None, HP, 1 << 40, None) == _lib.LA_EINVAL
    good = _loss_call()
    need = L.la_linear_loss_workspace(ctypes.byref(good))
    assert need > 0
    assert L.la_linear_loss(ctypes.byref(good), HP, need - 1, None) == _lib.LA_EINVAL
    assert L.la_linear_loss(ctypes.byref(good), HP + 16, 1 << 40, None) == _lib.LA_EINVAL


def test_loss_workspace_is_bounded_by_the_piece():
    """The softmax of one piece is held, not that of the batch."""
    L = _ops_lib.load()
    sizes = [L.la_linear_loss_workspace(ctypes.byref(_loss_call(n=n, hidden=64, vocab=50257, x_stride=64,
                                                                weight_stride=64, piece_rows=1024)))
             for n in (1024, 65536)]
    one_piece = 1024 * 50432 * 2
    assert sizes[0] > one_piece
    # what grows with the rows: the gathered states, row lists; and the fp32 sum over pieces
    assert sizes[1] - sizes[0] < 65536 * (2 * 64 + 16) + 50257 * 64 * 4 + (1 << 20)
    forward = L.la_linear_loss_workspace(ctypes.byref(_loss_call(n=65536, hidden=64, vocab=50257, x_stride=64,
                                                                 weight_stride=64, grads=0)))
    assert forward < 65536 * 50257 * 2 / 100


def test_python_refusals_on_host_tensors():
    w = torch.zeros(4, 8, dtype=torch.bfloat16)
    t = torch.zeros(3, dtype=torch.int64)
    x = torch.zeros(3, 8, dtype=torch.bfloat16)
    for call in (lambda: ops.embedding(t, w), lambda: ops.embedding_grad(t, x, w),
                 lambda: ops.rms_norm(x, w[0]), lambda: ops.rms_norm_8bit(x, w[0]),
                 lambda: ops.rms_norm_grad(x, x, torch.zeros(3), w[0]),
                 lambda: ops.linear_cross_entropy(x, w, t), lambda: ops.linear_cross_entropy_grad(x, w, t)):
        with pytest.raises(RuntimeError, match="expected a HIP device"):
            call()
    with pytest.raises(RuntimeError, match="8-bit dtype"):
        ops.rms_norm_8bit(x, w[0], dtype=torch.uint8)
    with pytest.raises(RuntimeError, match="reduction"):
        ops.linear_cross_entropy(x, w, t, reduction="max")
    with pytest.raises(RuntimeError, match="reduction"):
        ops.linear_cross_entropy_grad(x, w, t, reduction="none")
