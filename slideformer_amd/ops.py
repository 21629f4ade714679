"""The operators at a language model's two ends, on MI355X.

What lies outside the decoder layers of the model whose layers ``LayerAdam``
steps: the embedding matrix, the norms, and the vocabulary matrix with the loss.

``embedding`` / ``embedding_grad``            rows of a matrix by token, and the matrix's gradient
``rms_norm`` / ``rms_norm_8bit`` / ``rms_norm_grad``   the residual's addition and the norm over it
``linear_cross_entropy`` / ``linear_cross_entropy_grad``  the loss, a tile of scores at a time; with its gradients,
                                              a piece of the rows' softmax at a time

Gradients are explicit calls, as a layer-by-layer runtime makes them: each writes
into the tensor that the optimizer reads, a slice of a flat grad buffer for
instance, and with ``accumulate=True`` adds to what is there (a second
micro-batch, or the other use of tied weights).  Nothing is recorded for autograd:
outputs never require grad, whatever the inputs do.

Matrices have two dimensions; ``embedding`` of tokens [batch, length] returns
[batch, length, hidden], whose ``flatten(0, 1)`` the other calls take.

All tensors live on one HIP device.  Calls are asynchronous on the current
stream, or on ``stream``; results of one call belong to that stream.  Rows may be
any distance apart (a view of a wider matrix), their elements are contiguous.
Nothing is copied to the host, so what only the device can see raises no error:
an out-of-range token gives a row of NaN, an out-of-range target a NaN loss.
The kernels are in ``libslideformer_amd_ops.so`` (C-ABI ``include/model_ops.h``);
there is no fallback.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch

from . import _lib, _ops_lib
from .layer_adam import _on_device, _raw_current_stream, _stream_handle, _torch_stream

__all__ = ["embedding", "embedding_grad", "rms_norm", "rms_norm_8bit", "rms_norm_grad", "linear_cross_entropy",
           "linear_cross_entropy_grad", "PIECE_BYTES"]

_FLOAT = {torch.float32: _lib.LA_F32, torch.bfloat16: _lib.LA_BF16, torch.float16: _lib.LA_F16}
_TOKEN = {torch.int32: _ops_lib.LA_I32, torch.int64: _ops_lib.LA_I64}
_EIGHT = {torch.int8: _ops_lib.LA_I8, torch.float8_e4m3fn: _ops_lib.LA_F8E4M3}

# How much memory linear_cross_entropy_grad takes by default for the softmax of the
# rows it works on at a time, in 16 bits: 1 GiB, 4096 rows of a 128256-token vocabulary.
PIECE_BYTES = 1 << 30


def _check(rc: int, what: str) -> None:
    _ops_lib.load()
    _lib.check(rc, what)


def _matrix(t: torch.Tensor, name: str, device, hidden: Optional[int] = None, rows: Optional[int] = None,
            dtype=None) -> int:
    """Check a matrix of contiguous rows; returns the distance of its rows in elements."""
    if t.device != device or not t.is_cuda:
        raise RuntimeError(f"{name} on {t.device}, expected a HIP device"
                           + (f" ({device})" if device.type == "cuda" else ""))
    if t.dim() != 2:
        raise RuntimeError(f"{name} must have two dimensions, got {tuple(t.shape)}")
    if hidden is not None and t.shape[1] != hidden or rows is not None and t.shape[0] != rows:
        raise RuntimeError(f"size mismatch: {name} is {tuple(t.shape)}, expected "
                           f"({'any' if rows is None else rows}, {'any' if hidden is None else hidden})")
    if dtype is not None and t.dtype != dtype:
        raise RuntimeError(f"{name} is {t.dtype}, expected {dtype}")
    if t.dtype not in _FLOAT:
        raise RuntimeError(f"unsupported dtype of {name}: {t.dtype}")
    if t.numel() == 0 or t.shape[0] == 1 and t.shape[1] == 1:
        return t.shape[1]
    if t.shape[1] > 1 and t.stride(1) != 1 or t.shape[0] > 1 and t.stride(0) < t.shape[1]:
        raise RuntimeError(f"the rows of {name} must be contiguous")
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _vector(t: torch.Tensor, name: str, device, size: int, dtypes) -> None:
    if t.device != device:
        raise RuntimeError(f"{name} on {t.device}, expected {device}")
    if t.numel() != size:
        raise RuntimeError(f"size mismatch: {name} has {t.numel()} elements, expected {size}")
    if not t.is_contiguous():
        raise RuntimeError(f"{name} must be contiguous")
    if t.dtype not in dtypes:
        raise RuntimeError(f"unsupported dtype of {name}: {t.dtype}")


def _here():
    """(current device, its current stream's handle), what the native host module takes."""
    device = torch.cuda.current_device()
    return device, _stream_handle(None, torch.device("cuda", device)) if _raw_current_stream is None \
        else _raw_current_stream(device)


def _got(result, what: str):
    """What the native host module returned: outputs, or a code of the library's."""
    if type(result) is int:
        _check(result, what)
    return result


class _Scratch:
    """Allocations of one call, made on its stream so that the caching allocator
    orders their reuse after it."""

    def __init__(self, device, stream):
        self.device = device
        self.guard = None
        if stream is not None:
            self.guard = torch.cuda.stream(_torch_stream(stream, device))
        self.handle = _stream_handle(stream, device)

    def __enter__(self):
        if self.guard is not None:
            self.guard.__enter__()
        return self

    def __exit__(self, *exc):
        if self.guard is not None:
            self.guard.__exit__(*exc)

    def empty(self, shape, dtype):
        return torch.empty(shape, dtype=dtype, device=self.device)

    def workspace(self, size):
        # torch's blocks are aligned to 512 bytes
        return torch.empty(max(1, size), dtype=torch.uint8, device=self.device)


# ---------------------------------------------------------------------------
# embedding
# ---------------------------------------------------------------------------
def embedding(tokens: torch.Tensor, weight: torch.Tensor, *, scale: float = 1.0,
              out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """``scale * weight[tokens]``: [*tokens.shape, hidden] in weight's type, rounded once.

    tokens: int32 or int64; one outside [0, vocab) gives a row of NaN.  ``out``: a
    matrix [tokens.numel(), hidden] to write instead of a new tensor."""
    if out is None and stream is None and tokens.is_cuda:
        done = _ops_lib.calls().embedding(tokens, weight, scale, *_here())
        if done is not None:
            return _got(done, "la_embedding")
    stride = _matrix(weight, "weight", weight.device)
    vocab, hidden = weight.shape
    _vector(tokens, "tokens", weight.device, tokens.numel(), _TOKEN)
    n = tokens.numel()
    with _on_device(weight.device), _Scratch(weight.device, stream) as s:
        if out is None:
            out = s.empty((*tokens.shape, hidden), weight.dtype)
            out_stride = hidden
        else:
            out_stride = _matrix(out, "out", weight.device, hidden, n, weight.dtype)
        _check(_ops_lib.load().la_embedding(_TOKEN[tokens.dtype], tokens.data_ptr(), n, _FLOAT[weight.dtype],
                                            weight.data_ptr(), vocab, hidden, stride, scale, out.data_ptr(),
                                            out_stride, s.handle), "la_embedding")
    return out


def embedding_grad(tokens: torch.Tensor, grad_out: torch.Tensor, grad_weight: torch.Tensor, *, scale: float = 1.0,
                   padding_idx: Optional[int] = None, accumulate: bool = False, stream=None) -> torch.Tensor:
    """The gradient of ``embedding`` towards its matrix, into ``grad_weight``.

    ``grad_out``: [tokens.numel(), hidden] (or [*tokens.shape, hidden]).  Every row
    of ``grad_weight`` (grad_out's type or float32) is written: ``scale`` times the sum of its
    token's rows, zeros for tokens that do not occur; with ``accumulate`` the sums
    are added to what is there and other rows stay untouched.  ``padding_idx`` (a token;
    a negative one is none, and is not counted from the end as torch does) and
    out-of-range tokens contribute nothing.  Sums are fp32 in a fixed order: equal
    calls give equal bits."""
    if stream is None and tokens.is_cuda:
        done = _ops_lib.calls().embedding_grad(tokens, grad_out, grad_weight, scale,
                                               -1 if padding_idx is None else padding_idx, accumulate, *_here())
        if done is not None:
            return _got(done, "la_embedding_grad")
    device = grad_weight.device
    stride = _matrix(grad_weight, "grad_weight", device)
    vocab, hidden = grad_weight.shape
    _vector(tokens, "tokens", device, tokens.numel(), _TOKEN)
    n = tokens.numel()
    if grad_out.dim() != 2:
        if grad_out.shape != (*tokens.shape, hidden):
            raise RuntimeError(f"size mismatch: grad_out is {tuple(grad_out.shape)}, expected "
                               f"{(*tokens.shape, hidden)}")
        grad_out = grad_out.view(n, hidden)
    grad_stride = _matrix(grad_out, "grad_out", device, hidden, n)
    if grad_weight.dtype not in (grad_out.dtype, torch.float32):
        raise RuntimeError(f"grad_weight is {grad_weight.dtype}, expected {grad_out.dtype} or torch.float32")
    lib = _ops_lib.load()
    with _on_device(device), _Scratch(device, stream) as s:
        size = lib.la_embedding_grad_workspace(n, vocab, hidden)
        work = s.workspace(size)
        _check(lib.la_embedding_grad(_TOKEN[tokens.dtype], tokens.data_ptr(), n, _FLOAT[grad_out.dtype],
                                     grad_out.data_ptr(), grad_stride, _FLOAT[grad_weight.dtype],
                                     grad_weight.data_ptr(), vocab, hidden, stride, scale,
                                     -1 if padding_idx is None else padding_idx, int(accumulate), work.data_ptr(),
                                     size, s.handle), "la_embedding_grad")
    return grad_weight


# ---------------------------------------------------------------------------
# root-mean-square norm
# ---------------------------------------------------------------------------
def _norm_inputs(x, weight, residual):
    device = x.device
    x_stride = _matrix(x, "x", device)
    n, hidden = x.shape
    _vector(weight, "weight", device, hidden, (x.dtype,))
    r_stride = hidden if residual is None else _matrix(residual, "residual", device, hidden, n, x.dtype)
    return device, n, hidden, x_stride, r_stride


def rms_norm(x: torch.Tensor, weight: torch.Tensor, *, eps: float = 1e-6, residual: Optional[torch.Tensor] = None,
             stream=None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``z = x + residual``; ``out = z / sqrt(mean(z^2) + eps) * weight`` over each row.

    x, residual: [n, hidden]; weight: [hidden]; all of one type.  Returns
    ``(out, z, rstd)``: z (x itself without a residual) is what the next residual
    takes, and it and the fp32 ``rstd`` [n] are what ``rms_norm_grad`` takes.  The norm
    is that of the unrounded sum."""
    if stream is None and x.is_cuda:
        done = _ops_lib.calls().rms_norm(x, weight, eps, residual, *_here())
        if done is not None:
            return _got(done, "la_rms_norm")
    device, n, hidden, x_stride, r_stride = _norm_inputs(x, weight, residual)
    with _on_device(device), _Scratch(device, stream) as s:
        out = s.empty((n, hidden), x.dtype)
        summed = None if residual is None else s.empty((n, hidden), x.dtype)
        rstd = s.empty((n,), torch.float32)
        code = _FLOAT[x.dtype]
        _check(_ops_lib.load().la_rms_norm(
            code, x.data_ptr(), x_stride, None if residual is None else residual.data_ptr(), r_stride,
            weight.data_ptr(), n, hidden, eps, None if summed is None else summed.data_ptr(), hidden, code,
            out.data_ptr(), hidden, None, rstd.data_ptr(), s.handle), "la_rms_norm")
    return out, x if summed is None else summed, rstd


def rms_norm_8bit(x: torch.Tensor, weight: torch.Tensor, *, eps: float = 1e-6,
                  residual: Optional[torch.Tensor] = None, dtype: torch.dtype = torch.int8,
                  stream=None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``rms_norm`` with its output in 8 bits and one scale for each row.

    Returns ``(out, scales, z)``: ``out[i] * scales[i]`` stands for the norm's row i, with
    ``scales[i] = max|row| / 127`` (``torch.int8``) or ``/ 448`` (``torch.float8_e4m3fn``).  A row
    of zeros has scale 0; one that holds an infinity or NaN has scale NaN."""
    if dtype not in _EIGHT:
        raise RuntimeError(f"unsupported 8-bit dtype: {dtype}")
    if stream is None and x.is_cuda:
        done = _ops_lib.calls().rms_norm_8bit(x, weight, eps, residual, dtype is not torch.int8, *_here())
        if done is not None:
            return _got(done, "la_rms_norm")
    device, n, hidden, x_stride, r_stride = _norm_inputs(x, weight, residual)
    with _on_device(device), _Scratch(device, stream) as s:
        out = s.empty((n, hidden), dtype)
        scales = s.empty((n,), torch.float32)
        summed = None if residual is None else s.empty((n, hidden), x.dtype)
        _check(_ops_lib.load().la_rms_norm(
            _FLOAT[x.dtype], x.data_ptr(), x_stride, None if residual is None else residual.data_ptr(), r_stride,
            weight.data_ptr(), n, hidden, eps, None if summed is None else summed.data_ptr(), hidden, _EIGHT[dtype],
            out.data_ptr(), hidden, scales.data_ptr(), None, s.handle), "la_rms_norm")
    return out, scales, x if summed is None else summed


def rms_norm_grad(grad_out: torch.Tensor, summed: torch.Tensor, rstd: torch.Tensor, weight: torch.Tensor, *,
                  grad_summed: Optional[torch.Tensor] = None, grad_weight: Optional[torch.Tensor] = None,
                  accumulate: bool = False, stream=None) -> Tuple[torch.Tensor, torch.Tensor]:
    """The gradients of ``rms_norm`` towards z (that is, towards x and the residual) and weight.

    ``grad_summed``: the gradient that reaches z past the norm, through the next
    residual; it is added.  ``grad_weight``: the tensor [hidden] to write (weight's type
    or float32; new by default), added to with ``accumulate``.  Returns
    ``(grad_x, grad_weight)``.  Sums are fp32 in a fixed order."""
    if stream is None and grad_out.is_cuda:
        done = _ops_lib.calls().rms_norm_grad(grad_out, summed, rstd, weight, grad_summed, grad_weight, accumulate,
                                              *_here())
        if done is not None:
            return _got(done, "la_rms_norm_grad")
    device = grad_out.device
    go_stride = _matrix(grad_out, "grad_out", device)
    n, hidden = grad_out.shape
    dtype = grad_out.dtype
    z_stride = _matrix(summed, "summed", device, hidden, n, dtype)
    _vector(rstd, "rstd", device, n, (torch.float32,))
    _vector(weight, "weight", device, hidden, (dtype,))
    gs_stride = hidden if grad_summed is None else _matrix(grad_summed, "grad_summed", device, hidden, n, dtype)
    if grad_weight is not None:
        _vector(grad_weight, "grad_weight", device, hidden, (dtype, torch.float32))
    elif accumulate:
        raise RuntimeError("accumulate needs a grad_weight to add to")
    lib = _ops_lib.load()
    with _on_device(device), _Scratch(device, stream) as s:
        grad_x = s.empty((n, hidden), dtype)
        if grad_weight is None:
            grad_weight = s.empty((hidden,), dtype)
        size = lib.la_rms_norm_grad_workspace(n, hidden)
        work = s.workspace(size)
        _check(lib.la_rms_norm_grad(
            _FLOAT[dtype], grad_out.data_ptr(), go_stride, summed.data_ptr(), z_stride, rstd.data_ptr(),
            weight.data_ptr(), None if grad_summed is None else grad_summed.data_ptr(), gs_stride, n, hidden,
            grad_x.data_ptr(), hidden, _FLOAT[grad_weight.dtype], grad_weight.data_ptr(), int(accumulate),
            work.data_ptr(), size, s.handle), "la_rms_norm_grad")
    return grad_x, grad_weight


# ---------------------------------------------------------------------------
# loss
# ---------------------------------------------------------------------------
def _loss_call(x, weight, targets, ignore_index, reduction, allowed):
    if reduction not in allowed:
        raise RuntimeError(f"reduction must be one of {', '.join(allowed)}, got {reduction!r}")
    device = weight.device
    weight_stride = _matrix(weight, "weight", device)
    vocab, hidden = weight.shape
    x_stride = _matrix(x, "x", device, hidden, dtype=weight.dtype)
    if weight.dtype == torch.float32:
        raise RuntimeError("unsupported dtype of weight: torch.float32 (bfloat16 or float16)")
    if vocab == 0 or hidden == 0:
        raise RuntimeError(f"weight is empty: {tuple(weight.shape)}")
    _vector(targets, "targets", device, x.shape[0], (torch.int64,))
    call = _ops_lib.LaLinearLoss(
        dtype=_FLOAT[weight.dtype], x=x.data_ptr(), n=x.shape[0], hidden=hidden, x_stride=x_stride,
        weight=weight.data_ptr(), vocab=vocab, weight_stride=weight_stride, targets=targets.data_ptr(),
        ignore_index=ignore_index, mean=int(reduction == "mean"))
    return device, call


def _run_loss(lib, call, s):
    size = lib.la_linear_loss_workspace(ctypes.byref(call))
    work = s.workspace(size)
    _check(lib.la_linear_loss(ctypes.byref(call), work.data_ptr(), size, s.handle), "la_linear_loss")


def linear_cross_entropy(x: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, *, ignore_index: int = -100,
                         reduction: str = "mean", stream=None) -> torch.Tensor:
    """Softmax cross entropy of ``x @ weight.T`` against ``targets``, forward only.

    x: [n, hidden], weight: [vocab, hidden], bfloat16 or float16; targets: int64 [n].
    Rows whose target is ``ignore_index`` have no loss and are never read.
    reduction: "mean" over the other rows (0 where there are none), "sum", or
    "none" for the fp32 loss of each row.  The scores exist one tile at a time."""
    device, call = _loss_call(x, weight, targets, ignore_index, reduction, ("mean", "sum", "none"))
    lib = _ops_lib.load()
    with _on_device(device), _Scratch(device, stream) as s:
        if reduction == "none":
            out = s.empty((x.shape[0],), torch.float32)
            call.row_loss = out.data_ptr()
        else:
            out = s.empty((), torch.float32)
            call.loss = out.data_ptr()
        _run_loss(lib, call, s)
    return out


def linear_cross_entropy_grad(x: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor, *,
                              ignore_index: int = -100, reduction: str = "mean",
                              grad_scale: Optional[torch.Tensor] = None,
                              grad_weight: Optional[torch.Tensor] = None, accumulate: bool = False,
                              piece_bytes: int = PIECE_BYTES,
                              stream=None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """``linear_cross_entropy`` with its gradients: ``(loss, grad_x, grad_weight)``.

    The loss is where backward begins, so one call does both: ``grad_x`` is what
    the last norm's ``rms_norm_grad`` takes.  ``grad_scale``: one fp32 on the device that scales
    both gradients, not the loss (a loss scale, or one over the micro-batches).
    ``grad_weight``: the matrix to write (weight's type or float32; new by default), added to
    with ``accumulate``.  ``piece_bytes``: about how much memory the softmax of the rows in
    work may take, in 16 bits (at least 256 rows).  Beside it the call takes up to half as much
    again (or 64 MiB, or hidden fp32 values for each of these rows, if that is more) for partial
    sums of grad_x, and a copy of the trained rows of x.  Where not all rows fit, grad_weight is
    summed over the pieces in fp32, two passes over it a piece: in place if it is of float32, else in
    a buffer of 4 bytes an element.  Where that buffer takes more than the pieces save, all
    rows are worked on at once, so a smaller ``piece_bytes`` never takes more memory."""
    device, call = _loss_call(x, weight, targets, ignore_index, reduction, ("mean", "sum"))
    vocab, hidden = weight.shape
    if grad_weight is not None:
        stride = _matrix(grad_weight, "grad_weight", device, hidden, vocab)
        if grad_weight.dtype not in (weight.dtype, torch.float32):
            raise RuntimeError(f"grad_weight is {grad_weight.dtype}, expected {weight.dtype} or torch.float32")
    elif accumulate:
        raise RuntimeError("accumulate needs a grad_weight to add to")
    if grad_scale is not None:
        _vector(grad_scale, "grad_scale", device, 1, (torch.float32,))
        call.grad_scale = grad_scale.data_ptr()
    lib = _ops_lib.load()
    with _on_device(device), _Scratch(device, stream) as s:
        loss = s.empty((), torch.float32)
        grad_x = s.empty((x.shape[0], hidden), x.dtype)
        if grad_weight is None:
            grad_weight = s.empty((vocab, hidden), weight.dtype)
            stride = hidden
        call.loss, call.grads, call.accumulate = loss.data_ptr(), 1, int(accumulate)
        call.grad_x, call.grad_x_stride = grad_x.data_ptr(), hidden
        call.grad_weight, call.grad_weight_stride = grad_weight.data_ptr(), stride
        call.grad_weight_dtype = _FLOAT[grad_weight.dtype]
        call.piece_rows = min(max(256, piece_bytes // (2 * vocab) // 256 * 256), 1 << 22)
        _run_loss(lib, call, s)
    return loss, grad_x, grad_weight
