"""The operators of a language model, on MI355X.

What lies around the matrix products of the model whose layers ``LayerAdam`` steps: at
its two ends the embedding matrix, the norms, and the vocabulary matrix with the loss;
inside a decoder layer the attention.

``embedding`` / ``embedding_grad``            rows of a matrix by token, and the matrix's gradient
``rms_norm`` / ``rms_norm_8bit`` / ``rms_norm_grad``   the residual's addition and the norm over it
``qk_norm_rotary`` / ``qk_norm_rotary_grad``  the norm of each query and key head, and the rotation by position
``attention`` / ``attention_grad``            softmax attention over packed or padded sequences, or a cache
``linear_cross_entropy`` / ``linear_cross_entropy_grad``  the loss, a tile of scores at a time; with its gradients,
                                              a piece of the rows' softmax at a time

Gradients are explicit calls, as a layer-by-layer runtime makes them: each writes
into the tensor that the optimizer reads, a slice of a flat grad buffer for
instance, and with ``accumulate=True`` adds to what is there (a second
micro-batch, or the other use of tied weights).  Nothing is recorded for autograd:
outputs never require grad, whatever the inputs do.

Matrices have two dimensions; ``embedding`` of tokens [batch, length] returns
[batch, length, hidden], whose ``flatten(0, 1)`` the other calls take.  Heads are the
last two dimensions, [.., heads, dim]: a view of a projection's output
(``qkv[:, :n].unflatten(1, (heads, dim))``), or in any order of memory in which a head's elements are
contiguous.

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

__all__ = ["embedding", "embedding_grad", "rms_norm", "rms_norm_8bit", "rms_norm_grad", "qk_norm_rotary",
           "qk_norm_rotary_grad", "attention", "attention_grad", "linear_cross_entropy", "linear_cross_entropy_grad",
           "PIECE_BYTES"]

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
# heads
# ---------------------------------------------------------------------------
def _heads(t: torch.Tensor, name: str, device, dims: int, dtype=None, shape=None) -> "_ops_lib.LaHeads":
    """Check [.., heads, dim] and describe where it lies."""
    if t.device != device or not t.is_cuda:
        raise RuntimeError(f"{name} on {t.device}, expected a HIP device"
                           + (f" ({device})" if device.type == "cuda" else ""))
    if t.dim() != dims:
        raise RuntimeError(f"{name} must have {dims} dimensions, got {tuple(t.shape)}")
    if shape is not None and t.shape != shape:
        raise RuntimeError(f"size mismatch: {name} is {tuple(t.shape)}, expected {tuple(shape)}")
    if dtype is not None and t.dtype != dtype:
        raise RuntimeError(f"{name} is {t.dtype}, expected {dtype}")
    if t.dtype not in _FLOAT:
        raise RuntimeError(f"unsupported dtype of {name}: {t.dtype}")
    strides = t.stride()
    if t.numel() and t.shape[-1] > 1 and strides[-1] != 1:
        raise RuntimeError(f"the heads of {name} must be contiguous")
    return _ops_lib.LaHeads(data=t.data_ptr(), batch_stride=strides[0] if dims == 4 else 0, row_stride=strides[-3],
                            head_stride=strides[-2])


def _result(t: torch.Tensor, name: str, device, dims: int, dtype, shape) -> "_ops_lib.LaHeads":
    """The same for a tensor to write: no two of its elements may be one."""
    got = _heads(t, name, device, dims, dtype, shape)
    span = t.shape[-1]
    for stride, size in sorted((s, n) for s, n in zip(t.stride()[:-1], t.shape[:-1]) if n > 1):
        if t.numel() and stride < span:
            raise RuntimeError(f"the heads of {name} overlap: strides {t.stride()}")
        span = stride * (size - 1) + span
    return got


def _row_values(t: torch.Tensor, name: str, device, like: torch.Tensor) -> "_ops_lib.LaHeads":
    """fp32 values for every head of every row of `like`, in any order of memory."""
    if t.device != device:
        raise RuntimeError(f"{name} on {t.device}, expected {device}")
    if t.shape != like.shape[:-1]:
        raise RuntimeError(f"size mismatch: {name} is {tuple(t.shape)}, expected {tuple(like.shape[:-1])}")
    if t.dtype != torch.float32:
        raise RuntimeError(f"{name} is {t.dtype}, expected torch.float32")
    strides = t.stride()
    return _ops_lib.LaHeads(data=t.data_ptr(), batch_stride=strides[0] if t.dim() == 3 else 0, row_stride=strides[-2],
                            head_stride=strides[-1])


def _indices(t: Optional[torch.Tensor], name: str, device, size: int, dtype=None) -> Optional[int]:
    if t is None:
        return None
    _vector(t, name, device, size, _TOKEN)
    if dtype is not None and t.dtype != dtype:
        raise RuntimeError(f"{name} is {t.dtype}, expected {dtype}")
    return t.data_ptr()


def _rotary_call(q, k, like_q, like_k, cos, sin, q_weight, k_weight, positions, eps, interleaved):
    """The call without its results.  like_q, like_k: what the sizes are those of."""
    device, dtype = like_q.device, like_q.dtype
    of_q, of_k = _heads(like_q, "q", device, 3), _heads(like_k, "k", device, 3, dtype)
    n, heads, dim = like_q.shape
    if like_k.shape[0] != n or like_k.shape[2] != dim:
        raise RuntimeError(f"size mismatch: k is {tuple(like_k.shape)}, expected ({n}, any, {dim})")
    if dim > 256 or dim == 0:
        raise RuntimeError(f"heads of {dim} elements are not supported (1 to 256)")
    for t, name in ((cos, "cos"), (sin, "sin")):
        if t.device != device:
            raise RuntimeError(f"{name} on {t.device}, expected {device}")
        if t.dim() != 2 or t.shape != cos.shape or 2 * t.shape[1] > dim:
            raise RuntimeError(f"size mismatch: {name} is {tuple(t.shape)}, expected two tables [positions, pairs] of at "
                               f"most {dim // 2} pairs")
        if t.dtype != torch.float32 or not t.is_contiguous():
            raise RuntimeError(f"{name} must be a contiguous torch.float32 table, got {t.dtype}")
    call = _ops_lib.LaRotary(
        dtype=_FLOAT[dtype], n=n, heads=heads, kv_heads=like_k.shape[1], dim=dim, rotated=2 * cos.shape[1], eps=eps,
        cos=cos.data_ptr(), sin=sin.data_ptr(), positions=cos.shape[0], interleaved=int(interleaved),
        at=_indices(positions, "positions", device, n))
    if positions is not None:
        call.at_dtype = _TOKEN[positions.dtype]
    for weight, name in ((q_weight, "q_weight"), (k_weight, "k_weight")):
        if weight is not None:
            _vector(weight, name, device, dim, (dtype,))
            setattr(call, name, weight.data_ptr())
    if q is like_q:
        call.q = of_q
    elif q is not None:
        call.q = _heads(q, "q", device, 3, dtype, like_q.shape)
    if k is like_k:
        call.k = of_k
    elif k is not None:
        call.k = _heads(k, "k", device, 3, dtype, like_k.shape)
    return device, call, of_q, of_k


def _rotary_out(call, out, q, k, device, s):
    if out is None:
        out = s.empty(q.shape, q.dtype), s.empty(k.shape, k.dtype)
    call.q_out = _result(out[0], "out[0]", device, 3, q.dtype, q.shape)
    call.k_out = _result(out[1], "out[1]", device, 3, q.dtype, k.shape)
    return out


def qk_norm_rotary(q: torch.Tensor, k: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, *,
                   q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None,
                   positions: Optional[torch.Tensor] = None, eps: float = 1e-6, interleaved: bool = False,
                   out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None,
                   stream=None) -> Tuple[torch.Tensor, torch.Tensor]:
    """The root-mean-square norm of every query and key head, then the rotation by position.

    q: [n, heads, dim], k: [n, kv_heads, dim], of one type.  ``q_weight``, ``k_weight``: the
    norms' scales [dim]; without one its heads are not normed.  ``cos``, ``sin``: fp32 tables
    [positions, pairs]; the first ``2 * pairs`` elements of a head turn, (a, b) -> (a cos - b sin, b cos + a sin), pair
    j of elements (j, j + pairs), or (2 j, 2 j + 1) if ``interleaved``.  ``positions``: int32 or int64
    [n], row i of the tables for row i by default; one outside the tables makes the rotated elements NaN.
    ``out``: the two tensors to write instead of new ones: q and k themselves, each in its own place, or memory that the call
    does not read, rows of a cache for instance; not one in the other's.  All in fp32, rounded once."""
    if out is None and stream is None and q.is_cuda:
        done = _ops_lib.calls().qk_norm_rotary(q, k, cos, sin, q_weight, k_weight, positions, eps, interleaved, *_here())
        if done is not None:
            return _got(done, "la_qk_norm_rotary")
    device, call, _, _ = _rotary_call(q, k, q, k, cos, sin, q_weight, k_weight, positions, eps, interleaved)
    lib = _ops_lib.load()
    with _on_device(device), _Scratch(device, stream) as s:
        out = _rotary_out(call, out, q, k, device, s)
        _check(lib.la_qk_norm_rotary(ctypes.byref(call), s.handle), "la_qk_norm_rotary")
    return out


def qk_norm_rotary_grad(grad_q: torch.Tensor, grad_k: torch.Tensor, q: Optional[torch.Tensor],
                        k: Optional[torch.Tensor], cos: torch.Tensor, sin: torch.Tensor, *,
                        q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None,
                        positions: Optional[torch.Tensor] = None, eps: float = 1e-6, interleaved: bool = False,
                        grad_q_weight: Optional[torch.Tensor] = None, grad_k_weight: Optional[torch.Tensor] = None,
                        accumulate: bool = False, out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None, stream=None):
    """The gradients of ``qk_norm_rotary`` towards its q, k and weights, from those of its results.

    q and k are its inputs (None will do for heads that are not normed).  ``out``: where the
    gradients of q and k go, new tensors by default; ``grad_q`` and ``grad_k`` (or q and k) themselves, each in its own
    place, may be written over, nothing else that the call reads.  ``grad_q_weight``, ``grad_k_weight``: the tensors [dim] to write (of the weights' type or
    float32, both of one type, two tensors; new by default), added to with ``accumulate``.  Returns ``(grad_q, grad_k,
    grad_q_weight, grad_k_weight)``, None for a weight that there is not.  Sums are fp32 in a fixed order."""
    if grad_q_weight is None and grad_k_weight is None and not accumulate and out is None and stream is None \
            and grad_q.is_cuda:
        done = _ops_lib.calls().qk_norm_rotary_grad(grad_q, grad_k, q, k, cos, sin, q_weight, k_weight, positions, eps,
                                                    interleaved, *_here())
        if done is not None:
            return _got(done, "la_qk_norm_rotary_grad")
    for x, weight, name in ((q, q_weight, "q"), (k, k_weight, "k")):
        if x is None and weight is not None:
            raise RuntimeError(f"the gradient of a norm needs {name}, which was normed")
    device, call, call_grad_q, call_grad_k = _rotary_call(q, k, grad_q, grad_k, cos, sin, q_weight, k_weight, positions,
                                                          eps, interleaved)
    call.grad_q, call.grad_k = call_grad_q, call_grad_k
    grads = [grad_q_weight, grad_k_weight]
    for g, weight, name in ((grad_q_weight, q_weight, "grad_q_weight"), (grad_k_weight, k_weight, "grad_k_weight")):
        if g is not None:
            if weight is None:
                raise RuntimeError(f"{name} without its weight")
            _vector(g, name, device, weight.numel(), (weight.dtype, torch.float32))
        elif accumulate and weight is not None:
            raise RuntimeError(f"accumulate needs a {name} to add to")
    given = {g.dtype for g in grads if g is not None}
    if len(given) > 1:
        raise RuntimeError("grad_q_weight and grad_k_weight must be of one type")
    kind = given.pop() if given else grad_q.dtype
    lib = _ops_lib.load()
    with _on_device(device), _Scratch(device, stream) as s:
        out = _rotary_out(call, out, grad_q, grad_k, device, s)
        for i, weight in enumerate((q_weight, k_weight)):
            if weight is not None and grads[i] is None:
                grads[i] = s.empty((weight.numel(),), kind)
        call.weight_grad_dtype, call.accumulate = _FLOAT[kind], int(accumulate)
        call.grad_q_weight, call.grad_k_weight = (None if g is None else g.data_ptr() for g in grads)
        size = lib.la_qk_norm_rotary_grad_workspace(ctypes.byref(call))
        work = s.workspace(size)
        _check(lib.la_qk_norm_rotary_grad(ctypes.byref(call), work.data_ptr(), size, s.handle),
               "la_qk_norm_rotary_grad")
    return (*out, *grads)


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------
def _attention_call(q, k, v, causal, window, scale, starts, key_starts, lengths, key_lengths):
    device, dims = q.device, q.dim()
    if dims not in (3, 4):
        raise RuntimeError(f"q must have three dimensions (packed) or four (a batch), got {tuple(q.shape)}")
    of_q = _heads(q, "q", device, dims)
    of_k = _heads(k, "k", device, dims, q.dtype)
    of_v = _heads(v, "v", device, dims, q.dtype, k.shape)
    if q.dtype == torch.float32:
        raise RuntimeError("unsupported dtype of q: torch.float32 (bfloat16 or float16)")
    rows, heads, dim = q.shape[-3:]
    key_rows, kv_heads = k.shape[-3:-1]
    if k.shape[-1] != dim or dims == 4 and k.shape[0] != q.shape[0]:
        raise RuntimeError(f"size mismatch: k is {tuple(k.shape)}, expected "
                           f"({f'{q.shape[0]}, ' if dims == 4 else ''}any, any, {dim})")
    if kv_heads == 0 or heads == 0 or heads % kv_heads:
        raise RuntimeError(f"{heads} query heads cannot share {kv_heads} key heads evenly")
    if dim == 0 or dim > 128:
        raise RuntimeError(f"heads of {dim} elements are not supported (1 to 128)")
    if window is not None and (window < 1 or not causal):
        raise RuntimeError(f"window must be at least 1 and goes with causal, got {window}")
    scale = dim ** -0.5 if scale is None else float(scale)
    if not 0 < scale < float("inf"):
        raise RuntimeError(f"scale must be above 0 and finite, got {scale}")
    call = _ops_lib.LaAttention(dtype=_FLOAT[q.dtype], rows=rows, key_rows=key_rows, heads=heads, kv_heads=kv_heads,
                                dim=dim, q=of_q, k=of_k, v=of_v, causal=int(bool(causal)), window=min(window or 0, 1 << 40),
                                scale=scale)
    if dims == 3:
        if starts is None:
            raise RuntimeError("packed sequences need starts")
        if lengths is not None or key_lengths is not None:
            raise RuntimeError("lengths go with a batch (four dimensions); packed sequences have starts")
        if starts.numel() < 2:
            raise RuntimeError("starts must have an element more than there are sequences, and at least two")
        if key_starts is None and rows != key_rows:
            raise RuntimeError(f"size mismatch: {rows} queries and {key_rows} keys need key_starts")
        call.batch = starts.numel() - 1
        first = starts
        call.starts = _indices(starts, "starts", device, starts.numel())
        call.key_starts = _indices(key_starts, "key_starts", device, starts.numel(), starts.dtype)
    else:
        if starts is not None or key_starts is not None:
            raise RuntimeError("starts go with packed sequences (three dimensions); a batch has lengths")
        if key_lengths is None and lengths is not None:
            if rows != key_rows:
                raise RuntimeError(f"size mismatch: lengths of {rows} queries with {key_rows} keys need key_lengths")
            key_lengths = lengths
        call.batch = q.shape[0]
        first = lengths if lengths is not None else key_lengths
        call.lengths = _indices(lengths, "lengths", device, q.shape[0])
        call.key_lengths = _indices(key_lengths, "key_lengths", device, q.shape[0],
                                    None if lengths is None else lengths.dtype)
    if first is not None:
        call.index_dtype = _TOKEN[first.dtype]
    return device, call


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, causal: bool = True, window: Optional[int] = None,
              scale: Optional[float] = None, starts: Optional[torch.Tensor] = None,
              key_starts: Optional[torch.Tensor] = None, lengths: Optional[torch.Tensor] = None,
              key_lengths: Optional[torch.Tensor] = None, stream=None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Softmax attention: ``(out, lse)``, out like q and the fp32 log-sum-exp of every row's scores.

    A batch: q [batch, length, heads, dim], k and v [batch, key_length, kv_heads, dim], of which sequence b
    has the first ``lengths[b]`` queries and ``key_lengths[b]`` keys (all without them; ``key_lengths`` are ``lengths``
    by default).  A step of generation is a batch of length 1 against a cache with ``key_lengths``.
    Packed sequences: q [n, heads, dim], k and v [m, kv_heads, dim], sequence b the rows ``starts[b]`` to
    ``starts[b + 1]``, its keys by ``key_starts`` (``starts`` by default); indices do not decrease.
    All indices are int32 or int64 on the device, of one type.

    heads may be a multiple of kv_heads: neighbouring query heads share a key head.  dim is at most
    128; bfloat16 or float16.  ``causal``: a sequence's last query sees its last key, each query before it one key
    less; ``window``: of these only the last ``window``.  ``scale``: ``dim ** -0.5`` by default.

    A row that sees no key, or is of no sequence, has out 0 and lse -inf.  Keys and values beyond a
    sequence's are not looked at, whatever they hold; one that is NaN or infinite inside a sequence may also reach
    rows that do not see it, as it does in a product with a probability of 0.  Statistics and sums are fp32,
    in a fixed order; probabilities are rounded to the operands' 16 bits."""
    if stream is None and q.is_cuda and (window is None or window > 0):
        done = _ops_lib.calls().attention(q, k, v, causal, window or 0, scale, starts, key_starts, lengths, key_lengths,
                                          *_here())
        if done is not None:
            return _got(done, "la_attention")
    device, call = _attention_call(q, k, v, causal, window, scale, starts, key_starts, lengths, key_lengths)
    lib = _ops_lib.load()
    with _on_device(device), _Scratch(device, stream) as s:
        out = s.empty(q.shape, q.dtype)
        lse = s.empty(q.shape[:-1], torch.float32)
        if out.numel() == 0:
            return out, lse
        call.out, call.lse = _heads(out, "out", device, q.dim()), _row_values(lse, "lse", device, q)
        size = lib.la_attention_workspace(ctypes.byref(call))
        work = s.workspace(size)
        _check(lib.la_attention(ctypes.byref(call), work.data_ptr(), size, s.handle), "la_attention")
    return out, lse


def attention_grad(grad_out: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor,
                   lse: torch.Tensor, *, causal: bool = True, window: Optional[int] = None,
                   scale: Optional[float] = None, starts: Optional[torch.Tensor] = None,
                   key_starts: Optional[torch.Tensor] = None, lengths: Optional[torch.Tensor] = None,
                   key_lengths: Optional[torch.Tensor] = None,
                   grads: Optional[Tuple[torch.Tensor, torch.Tensor, torch.Tensor]] = None,
                   stream=None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The gradients of ``attention`` towards q, k and v, from that of its out.

    ``out`` and ``lse`` are its results (lse in any order of memory), the other arguments those that it had.
    Probabilities are computed again.  ``grads``: the three tensors to write, like q, k and v (parts of one projection's
    gradient, for instance), not in memory that the call reads, nor one in another's; rows of no sequence stay as they
    were in them.  Without it they are new, and zero there.
    The gradients of a key head are sums over the query heads that share it.  Sums are fp32 in a fixed
    order: equal calls give equal bits."""
    if grads is None and stream is None and q.is_cuda and (window is None or window > 0):
        done = _ops_lib.calls().attention_grad(grad_out, q, k, v, out, lse, causal, window or 0, scale, starts,
                                               key_starts, lengths, key_lengths, *_here())
        if done is not None:
            return _got(done, "la_attention_grad")
    device, call = _attention_call(q, k, v, causal, window, scale, starts, key_starts, lengths, key_lengths)
    dims = q.dim()
    call.grad_out = _heads(grad_out, "grad_out", device, dims, q.dtype, q.shape)
    call.out = _heads(out, "out", device, dims, q.dtype, q.shape)
    call.lse = _row_values(lse, "lse", device, q)
    if grads is not None:
        call.keep_rest = 1
    lib = _ops_lib.load()
    with _on_device(device), _Scratch(device, stream) as s:
        if grads is None:
            grads = tuple(s.empty(t.shape, t.dtype) for t in (q, k, v))
        call.grad_q, call.grad_k, call.grad_v = (_result(g, name, device, dims, q.dtype, t.shape) for g, t, name in
                                                 zip(grads, (q, k, v), ("grad_q", "grad_k", "grad_v")))
        if q.numel() == 0 and k.numel() == 0:
            return grads
        size = lib.la_attention_grad_workspace(ctypes.byref(call))
        work = s.workspace(size)
        _check(lib.la_attention_grad(ctypes.byref(call), work.data_ptr(), size, s.handle), "la_attention_grad")
    return grads


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
