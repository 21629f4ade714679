"""How much memory the loss with gradients takes beside its operands, and what it is made of.
Sizes come from the library; nothing is launched."""
from __future__ import annotations

import ctypes

from slideformer_amd import _lib, _ops_lib

MIB = 1 << 20


def _bytes(n, vocab, hidden, piece_bytes, grad_weight=_lib.LA_BF16):
    """The workspace of a call as linear_cross_entropy_grad makes it."""
    call = _ops_lib.LaLinearLoss(
        dtype=_lib.LA_BF16, n=n, hidden=hidden, x_stride=hidden, weight=256, vocab=vocab, weight_stride=hidden,
        grads=1, grad_x_stride=hidden, grad_weight_dtype=grad_weight, grad_weight_stride=hidden,
        piece_rows=min(max(256, piece_bytes // (2 * vocab) // 256 * 256), 1 << 22))
    return _ops_lib.load().la_linear_loss_workspace(ctypes.byref(call))


def _up(x, to):
    return -(-x // to) * to


def _parts(n, vocab, hidden, rows):
    """(softmax of `rows` rows in 16 bits, what all of a call's other buffers but the partial and running sums take
    at most: the gathered states, a part of each row for 128 columns at the least, and lists)."""
    columns = _up(vocab, 256)
    return rows * columns * 2, _up(n, 256) * (_up(hidden, 64) * 2 + 32) + rows * (columns // 128 * 8 + 8) + MIB


def test_partial_sums_take_half_of_the_softmax():
    """The sums of the states' gradient over runs of k: at most half of the softmax in 16 bits, or 64 MiB, or one
    run."""
    for n, vocab, hidden in ((4096, 128256, 4096), (2048, 128256, 8192), (1024, 50257, 768), (4096, 32000, 4096),
                             (4096, 1000, 4096), (300, 700, 64)):
        softmax, others = _parts(n, vocab, hidden, _up(n, 256))
        sums = max(softmax // 2, 64 * MIB, _up(n, 256) * hidden * 4)
        assert _bytes(n, vocab, hidden, 1 << 40) <= softmax + sums + others, (n, vocab, hidden)


def test_an_fp32_gradient_is_its_own_sum_over_pieces():
    """A grad_weight in fp32 holds the sum over the pieces itself: no second matrix beside it."""
    n, vocab, hidden = 8192, 128256, 4096
    softmax, others = _parts(n, vocab, hidden, 1024)
    assert _bytes(n, vocab, hidden, 1024 * 2 * vocab, _lib.LA_F32) <= softmax * 3 // 2 + others


def test_smaller_pieces_never_take_more_memory():
    for n, vocab, hidden in ((4096, 128256, 4096), (8192, 128256, 4096), (16384, 128256, 4096), (32768, 32000, 4096),
                             (8192, 50257, 768), (60000, 32000, 1024), (1000, 1000, 64)):
        for grad_weight in (_lib.LA_BF16, _lib.LA_F32):
            sizes = [_bytes(n, vocab, hidden, b << 20, grad_weight) for b in (1 << 20, 4096, 2048, 1024, 512, 128, 16, 1)]
            assert all(a >= b for a, b in zip(sizes, sizes[1:])), (n, vocab, hidden, sizes)
        # and eight pieces or more do take less than all rows' scores in 16 bits, where the matrix is small beside them
        if vocab * hidden * 4 * 3 < n * vocab * 2 and n * vocab * 2 > 8 * (128 << 20):
            assert _bytes(n, vocab, hidden, 128 << 20) < n * vocab * 2, (n, vocab, hidden)


def test_a_piece_more_does_not_cost_a_matrix():
    """One row more than a piece of the default size holds, of 128256 x 4096 in bf16."""
    assert _bytes(4097, 128256, 4096, 1 << 30) < 1.1 * _bytes(4096, 128256, 4096, 1 << 30)


def test_all_rows_at_once_are_as_many_as_a_launch_takes():
    """piece_rows 0 asks for all rows: pieces of 32768 where there are more."""
    def size(n, piece_rows):
        call = _ops_lib.LaLinearLoss(
            dtype=_lib.LA_BF16, n=n, hidden=64, x_stride=64, weight=256, vocab=300, weight_stride=64, grads=1,
            grad_x_stride=64, grad_weight_dtype=_lib.LA_BF16, grad_weight_stride=64, piece_rows=piece_rows)
        return _ops_lib.load().la_linear_loss_workspace(ctypes.byref(call))

    for n in (1, 256, 32768, 32769, 65536, 100000, 1 << 22):
        assert size(n, 0) == size(n, 32768), n
