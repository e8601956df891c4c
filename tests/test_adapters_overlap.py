"""Adapters into a y that shares memory with x are refused: other rows' products would read what has been written."""
import ctypes

import pytest
import torch

from nanochat_b200 import _lib

N, K, ROWS = 64, 48, 3


def call(y, y_stride, x, x_stride, out, out_stride, rows=ROWS):
    """The C entry on host addresses: refused before anything is read."""
    hold = ctypes.create_string_buffer(4096)
    at = (ctypes.addressof(hold) + 255) // 256 * 256
    _lib.call("nckv_adapters", y, y_stride, x, x_stride, at, at, at, at, out, out_stride, rows, 1, K, N, 8, 1, None, 0, at, None)


@pytest.mark.skipif(torch.cuda.is_available(), reason="host addresses")
@pytest.mark.parametrize("x_at,x_stride,y_stride,rows", [
    (0, 128, 128, 3),      # one and the same
    (56, 128, 128, 3),     # x begins in y's last columns
    (96, 128, 128, 3),     # x ends in the next row's first columns
    (2 * 128 + 56, 128, 128, 3),
    (0, 96, 128, 3),       # rows at other distances
    (32, 64, 64, 1),       # one row
    (-40, 64, 64, 1),
])
def test_the_library_refuses(x_at, x_stride, y_stride, rows):
    y = 1 << 20
    with pytest.raises(_lib.NckvError, match="share"):
        call(y, y_stride, y + 2 * x_at, x_stride, y, y_stride, rows)
    with pytest.raises(_lib.NckvError, match="share"):  # a result beside y: the same
        call(1 << 24, y_stride, y + 2 * x_at, x_stride, y, y_stride, rows)


@pytest.mark.skipif(torch.cuda.is_available(), reason="host addresses")
def test_a_result_is_y_or_beside_it():
    y, x = 1 << 20, 1 << 24
    for out, stride in ((y, 192), (y + 64, 128), (y + 2 * 128, 128)):
        with pytest.raises(_lib.NckvError, match="share"):
            call(y, 128, x, 48, out, stride)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 3, 260])
def test_slices_of_one_product_beside_each_other(T):
    from nanochat_b200 import ops
    from .test_adapters_gpu import make
    y, x, *rest = make(4, T, K, N, 8, 3, seed=T, slots=[0, 2, -1, 1])
    want = ops.add_adapters(y, x, *rest)
    for x_first in (False, True):
        wide = torch.full((4, T, 128), 7.0, device="cuda", dtype=torch.bfloat16)
        part, other = (wide[..., 48:112], wide[..., :48]) if x_first else (wide[..., 8:72], wide[..., 72:120])
        part.copy_(y)
        other.copy_(x)
        assert torch.equal(ops.add_adapters_(part, other, *rest), want) and torch.equal(other, x)
        assert (wide[..., 120:] == 7).all()
        with pytest.raises(RuntimeError, match="share"):
            ops.add_adapters_(part, wide[..., 64:112], *rest)
        assert torch.equal(part, want)
        got = ops.add_adapters(part, wide[..., 64:112], *rest)  # beside y: any x
        assert torch.equal(got, ops.add_adapters(part.contiguous(), wide[..., 64:112].contiguous(), *rest))
    with pytest.raises(RuntimeError, match="share"):
        square = make(4, T, N, N, 8, 3, seed=T)
        ops.add_adapters_(square[0], square[0], *square[2:])
