"""GPU tests of the row operators (norm_residual, quantize_rows / linear_int8, grouped_linear) at the edges of what their calls take: the largest launches, every tile of the
product kernels, empty and tiny operands, partial gradients.  The 64-bit statements and bounds are those of row_ops_ref."""
import pytest
import torch

import row_ops_ref as ref
from test_hip_row_ops_gpu import check_grouped, int8_reference

pytestmark = pytest.mark.gpu
DEV = 'cuda'
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def randn(g, *shape, dtype=F32, scale=1.0):
    return (torch.randn(*shape, device=DEV, generator=g) * scale).to(dtype)


# ---- launches ----------------------------------------------------------------------------------------------------------------------------
def test_linear_int8_more_outputs_than_a_launch_has_threads():
    from spi_amd.torch_utils.ops.linear_int8 import linear_int8
    n, odd = 1 << 28, 37                                              # sixteen outputs to a block of 256 threads: 2^32 of them and a few more
    w = torch.ones(n + odd, 1, device=DEV, dtype=torch.int8)
    w[-odd:, 0] = torch.arange(odd, device=DEV, dtype=torch.int8)
    scale = torch.ones(n + odd, device=DEV)
    q, one = torch.full((1, 1), 3, device=DEV, dtype=torch.int8), torch.ones(1, device=DEV)
    y = linear_int8(q, w, scale, x_scale=one, out_dtype=F16)          # whole numbers: exact in fp16
    assert torch.equal(y[0, -odd:], 3 * torch.arange(odd, device=DEV).half())
    assert all((part == 3).all() for part in y[0, :n].split(1 << 26))


def test_products_of_more_narrow_rows_than_a_launch_has_threads():
    """one output for each of 2^30 rows, weights of less than 16 bytes: 2^24 tiles of 256 threads"""
    from spi_amd.torch_utils.ops.grouped_linear import grouped_linear
    from spi_amd.torch_utils.ops.linear_int8 import linear_int8
    rows, odd = 1 << 30, 37
    q = torch.ones(rows, 1, device=DEV, dtype=torch.int8)
    q[-odd:, 0] = torch.arange(odd, device=DEV, dtype=torch.int8)
    one = torch.ones(1, device=DEV)
    y = linear_int8(q, torch.full((1, 1), 3, device=DEV, dtype=torch.int8), one, x_scale=one.expand(rows), out_dtype=F16)
    assert torch.equal(y[-odd:, 0], 3 * torch.arange(odd, device=DEV).half())
    assert all((part == 3).all() for part in y[:-odd].split(1 << 27))
    del y
    x = q.half()
    with torch.no_grad():
        y = grouped_linear(x, torch.tensor([[[3.0]], [[5.0]]], device=DEV, dtype=F16), torch.tensor([0, rows - odd, rows], device=DEV, dtype=torch.int32))
    assert torch.equal(y[-odd:, 0], 5 * torch.arange(odd, device=DEV).half())
    assert all((part == 3).all() for part in y[:-odd].split(1 << 27))


# ---- empty and tiny operands -------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize('sizes,k,n', [([0] * 8, 1003, 1003), ([0] * 8, 1003, 771), ([0] * 3, 5, 7), ([1] + [0] * 99, 5, 1003), ([0] * 399 + [1], 5, 3), ([0, 1, 0, 2] + [0] * 60, 3, 1003),
                                       ([1] * 5, 1, 4099), ([700, 1300], 3, 1), ([50_000], 1, 7)])
def test_grouped_without_rows_or_with_hardly_any(sizes, k, n):
    for dtype in (F32, F16, BF16):
        check_grouped(sizes, k, n, dtype)
        check_grouped(sizes, k, n, dtype, head=1, behind=2, bias=False)


@pytest.mark.parametrize('m,n,k', [(50_000, 1, 15), (50_000, 1, 1), (49_153, 5, 3), (17, 1, 9), (70_000, 2, 7)])
def test_linear_int8_with_weights_of_less_than_16_bytes(m, n, k):
    from spi_amd.torch_utils.ops.linear_int8 import linear_int8, quantize_rows
    g = gen(m + n)
    wq, ws = quantize_rows(randn(g, n, k))
    wq = wq.contiguous()                                              # (out of its padded rows: n * k bytes)
    for dtype in (F32, BF16):
        x = randn(g, m, k, dtype=dtype)
        q, s = quantize_rows(x)
        r, mag = int8_reference(q, s, wq, ws, None, 'lrelu', 2 ** 0.5, None)
        ref.check(linear_int8(x, wq, ws, act='lrelu'), r, mag, 8, f'{m} x {n} x {k}')
        ref.check(linear_int8(q.contiguous(), wq, ws, x_scale=s, act='lrelu'), r, mag, 8, f'{m} x {n} x {k} integers')
