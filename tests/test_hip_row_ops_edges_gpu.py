"""GPU tests of the row operators (norm_residual, quantize_rows / linear_int8, grouped_linear) at the edges of what their calls take: the largest launches, every tile of the
product kernels, empty and tiny operands, partial gradients.  The 64-bit statements and bounds are those of row_ops_ref."""
import pytest
import torch

import row_ops_ref as ref

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
