"""Refusals of the row operators, and of the C entry points behind them: everything here is decided on the host, before a launch."""
import ctypes
import pytest
import torch

from spi_amd import hip
from spi_amd.torch_utils.ops import grouped_linear, linear_int8, norm_residual

F64, F32, F16, BF16, I8, I32 = torch.float64, torch.float32, torch.float16, torch.bfloat16, torch.int8, torch.int32
t = lambda *shape, dtype=F32: torch.zeros(*shape, dtype=dtype)  # noqa: E731


@pytest.mark.parametrize('kw,error', [
    (dict(residual=t(3, 9)), ValueError), (dict(residual=t(3, 8, dtype=F16)), ValueError), (dict(h=t(3, 8, dtype=F64), residual=t(3, 8, dtype=F64)), TypeError),
    (dict(norm='batch'), ValueError), (dict(where='inside'), ValueError), (dict(gate_act='lrelu'), ValueError), (dict(eps=0.0), ValueError), (dict(eps=float('nan')), ValueError),
    (dict(post_weight=None), ValueError), (dict(where='before'), ValueError), (dict(where='after', quantize=True), ValueError), (dict(where='after', pre_weight=None,
                                                                                                                                     pre_bias=t(8)), ValueError),
    (dict(pre_weight=t(7)), ValueError), (dict(pre_weight=t(8, dtype=F16)), TypeError), (dict(gate=t(8, dtype=BF16)), TypeError), (dict(gate=t(7)), ValueError),
    (dict(gate=t(3, 1)), ValueError), (dict(gate=t(2, 8)), ValueError), (dict(h=t(2, 3, 8), residual=t(2, 3, 8), gate=t(3, 8)), ValueError),
    (dict(h=t(3, 0), residual=t(3, 0), post_weight=t(0), pre_weight=t(0)), ValueError), (dict(h=t(()), residual=t(())), ValueError),
    (dict(h=t(1, 32769), residual=t(1, 32769), post_weight=t(32769), pre_weight=t(32769)), ValueError), ({}, RuntimeError)])
def test_norm_residual_refuses(kw, error):
    with pytest.raises(error):
        norm_residual.norm_residual(**{**dict(h=t(3, 8), residual=t(3, 8), post_weight=t(8), pre_weight=t(8)), **kw})


@pytest.mark.parametrize('kw,error', [
    (dict(act='gelu'), KeyError), (dict(weight_q=t(4, 8)), ValueError), (dict(weight_q=t(8, dtype=I8)), ValueError), (dict(x=t(3, 9)), ValueError),
    (dict(weight_scale=t(5)), ValueError), (dict(weight_scale=t(4, dtype=F16)), ValueError), (dict(bias=t(5)), ValueError), (dict(bias=t(4, dtype=F16)), ValueError),
    (dict(x=t(3, 8, dtype=I8)), ValueError), (dict(x=t(3, 8, dtype=I8), x_scale=t(4)), ValueError), (dict(x_scale=t(3)), ValueError), (dict(x=t(3, 8, dtype=F64)), TypeError),
    (dict(out_dtype=F64), TypeError), (dict(x=t(1, 131072), weight_q=t(4, 131072, dtype=I8)), ValueError), (dict(weight_q=t(0, 8, dtype=I8), weight_scale=t(0)), ValueError),
    (dict(x=torch.zeros(3, 8, requires_grad=True)), RuntimeError), ({}, RuntimeError)])
def test_linear_int8_refuses(kw, error):
    with pytest.raises(error):
        linear_int8.linear_int8(**{**dict(x=t(3, 8), weight_q=t(4, 8, dtype=I8), weight_scale=t(4)), **kw})


@pytest.mark.parametrize('x,error', [(t(3, 8, dtype=F64), TypeError), (t(3, 0), ValueError), (t(()), ValueError), (t(1, 131072), ValueError), (t(3, 8), RuntimeError)])
def test_quantize_rows_refuses(x, error):
    with pytest.raises(error):
        linear_int8.quantize_rows(x)


@pytest.mark.parametrize('kw,error', [
    (dict(x=t(3, 9)), ValueError), (dict(x=t(8)), ValueError), (dict(weight=t(4, 8)), ValueError), (dict(weight=t(0, 4, 8), offsets=t(1, dtype=I32)), ValueError),
    (dict(x=t(3, 8, dtype=F16)), TypeError), (dict(x=t(3, 8, dtype=F64), weight=t(2, 4, 8, dtype=F64)), TypeError), (dict(bias=t(2, 4, dtype=BF16)), TypeError),
    (dict(offsets=t(2, dtype=I32)), ValueError), (dict(offsets=t(3, dtype=torch.int64)), ValueError), (dict(bias=t(2, 8)), ValueError), ({}, RuntimeError)])
def test_grouped_linear_refuses(kw, error):
    with pytest.raises(error):
        grouped_linear.grouped_linear(**{**dict(x=t(3, 8), weight=t(2, 4, 8), offsets=t(3, dtype=I32)), **kw})


def test_c_entries_return_errors():
    """wrong descriptors come back as SPI_ERR_BAD_ARG with a text, never as an abort; nothing is launched"""
    L = hip.lib()
    assert L.spi_norm_residual_fwd(None, None) == L.spi_linear_int8(None, None) == L.spi_grouped_linear_fwd(None, None) == -1
    p = 0x1000
    n = hip.NormResidualDesc(4, 1, 64, 0, 0, 0, 0, 1, 0, 1, 1, 1.0, 1e-6, p, p, None, p, None, p, None)
    for field, value in (('width', 0), ('width', 32769), ('dtype', 2), ('weight_dtype', 1), ('gate_mode', 1), ('gate_mode', 9), ('gate_act', 3), ('eps', 0.0), ('h', None),
                         ('pre_weight', None), ('rows', -1), ('rows', 1 << 31), ('stream_out', None), ('stats', p + 8)):
        d = hip.NormResidualDesc.from_buffer_copy(n)
        setattr(d, field, value)
        assert L.spi_norm_residual_fwd(ctypes.byref(d), None) == -1 and L.spi_last_error(), field
    n.width, n.stats, n.d_normed = 8193, p, p
    assert L.spi_norm_residual_bwd(ctypes.byref(n), None) == -1 and b'8193' in L.spi_last_error()
    n.width = 64
    n.d_pre_weight = p
    assert L.spi_norm_residual_bwd_workspace(ctypes.byref(n)) > 0 and L.spi_norm_residual_bwd(ctypes.byref(n), None) == -1 and b'workspace' in L.spi_last_error()
    i = hip.LinearInt8Desc(40, 8, 32, 0, 0, 32, 32, 256, p, None, p, p, None, p, 1, 0.0, 1.0, -1.0)
    for field, value in (('M', -1), ('M', (1 << 30) + 1), ('N', 0), ('K', 131072), ('x_dtype', 2), ('x_dtype', 4), ('y_dtype', 4), ('x_stride', 31), ('w_stride', 31), ('w_bytes', 255), ('act', 0), ('act', 10),
                         ('x', None), ('y', None), ('w', None), ('w_scale', None)):
        d = hip.LinearInt8Desc.from_buffer_copy(i)
        setattr(d, field, value)
        assert L.spi_linear_int8(ctypes.byref(d), None) == -1 and L.spi_last_error(), field
    assert L.spi_linear_int8_workspace(ctypes.byref(i)) > 0 and L.spi_linear_int8(ctypes.byref(i), None) == -1 and b'workspace' in L.spi_last_error()
    g = hip.GroupedLinearDesc(4, 2, 8, 8, 0, 1.0, p, p, None, p)
    for field, value in (('T', -1), ('E', 0), ('E', 65536), ('N', 0), ('K', 0), ('dtype', 2), ('offsets', None), ('x', None)):
        d = hip.GroupedLinearDesc.from_buffer_copy(g)
        setattr(d, field, value)
        assert L.spi_grouped_linear_fwd(ctypes.byref(d), None) == -1 and L.spi_last_error(), field
    assert L.spi_grouped_linear_dgrad(ctypes.byref(g), None) == -1
    assert L.spi_grouped_linear_wgrad(ctypes.byref(g), None) == -1
    assert L.spi_quantize_rows(p, 4, 32, 31, 0, p, 32, p, None) == -1 and L.spi_quantize_rows(p, 4, 32, 32, 2, p, 32, p, None) == -1
