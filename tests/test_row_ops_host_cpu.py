"""What the row operators decide on the host, beyond their refusals: which descriptors their C entries take, how a gate lies over the rows, which calls record a derivative."""
import ctypes

import pytest
import torch
from torch.autograd import forward_ad

from spi_amd import hip
from spi_amd.torch_utils.ops import linear_int8, norm_residual

P = 0x1000                                                             # never read


def test_backward_takes_a_pass_in_which_no_norm_is_left():
    """norms before the block only, and only the stream was used: its gradients go through no norm.  (The call is ended by its workspace, so that nothing is launched.)"""
    d = hip.NormResidualDesc(100, 1, 64, 0, 0, 0, 1, 1, 0, 0, 0, 1.0, 1e-6, P, P, P)
    d.stats, d.d_stream, d.d_gate = P, P, P
    L = hip.lib()
    assert L.spi_norm_residual_bwd_workspace(ctypes.byref(d)) > 0
    assert L.spi_norm_residual_bwd(ctypes.byref(d), None) == -1 and b'workspace' in L.spi_last_error()
    d.stream_out = P
    assert L.spi_norm_residual_fwd(ctypes.byref(d), None) == -1 and b'no norm' in L.spi_last_error()


@pytest.mark.parametrize('h,gate,mode', [((0, 5, 8), (0, 1, 8), (2, 5)), ((0, 5, 8), (0, 8), (2, 5)), ((0, 5, 8), (0, 5, 8), (3, 1)), ((0, 5, 8), (8,), (1, 1)), ((2, 0, 8), (2, 1, 8), (3, 1)),
                                         ((0, 8), (0, 8), (3, 1)), ((2, 5, 8), (2, 1, 8), (2, 5)), ((2, 3, 5, 8), (2, 8), (2, 15)), ((2, 1, 8), (2, 8), (3, 1)), ((1, 5, 8), (1, 1, 8), (1, 1))])
def test_gates_of_empty_batches(h, gate, mode):
    assert norm_residual._gate_mode(torch.zeros(h), torch.zeros(gate)) == mode
    with pytest.raises(RuntimeError, match='GPU'):                     # a legal call but for its device
        norm_residual.norm_residual(torch.zeros(h), torch.zeros(h), gate=torch.zeros(gate), post_weight=torch.zeros(8), pre_weight=torch.zeros(8))


@pytest.mark.parametrize('h,gate', [((0, 5, 8), (0, 3, 8)), ((0, 5, 8), (0, 0, 8)), ((0, 5, 8), (1, 5, 8)), ((2, 0, 8), (3, 8)), ((2, 5, 8), (2, 5, 1, 8))])
def test_gates_that_do_not_fit_an_empty_batch(h, gate):
    with pytest.raises(ValueError, match='neither'):
        norm_residual._gate_mode(torch.zeros(h), torch.zeros(gate))


def test_quantize_rows_loses_no_gradient():
    x = torch.zeros(3, 8, requires_grad=True)
    with pytest.raises(RuntimeError, match='no gradient'):
        linear_int8.quantize_rows(x)
    for legal in (lambda: linear_int8.quantize_rows(x.detach()), torch.no_grad()(lambda: linear_int8.quantize_rows(x))):
        with pytest.raises(RuntimeError, match='GPU'):                 # but for its device
            legal()


def test_which_calls_record_a_derivative():
    plain, leaf = torch.zeros(3, 8), torch.zeros(3, 8, requires_grad=True)
    assert not hip.records() and not hip.records(plain, None) and hip.records(plain, None, leaf) and hip.records(leaf * 2)
    with torch.no_grad():
        assert not hip.records(leaf)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(plain, torch.ones(3, 8))
        assert hip.records(None, dual) and not hip.records(plain) and not hip.records(torch.zeros(3, 8, dtype=torch.int8))
        with torch.no_grad():                                          # (which has no say in forward mode)
            assert hip.records(dual[:, :4])
        for call in (lambda: linear_int8.quantize_rows(dual), lambda: linear_int8.linear_int8(dual, torch.zeros(4, 8, dtype=torch.int8), torch.zeros(4)),
                     torch.no_grad()(lambda: linear_int8.linear_int8(plain, torch.zeros(4, 8, dtype=torch.int8), torch.zeros(4), bias=dual[0, :4]))):
            with pytest.raises(RuntimeError, match='no gradient'):
                call()
    assert not hip.records(dual)
