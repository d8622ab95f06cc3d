"""What the row operators decide on the host beyond their refusals: which descriptors their C entries take."""
import ctypes


from spi_amd import hip

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
