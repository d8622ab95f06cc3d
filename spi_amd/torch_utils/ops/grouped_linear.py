"""Fully connected layers over ragged groups of rows, each group with a weight of its own, with autograd.

    y[t] = gain * weight[e] @ x[t] + bias[e]        for offsets[e] <= t < offsets[e + 1]

Rows sorted by what chooses their weight: the rows of W+ by the mapper of their resolution level, the rows of several people by the tuned generator they belong
to, tokens by expert.  One launch for all groups, and the group sizes stay on the GPU: no host synchronisation, and a captured graph replays with other sizes.
``gain`` is the equalised learning rate's factor of ``FullyConnectedLayer`` (networks_stylegan2.py:95-127).
"""
import ctypes
import torch
from ... import hip


def _desc(cfg, x, weight, offsets):
    t, e, n, k, dtype, gain = cfg
    return hip.GroupedLinearDesc(t, e, n, k, dtype, gain, None if x is None else x.data_ptr(), None if weight is None else weight.data_ptr(), None, offsets.data_ptr())


def _launch(name, pass_id, d, device):
    ref = ctypes.byref(d)
    nbytes = hip.lib().spi_grouped_linear_workspace(ref, pass_id)
    if nbytes:
        workspace = torch.empty(nbytes, device=device, dtype=torch.uint8)
        d.workspace, d.workspace_bytes = workspace.data_ptr(), nbytes
    hip.call(name, ref, hip.stream())


def _forward(cfg, x, weight, bias, offsets):
    y = torch.empty(x.shape[0], weight.shape[1], device=x.device, dtype=x.dtype)
    d = _desc(cfg, x, weight, offsets)
    d.bias, d.y = None if bias is None else bias.data_ptr(), y.data_ptr()
    _launch('spi_grouped_linear_fwd', 0, d, x.device)
    return y


class _GroupedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, cfg, x, weight, bias, offsets):
        ctx.cfg = cfg
        ctx.save_for_backward(x, weight, offsets)
        return _forward(cfg, x, weight, bias, offsets)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, offsets = ctx.saved_tensors
        return (None, *hip.on(x.get_device(), _backward, ctx.cfg, ctx.needs_input_grad[1:4], x, weight, offsets, dy), None)


def _backward(cfg, need, x, weight, offsets, dy):
    dx = dw = db = None
    if not dy.is_contiguous():
        dy = dy.contiguous()
    if need[0]:
        dx = torch.empty_like(x)
        d = _desc(cfg, None, weight, offsets)
        d.dy, d.dx = dy.data_ptr(), dx.data_ptr()
        _launch('spi_grouped_linear_dgrad', 1, d, x.device)
    if need[1] or need[2]:
        d = _desc(cfg, x, None, offsets)
        d.dy = dy.data_ptr()
        if need[1]:
            dw = torch.empty_like(weight)
            d.dw = dw.data_ptr()
        if need[2]:
            db = torch.empty(weight.shape[:2], device=x.device, dtype=x.dtype)
            d.db = db.data_ptr()
        _launch('spi_grouped_linear_wgrad', 2, d, x.device)
    return dx, dw, db


def grouped_linear(x, weight, offsets, bias=None, gain=1.0):
    """x [T, K], weight [E, N, K], bias [E, N] or None, of one type (fp32 / fp16 / bf16); offsets int32 [E + 1] on the GPU -> y [T, N].

    Groups may be empty.  Rows in no group (before offsets[0], from offsets[E] on) give 0 and get gradient 0; an empty group's weight and bias get gradient 0.
    The offsets are read on the GPU, as their running maximum clamped to 0 .. T."""
    if x.ndim != 2 or weight.ndim != 3 or weight.shape[2] != x.shape[1] or 0 in weight.shape:
        raise ValueError(f'rows {tuple(x.shape)} [T, K] and weights {tuple(weight.shape)} [E, N, K] do not fit')
    if x.dtype not in hip.ROW_DTYPES or weight.dtype != x.dtype or (bias is not None and bias.dtype != x.dtype):
        raise TypeError(f'x {x.dtype}, weight {weight.dtype}, bias {None if bias is None else bias.dtype}: one of float32, float16, bfloat16 for all')
    if offsets.shape != (weight.shape[0] + 1,) or offsets.dtype != torch.int32:
        raise ValueError(f'offsets {tuple(offsets.shape)} {offsets.dtype}: int32 [{weight.shape[0] + 1}]')
    if bias is not None and bias.shape != weight.shape[:2]:
        raise ValueError(f'bias {tuple(bias.shape)} for weights {tuple(weight.shape)}')
    device = hip.same_device(x, weight, offsets, bias)
    wants_grad = hip.records(x, weight, bias)                          # (forward-mode tangents end in an error of the autograd function, which has none)
    x, weight, offsets = x.contiguous(), weight.contiguous(), offsets.contiguous()
    bias = None if bias is None else bias.contiguous()
    cfg = (x.shape[0], weight.shape[0], weight.shape[1], x.shape[1], hip.ROW_DTYPES[x.dtype], float(gain))
    if wants_grad:
        return hip.on(device, _GroupedLinear.apply, cfg, x, weight, bias, offsets)
    return hip.on(device, _forward, cfg, x, weight, bias, offsets)
