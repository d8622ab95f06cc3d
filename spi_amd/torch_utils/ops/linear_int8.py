"""Fully connected layers in 8-bit integers, with a scale for each row (token) and each output channel.

    y = clamp(act(x_scale * weight_scale * (q @ weight_q.T) + bias) * gain)

For FROZEN layers (stage 1 and the mapping network never change their weights): ``quantize_rows`` lays a weight ``[out, in]`` out once, ``linear_int8`` takes
the layer's place, with the activations of ``bias_act`` in its epilogue.  The integer sums are exact; the only losses are the two roundings to 8 bits.
"""
import ctypes
import torch
from ... import hip
from . import bias_act as _ba

MAX_IN_FEATURES = 131071         # SPI_LINEAR_INT8_MAX_K: 127 * 127 * in_features stays below 2^31


def _rows(x):
    """[..., K] -> [rows, K] with adjacent values, and rows that are K .. 2^22 values apart"""
    if x.ndim == 2 and x.is_contiguous():
        return x
    k = x.shape[-1]
    x = x.reshape(-1, k)
    return x if (k == 1 or x.stride(1) == 1) and (x.shape[0] <= 1 or k <= x.stride(0) <= 1 << 22) else x.contiguous()


def _stride(x):
    return x.stride(0) if x.shape[0] > 1 else x.shape[1]


def quantize_rows(x):
    """x [..., K] (fp32 / fp16 / bf16) -> (q int8 [..., K], scale fp32 [...]): ``scale = max|row| / 127``, ``q = round(row / scale)``, ties to even, the division in
    fp32.  A row of zeros has scale 0; a row that holds an infinity or NaN has scale NaN (so its products are NaN) and q = 0.  The rows of q begin on 16 bytes:
    q is a view of a buffer with K rounded up to 16.  Inference only: a call that would have to record a gradient raises."""
    if x.ndim < 1 or not 1 <= x.shape[-1] <= MAX_IN_FEATURES:
        raise ValueError(f'rows of {tuple(x.shape)[-1:]} values: 1 to {MAX_IN_FEATURES}')
    if x.dtype not in hip.ROW_DTYPES:
        raise TypeError(f'rows of {x.dtype}: float32, float16 or bfloat16')
    if hip.records(x):
        raise RuntimeError('quantize_rows: rounded rows have no gradient; call it under torch.no_grad() or on tensors that need none')
    return hip.on(hip.same_device(x), _quantize, x)


def _quantize(x):
    k = x.shape[-1]
    pitch = (k + 15) // 16 * 16
    q = torch.empty(x.shape[:-1] + (pitch,), device=x.device, dtype=torch.int8)
    scale = torch.empty(x.shape[:-1], device=x.device, dtype=torch.float32)
    r = _rows(x)
    hip.call('spi_quantize_rows', r.data_ptr(), r.shape[0], k, _stride(r), hip.ROW_DTYPES[x.dtype], q.data_ptr(), pitch, scale.data_ptr(), hip.stream())
    return (q if pitch == k else q[..., :k]), scale


def linear_int8(x, weight_q, weight_scale, bias=None, x_scale=None, act='linear', alpha=None, gain=None, clamp=None, out_dtype=None):
    """x [..., K] -> y [..., N].

    x             fp32 / fp16 / bf16 rows, quantised by the call as ``quantize_rows`` does, or int8 rows with their ``x_scale`` [...] (fp32)
    weight_q      int8 [N, K] and weight_scale fp32 [N], from ``quantize_rows(weight)``, whose rows begin on 16 bytes: fastest.  Rows of adjacent values at other places, at most
                  2^22 bytes apart, are read as they lie; any others are copied by every call
    bias          [N] (fp32) or None;  act, alpha, gain, clamp as in ``bias_act``
    out_dtype     fp32 / fp16 / bf16; default: x's type, fp32 for int8 rows

    Inference only: the rounding has no gradient, so a call that would have to record one raises."""
    if act not in _ba.activation_funcs:
        raise KeyError(act)
    act_id, d_alpha, d_gain, _ = _ba.activation_funcs[act]
    if weight_q.ndim != 2 or weight_q.dtype != torch.int8 or 0 in weight_q.shape:
        raise ValueError(f'weight_q {tuple(weight_q.shape)} {weight_q.dtype}: int8 [out_features, in_features]')
    n, k = weight_q.shape
    if x.ndim < 1 or x.shape[-1] != k:
        raise ValueError(f'rows {tuple(x.shape)} for a weight {tuple(weight_q.shape)}')
    if k > MAX_IN_FEATURES:
        raise ValueError(f'{k} in_features: at most {MAX_IN_FEATURES} (the sums are 32-bit integers)')
    if weight_scale.shape != (n,) or weight_scale.dtype != torch.float32:
        raise ValueError(f'weight_scale {tuple(weight_scale.shape)} {weight_scale.dtype}: float32 [{n}]')
    if bias is not None and (bias.shape != (n,) or bias.dtype != torch.float32):
        raise ValueError(f'bias {tuple(bias.shape)} {bias.dtype}: float32 [{n}]')
    int_rows = x.dtype == torch.int8
    if int_rows:
        if x_scale is None or x_scale.shape != x.shape[:-1] or x_scale.dtype != torch.float32:
            raise ValueError(f'int8 rows {tuple(x.shape)} want x_scale, float32 {tuple(x.shape[:-1])}')
    elif x_scale is not None:
        raise ValueError('x_scale belongs to int8 rows')
    elif x.dtype not in hip.ROW_DTYPES:
        raise TypeError(f'rows of {x.dtype}: float32, float16, bfloat16 or int8')
    out_dtype = out_dtype or (torch.float32 if int_rows else x.dtype)
    if out_dtype not in hip.ROW_DTYPES:
        raise TypeError(f'out_dtype {out_dtype}: float32, float16 or bfloat16')
    if hip.records(x, weight_scale, bias, x_scale):
        raise RuntimeError('linear_int8: rounded rows have no gradient; call it under torch.no_grad() or on tensors that need none')
    return hip.on(hip.same_device(x, weight_q, weight_scale, bias, x_scale), _linear, x, weight_q, weight_scale, bias, x_scale, act_id, float(d_alpha if alpha is None else alpha),
                  float(d_gain if gain is None else gain), float(-1 if clamp is None else clamp), out_dtype)


def _linear(x, weight_q, weight_scale, bias, x_scale, act_id, alpha, gain, clamp, out_dtype):
    n, k = weight_q.shape
    y = torch.empty(x.shape[:-1] + (n,), device=x.device, dtype=out_dtype)
    r, w = _rows(x), _rows(weight_q)
    m = r.shape[0]
    if m == 0:
        return y
    if not weight_scale.is_contiguous():
        weight_scale = weight_scale.contiguous()
    if bias is not None and not bias.is_contiguous():
        bias = bias.contiguous()
    if x_scale is not None and not x_scale.is_contiguous():
        x_scale = x_scale.contiguous()
    d = hip.LinearInt8Desc(m, n, k, hip.DTYPE_I8 if x_scale is not None else hip.ROW_DTYPES[x.dtype], hip.ROW_DTYPES[out_dtype], _stride(r), _stride(w),
                           w.untyped_storage().nbytes() - w.storage_offset(), r.data_ptr(), None if x_scale is None else x_scale.data_ptr(), w.data_ptr(),
                           weight_scale.data_ptr(), None if bias is None else bias.data_ptr(), y.data_ptr(), act_id, alpha, gain, clamp)
    ref = ctypes.byref(d)
    nbytes = hip.lib().spi_linear_int8_workspace(ref)
    if nbytes:
        workspace = torch.empty(nbytes, device=x.device, dtype=torch.uint8)
        d.workspace, d.workspace_bytes = workspace.data_ptr(), nbytes
    hip.call('spi_linear_int8', ref, hip.stream())
    return y
