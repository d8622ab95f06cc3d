"""Norms before and after a residual block, fused with the block's gate and residual scale, with autograd.

``norm_residual`` is everything a residual stack of vectors (latent rows through fully connected layers) does between two blocks:

    z      = Norm(h; post_weight, post_bias)            the block's output, normalised (``where='before'``: z = h)
    stream = residual + scale * act(gate) * z
    normed = Norm(stream; pre_weight, pre_bias)         the next block's input (``where='after'``: None)

with Norm the RMS norm of ``normalize_2nd_moment`` (networks_stylegan2.py:27-29) or, with ``norm='layer'``, the layer norm, each with a learned weight and
an optional bias.  One launch forward; backward one launch and, for the gradients that are sums over rows, a second.  The sums are fp32; ``stream`` and
``normed`` are rounded once, ``normed`` from the unrounded stream.
"""
import ctypes
import torch
from ... import hip
from . import bias_act as _ba

MAX_WIDTH = 32768                # SPI_NORM_MAX_WIDTH
MAX_WIDTH_BACKWARD = 8192        # SPI_NORM_MAX_WIDTH_BWD
_GATE_ACTS = ('linear', 'tanh', 'sigmoid')
_GATE_NONE, _GATE_CHANNEL, _GATE_SAMPLE, _GATE_FULL = range(4)


def _p(t):
    return None if t is None else t.data_ptr()


def _desc(cfg, h, residual, gate, weights):
    """``weights``: (post_weight, post_bias, pre_weight, pre_bias).  Contiguous tensors."""
    rows, width, per_sample, mode, act, layer, after, before, scale, eps = cfg
    w = weights[0] if after else weights[2]
    return hip.NormResidualDesc(rows, per_sample, width, hip.ROW_DTYPES[h.dtype], 0 if w is None else hip.ROW_DTYPES[w.dtype],
                                0 if gate is None else hip.ROW_DTYPES[gate.dtype], mode, act, layer, after, before, scale, eps, h.data_ptr(), residual.data_ptr(),
                                _p(gate), *map(_p, weights))


def _forward(cfg, h, residual, gate, weights, want_stats, quantize=False):
    rows, width, before = cfg[0], cfg[1], cfg[7]
    d = _desc(cfg, h, residual, gate, weights)
    stream = torch.empty_like(residual)
    d.stream_out = stream.data_ptr()
    normed = stats = None
    if before and quantize:
        pitch = (width + 15) // 16 * 16
        q = torch.empty(h.shape[:-1] + (pitch,), device=h.device, dtype=torch.int8)
        q_scale = torch.empty(h.shape[:-1], device=h.device, dtype=torch.float32)
        d.q, d.q_scale, d.q_stride = q.data_ptr(), q_scale.data_ptr(), pitch
        normed = (q if pitch == width else q[..., :width], q_scale)
    elif before:
        normed = torch.empty_like(residual)
        d.normed = normed.data_ptr()
    if want_stats:
        stats = torch.empty(rows, 4, device=h.device, dtype=torch.float32)
        d.stats = stats.data_ptr()
    if rows:
        hip.call('spi_norm_residual_fwd', ctypes.byref(d), hip.stream())
    return stream, normed, stats


class _NormResidual(torch.autograd.Function):
    @staticmethod
    def forward(ctx, cfg, h, residual, gate, *weights):
        stream, normed, stats = _forward(cfg, h, residual, gate, weights, True)
        ctx.cfg = cfg
        ctx.save_for_backward(stats, h, residual, gate, *weights)
        ctx.set_materialize_grads(False)
        return stream, normed

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_stream, d_normed):
        stats, h, residual, gate, *weights = ctx.saved_tensors
        cfg, need = ctx.cfg, ctx.needs_input_grad[1:]
        if d_stream is None and d_normed is None:
            return (None,) * 8
        if d_normed is None:                             # (only the stream was used: its norm has no part in the gradients)
            cfg = cfg[:7] + (False,) + cfg[8:]
            weights = weights[:2] + [None, None]
            need = need[:5] + (False, False)
        inputs = (h, residual, gate, *weights)
        return (None, *hip.on(h.get_device(), _backward, cfg, need, stats, inputs, d_stream, d_normed))


def _backward(cfg, need, stats, inputs, d_stream, d_normed):
    if cfg[0] == 0:
        return [torch.zeros_like(t) if n else None for t, n in zip(inputs, need)]
    h, residual, gate, *weights = inputs
    grads = [torch.empty_like(t) if n else None for t, n in zip(inputs, need)]
    d = _desc(cfg, h, residual, gate, weights)
    d.stats = stats.data_ptr()
    if d_stream is not None:
        d_stream = d_stream.contiguous()
        d.d_stream = d_stream.data_ptr()
    if d_normed is not None:
        d_normed = d_normed.contiguous()
        d.d_normed = d_normed.data_ptr()
    d.d_h, d.d_residual, d.d_gate, d.d_post_weight, d.d_post_bias, d.d_pre_weight, d.d_pre_bias = map(_p, grads)
    ref = ctypes.byref(d)
    nbytes = hip.lib().spi_norm_residual_bwd_workspace(ref)
    workspace = torch.empty(nbytes, device=h.device, dtype=torch.uint8)
    d.workspace, d.workspace_bytes = workspace.data_ptr(), nbytes
    hip.call('spi_norm_residual_bwd', ref, hip.stream())
    return grads


def _gate_mode(h, gate):
    """-> (mode, rows that share a gate vector)"""
    if gate is None:
        return _GATE_NONE, 1
    width = h.shape[-1]
    if gate.ndim >= 1 and gate.shape[-1] == width:
        if gate.numel() == width:
            return _GATE_CHANNEL, 1
        if gate.shape == h.shape:
            return _GATE_FULL, 1
        if h.ndim >= 3 and gate.shape[0] == h.shape[0] and gate.shape[1:-1].numel() == 1 and (gate.ndim == 2 or gate.ndim == h.ndim):
            rows = h.shape[1:-1].numel()
            return (_GATE_SAMPLE, rows) if rows > 1 else (_GATE_FULL, 1)
    raise ValueError(f'gate {tuple(gate.shape)} is neither one vector of {width}, nor one for each sample, nor one value for each of {tuple(h.shape)}')


def norm_residual(h, residual, gate=None, scale=1.0, post_weight=None, post_bias=None, pre_weight=None, pre_bias=None, norm='rms', where='both', eps=1e-8,
                  gate_act='linear', quantize=False):
    """-> ``(stream, normed)``, see the module's text.

    h, residual   [..., C], one type of fp32 / fp16 / bf16, C <= 32768 (<= 8192 where gradients are wanted)
    gate          None, [C], one vector per sample ([B, C] or [B, 1, .., C] for rows [B, .., C]) or the shape of h; through ``gate_act``: 'linear', 'tanh', 'sigmoid'
    *_weight      [C], wanted for the norms that ``where`` ('both', 'before', 'after' the block) asks for; biases are optional.  Weights and gate: fp32 or h's type
    quantize      (inference) ``normed`` is ``(q, q_scale)``: int8 rows, 16-byte aligned, and their fp32 scales, as ``linear_int8.quantize_rows`` gives them
    """
    if norm not in ('rms', 'layer'):
        raise ValueError(f'norm={norm!r}: rms or layer')
    if where not in ('both', 'before', 'after'):
        raise ValueError(f'where={where!r}: both, before or after')
    if gate_act not in _GATE_ACTS:
        raise ValueError(f'gate_act={gate_act!r}: {", ".join(_GATE_ACTS)}')
    if not eps > 0:
        raise ValueError(f'eps={eps}: has to be positive (a row of zeros has no norm)')
    after, before = where != 'before', where != 'after'
    if h.ndim < 1 or h.shape != residual.shape or h.dtype != residual.dtype:
        raise ValueError(f'h {tuple(h.shape)} {h.dtype} and residual {tuple(residual.shape)} {residual.dtype} have to be alike')
    if h.dtype not in hip.ROW_DTYPES:
        raise TypeError(f'rows of {h.dtype}: float32, float16 or bfloat16')
    width = h.shape[-1]
    if not 1 <= width <= MAX_WIDTH:
        raise ValueError(f'rows of {width} values: 1 to {MAX_WIDTH}')
    if (post_weight is not None) != after or (pre_weight is not None) != before:
        raise ValueError(f'where={where!r} wants ' + ' and '.join(n for n, on in (('post_weight', after), ('pre_weight', before)) if on) + ', and no others')
    if (post_bias is not None and not after) or (pre_bias is not None and not before):
        raise ValueError(f'where={where!r}: a bias without its norm')
    if quantize and not before:
        raise ValueError("quantize: where='after' has no normed rows")
    weights = (post_weight, post_bias, pre_weight, pre_bias)
    kind = (post_weight if after else pre_weight).dtype
    if kind is not h.dtype and kind is not torch.float32:
        raise TypeError(f'norm weights of {kind}: float32 or {h.dtype}')
    if gate is not None and gate.dtype is not h.dtype and gate.dtype is not torch.float32:
        raise TypeError(f'gate of {gate.dtype}: float32 or {h.dtype}')
    vector = (width,)
    for t in weights:
        if t is not None:
            if t.shape != vector:
                raise ValueError(f'a norm weight of {tuple(t.shape)} for rows of {width}')
            if t.dtype is not kind:
                raise TypeError(f'norm weights of {kind} and {t.dtype}: one type for all')
    mode, per_sample = _gate_mode(h, gate)
    device = hip.same_device(h, residual, gate, *weights)
    wants_grad = hip.records(h, residual, gate, *weights)             # (forward-mode tangents end in an error of the autograd function, which has none)
    if wants_grad and quantize:
        raise RuntimeError('norm_residual: rounded rows have no gradient; call quantize=True under torch.no_grad() or on tensors that need none')
    if wants_grad and width > MAX_WIDTH_BACKWARD:
        raise ValueError(f'rows of {width} values: gradients are provided up to {MAX_WIDTH_BACKWARD}')
    h, residual, gate, *weights = [t if t is None else t.contiguous() for t in (h, residual, gate) + weights]
    cfg = (h.numel() // width, width, per_sample, mode, _ba.activation_funcs[gate_act][0], norm == 'layer', after, before, float(scale), float(eps))
    if wants_grad:
        return hip.on(device, _NormResidual.apply, cfg, h, residual, gate, *weights)
    return hip.on(device, _forward, cfg, h, residual, gate, weights, False, quantize)[:2]
