"""64-bit statements of the row operators (norm_residual, linear_int8, grouped_linear) and the bounds their kernels are held to.

Bounds.  Every kernel computes in fp32 and rounds a result to its type once: |out - exact| <= u |exact| + n * 2^-24 * mag, with u = eps / 2 of the type, mag the sum of
the magnitudes of the terms the result is made of, and n the number of fp32 roundings that can pile up on the longest path to it."""
import torch

U32 = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def check(out, ref, mag, n, what):
    """|out - ref| <= u |ref| + n 2^-24 mag, value by value (a value too small for the type's normal range: to its smallest step)"""
    u, tiny = half_step(out.dtype), torch.finfo(out.dtype).smallest_normal * torch.finfo(out.dtype).eps
    out, ref = out.detach().double().cpu(), ref.detach().double().cpu()
    assert out.shape == ref.shape, (what, out.shape, ref.shape)
    bound = u * ref.abs() + n * U32 * (1 + u) * mag.detach().double().cpu() + tiny
    off = (out - ref).abs()
    assert torch.isfinite(out).all(), f'{what}: not finite'
    worst = (off / bound).max().item() if out.numel() else 0.0
    assert worst <= 1.0, f'{what}: {worst:.2f} times the bound (largest difference {off.max().item():.3e})'


# ---- norms -------------------------------------------------------------------------------------------------------------------------------
def norm_rows(x, w, b, layer, eps):
    m = x.mean(-1, keepdim=True) if layer else torch.zeros_like(x[..., :1])
    y = (x - m) / torch.sqrt(((x - m) ** 2).mean(-1, keepdim=True) + eps) * w
    return y if b is None else y + b


def gate_act(name, g):
    return {'linear': lambda v: v, 'tanh': torch.tanh, 'sigmoid': torch.sigmoid}[name](g)


def norm_residual(h, res, gate, scale, pw, pb, qw, qb, norm, where, eps, act):
    layer = norm == 'layer'
    z = h if where == 'before' else norm_rows(h, pw, pb, layer, eps)
    g = 1.0 if gate is None else gate_act(act, gate.reshape(h.shape[0], *([1] * (h.ndim - 2)), h.shape[-1]) if gate.ndim == 2 and h.ndim > 2 and gate.shape[0] > 1 else gate)
    s = res + scale * g * z
    return s, None if where == 'after' else norm_rows(s, qw, qb, layer, eps)


def norm_magnitudes(h, res, gate, scale, pw, pb, qw, qb, norm, where, eps, act, ds=None, dy=None):
    """What the results (and, given ds, the gradients) are made of, with every term's magnitude.  A norm of x: |x| + mean|x| over the deviation, times the weight."""
    layer = norm == 'layer'

    def unit(x):
        m = x.mean(-1, keepdim=True) if layer else 0.0
        r = 1 / torch.sqrt(((x - m) ** 2).mean(-1, keepdim=True) + eps)
        return (x - m) * r, (x.abs() + (x.abs().mean(-1, keepdim=True) if layer else 0.0)) * r, r
    zero = lambda b: 0.0 if b is None else b.abs()  # noqa: E731
    hat1, hmag, r1 = unit(h)
    zmag = h.abs() if where == 'before' else hmag * pw.abs() + zero(pb)
    g = torch.ones_like(h[..., :1]) if gate is None else gate_act(act, gate.reshape(h.shape[0], *([1] * (h.ndim - 2)), h.shape[-1]) if gate.ndim == 2 and h.ndim > 2 and
                                                                  gate.shape[0] > 1 else gate)
    smag = res.abs() + abs(scale) * g.abs() * zmag
    out = dict(stream=smag)
    if where != 'after':
        s, _ = norm_residual(h, res, gate, scale, pw, pb, qw, qb, norm, where, eps, act)
        shat, _, r2 = unit(s)
        own = (smag + (smag.mean(-1, keepdim=True) if layer else 0.0)) * r2
        # (an error of the stream moves its deviation too: at most by its share of the row's mean square)
        shmag = own + shat.abs() * (own * shat.abs()).mean(-1, keepdim=True)
        out['normed'] = shmag * qw.abs() + zero(qb)
    if ds is None:
        return out
    t = ds.abs()
    if where != 'after':
        u = dy.abs() * qw.abs()
        t = t + r2 * (u + shmag * (u * shmag).mean(-1, keepdim=True) + (u.mean(-1, keepdim=True) if layer else 0.0))
        out['pre_weight'], out['pre_bias'] = (dy.abs() * shmag), dy.abs()
    out['residual'] = t
    out['gate'] = abs(scale) * zmag * t
    dz = abs(scale) * g.abs() * t
    if where != 'before':
        out['post_weight'], out['post_bias'] = dz * hmag, dz
        v = dz * pw.abs()
        dz = r1 * (v + hmag * (v * hmag).mean(-1, keepdim=True) + (v.mean(-1, keepdim=True) if layer else 0.0))
    out['h'] = dz
    return out


# ---- 8-bit integers ----------------------------------------------------------------------------------------------------------------------
def quantize(x):
    """(q, scale) as 64-bit numbers; the scale and the quotient are rounded to 32 bits, as the definition says (a 64-bit quotient of 32-bit numbers rounds to the
    32-bit quotient)"""
    x = x.double()
    amax = x.abs().amax(-1, keepdim=True)
    scale = (amax / 127).float().double()
    q = torch.where(scale > 0, torch.round((x / torch.where(scale > 0, scale, 1.0)).float()).double().clamp(-127, 127), 0.0)
    bad = ~torch.isfinite(x).all(-1, keepdim=True)
    return torch.where(bad, 0.0, q), torch.where(bad, float('nan'), scale)[..., 0]


def activation(name, x, alpha=0.2):
    import torch.nn.functional as F
    return {'linear': lambda v: v, 'relu': torch.relu, 'lrelu': lambda v: torch.where(v > 0, v, alpha * v), 'tanh': torch.tanh, 'sigmoid': torch.sigmoid, 'elu': F.elu,
            'selu': F.selu, 'softplus': lambda v: torch.log1p(torch.exp(-v.abs())) + v.clamp_min(0), 'swish': lambda v: v * torch.sigmoid(v)}[name](x)


# ---- groups ------------------------------------------------------------------------------------------------------------------------------
def grouped(x, w, b, offsets, gain):
    y, mag = x.new_zeros(x.shape[0], w.shape[1]), x.new_zeros(x.shape[0], w.shape[1])
    for e in range(w.shape[0]):
        s = slice(offsets[e], offsets[e + 1])
        y[s] = gain * (x[s] @ w[e].T) + (0 if b is None else b[e])
        mag[s] = abs(gain) * (x[s].abs() @ w[e].abs().T) + (0 if b is None else b[e].abs())
    return y, mag


def grouped_gradients(x, w, offsets, gain, dy):
    dx, dw, db = torch.zeros_like(x), torch.zeros_like(w), w.new_zeros(w.shape[:2])
    mx, mw, mb = torch.zeros_like(x), torch.zeros_like(w), w.new_zeros(w.shape[:2])
    for e in range(w.shape[0]):
        s = slice(offsets[e], offsets[e + 1])
        dx[s], mx[s] = gain * (dy[s] @ w[e]), abs(gain) * (dy[s].abs() @ w[e].abs())
        dw[e], mw[e] = gain * (dy[s].T @ x[s]), abs(gain) * (dy[s].abs().T @ x[s].abs())
        db[e], mb[e] = dy[s].sum(0), dy[s].abs().sum(0)
    return (dx, dw, db), (mx, mw, mb)
