"""GPU tests of the row operators: norm_residual, quantize_rows / linear_int8, grouped_linear, against 64-bit statements of their definitions."""
import pytest
import torch

import row_ops_ref as ref

pytestmark = pytest.mark.gpu
DEV = 'cuda'
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = [F32, F16, BF16]
ids = lambda v: str(v).replace('torch.', '') if isinstance(v, torch.dtype) else None  # noqa: E731


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def randn(g, *shape, dtype=F32, scale=1.0):
    return (torch.randn(*shape, device=DEV, generator=g) * scale).to(dtype)


# ---- norm_residual -----------------------------------------------------------------------------------------------------------------------
def norm_inputs(shape, dtype, norm, where, gate, bias, seed=0, wdtype=F32):
    g, c = gen(seed), shape[-1]
    vec = lambda on, base: (base + 0.2 * randn(g, c)).to(wdtype) if on else None  # noqa: E731
    gates = {None: None, 'channel': (c,), 'sample': (shape[0],) + (1,) * (len(shape) - 2) + (c,), 'sample2': (shape[0], c), 'full': shape}
    return dict(h=randn(g, *shape, dtype=dtype, scale=3.0), residual=randn(g, *shape, dtype=dtype),
                gate=None if gate is None else randn(g, *gates[gate], dtype=wdtype if gate == 'channel' else dtype),
                post_weight=vec(where != 'before', 1.0), post_bias=vec(bias and where != 'before', 0.0), pre_weight=vec(where != 'after', 1.0),
                pre_bias=vec(bias and where != 'after', 0.0))


ORDER = ('h', 'residual', 'gate', 'scale', 'post_weight', 'post_bias', 'pre_weight', 'pre_bias')


def norm_case(inputs, scale, norm, where, eps, act, ds=None, dy=None, fn=ref.norm_magnitudes):
    v = [scale if k == 'scale' else (None if inputs[k] is None else inputs[k].detach().double()) for k in ORDER]
    return fn(*v, norm, where, eps, act, *([] if ds is None else [ds.double(), None if dy is None else dy.double()]))


def run_norm(inputs, scale, norm, where, eps, act, **kw):
    from spi_amd.torch_utils.ops import norm_residual as op
    return op.norm_residual(inputs['h'], inputs['residual'], gate=inputs['gate'], scale=scale, post_weight=inputs['post_weight'], post_bias=inputs['post_bias'],
                            pre_weight=inputs['pre_weight'], pre_bias=inputs['pre_bias'], norm=norm, where=where, eps=eps, gate_act=act, **kw)


def piled(width):
    """fp32 roundings on the way to a normalised value: a thread's own chain (at most 32 values), the tree over 1024 threads, and a dozen elementary steps, for each of
    two norms"""
    return 2 * (min(32, -(-width // 64)) + 10 + 16)


def check_norm(inputs, scale, norm, where, eps, act, what):
    s, y = run_norm(inputs, scale, norm, where, eps, act)
    rs, ry = norm_case(inputs, scale, norm, where, eps, act, fn=ref.norm_residual)
    mag = norm_case(inputs, scale, norm, where, eps, act)
    n = piled(inputs['h'].shape[-1])
    ref.check(s, rs, mag['stream'], n, f'{what} stream')
    if where == 'after':
        assert y is None
    else:
        ref.check(y, ry, mag['normed'], n, f'{what} normed')


@pytest.mark.parametrize('dtype', TYPES, ids=ids)
@pytest.mark.parametrize('shape', [(1, 1), (1, 512), (3, 7), (5, 130), (2, 3, 1003), (4, 2048), (2, 2, 4101), (3, 8192), (2, 20001), (1, 32768)])
def test_norm_forward_sizes(shape, dtype):
    for norm, where, gate in (('rms', 'both', 'channel'), ('layer', 'both', 'full')):
        check_norm(norm_inputs(shape, dtype, norm, where, gate, norm == 'layer'), 0.1, norm, where, 1e-6, 'linear', f'{norm} {shape}')


@pytest.mark.parametrize('where', ['both', 'before', 'after'])
@pytest.mark.parametrize('norm', ['rms', 'layer'])
@pytest.mark.parametrize('gate,act', [(None, 'linear'), ('channel', 'tanh'), ('sample', 'sigmoid'), ('sample2', 'linear'), ('full', 'tanh')])
def test_norm_forward_forms(norm, where, gate, act):
    for dtype, wdtype in ((F32, F32), (F16, F16), (BF16, F32)):
        check_norm(norm_inputs((3, 5, 200), dtype, norm, where, gate, True, wdtype=wdtype), -0.7, norm, where, 1e-8, act, f'{norm} {where} {gate}')


def check_norm_gradients(inputs, scale, norm, where, eps, act, what, seed=5):
    g, h = gen(seed), inputs['h']
    leaves = {k: v.clone().requires_grad_() for k, v in inputs.items() if v is not None}
    s, y = run_norm({k: leaves.get(k) for k in inputs}, scale, norm, where, eps, act)
    ds = randn(g, *h.shape, dtype=h.dtype)
    dy = None if y is None else randn(g, *h.shape, dtype=h.dtype)
    outs, grads = ([s], [ds]) if y is None else ([s, y], [ds, dy])
    got = dict(zip(leaves, torch.autograd.grad(outs, list(leaves.values()), grads)))
    wide = {k: v.detach().double().requires_grad_() for k, v in leaves.items()}
    rs, ry = ref.norm_residual(*[scale if k == 'scale' else wide.get(k) for k in ORDER], norm, where, eps, act)
    exact = dict(zip(wide, torch.autograd.grad([rs] if y is None else [rs, ry], list(wide.values()), [v.double() for v in grads])))
    mag = norm_case(inputs, scale, norm, where, eps, act, ds, dy)
    rows, width = h.numel() // h.shape[-1], h.shape[-1]
    n = 4 * piled(width)                 # the two sums of each norm's gradient, of values that carry the forward's roundings
    for k, v in got.items():
        assert v.dtype == leaves[k].dtype and v.shape == leaves[k].shape
        m, add = mag[k], 0
        if v.shape != h.shape:           # a sum over rows, of at most all of them in one chain
            while m.ndim > v.ndim:
                m = m.sum(0) if v.ndim == 1 else m.sum(tuple(range(1, m.ndim - 1)))
            for i in range(m.ndim):
                if v.shape[i] == 1 and m.shape[i] > 1:
                    m = m.sum(i, keepdim=True)
            add = rows
        ref.check(v, exact[k], m.expand(v.shape), n + add, f'{what} d_{k}')


@pytest.mark.parametrize('dtype', TYPES, ids=ids)
@pytest.mark.parametrize('shape', [(1, 1), (1, 512), (37, 7), (2, 3, 1003), (3, 700, 64), (2, 2, 2048), (3, 4101), (5, 8192)])
def test_norm_gradient_sizes(shape, dtype):
    for norm, gate in (('rms', 'channel'), ('layer', 'full')):
        check_norm_gradients(norm_inputs(shape, dtype, norm, 'both', gate, norm == 'layer'), 0.1, norm, 'both', 1e-6, 'linear', f'{norm} {shape}')


@pytest.mark.parametrize('where', ['both', 'before', 'after'])
@pytest.mark.parametrize('gate,act', [(None, 'linear'), ('channel', 'tanh'), ('sample', 'sigmoid'), ('sample2', 'linear'), ('full', 'tanh')])
def test_norm_gradient_forms(where, gate, act):
    for norm, dtype, wdtype in (('rms', F32, F32), ('layer', F16, F16), ('layer', BF16, F32)):
        check_norm_gradients(norm_inputs((3, 5, 200), dtype, norm, where, gate, True, wdtype=wdtype), -0.7, norm, where, 1e-6, act, f'{norm} {where} {gate}')


@pytest.mark.parametrize('samples,rows', [(1, 5000), (600, 3), (1500, 2), (7, 333)])
def test_norm_gradient_of_shared_gates(samples, rows):
    """more rows or samples than the backward has blocks: every sum is joined over several blocks, and a gate's stays within its sample"""
    check_norm_gradients(norm_inputs((samples, rows, 72), BF16, 'rms', 'both', 'sample', False), 0.3, 'rms', 'both', 1e-6, 'linear', f'{samples} x {rows}')
    check_norm_gradients(norm_inputs((samples, rows, 72), F32, 'layer', 'both', 'channel', True), 0.3, 'layer', 'both', 1e-6, 'tanh', f'{samples} x {rows}')


def test_norm_gradient_of_parts():
    """an unused result, leaves that want no gradient"""
    from spi_amd.torch_utils.ops.norm_residual import norm_residual
    i = norm_inputs((6, 96), F32, 'rms', 'both', 'channel', False)
    leaves = {k: v.clone().requires_grad_() for k, v in i.items() if v is not None}
    wide = {k: v.detach().double().requires_grad_() for k, v in leaves.items()}
    s, y = run_norm({k: leaves.get(k) for k in i}, 0.5, 'rms', 'both', 1e-6, 'linear')
    rs, ry = ref.norm_residual(*[0.5 if k == 'scale' else wide.get(k) for k in ORDER], 'rms', 'both', 1e-6, 'linear')
    for out, r in ((s, rs), (y, ry)):
        got = torch.autograd.grad(out.sum(), list(leaves.values()), retain_graph=True, allow_unused=True)
        exact = torch.autograd.grad(r.sum(), list(wide.values()), retain_graph=True, allow_unused=True)
        for k, a, b in zip(leaves, got, exact):
            if b is None:
                assert a is None or not a.any()
            else:
                assert (a.double() - b).abs().max() <= 1000 * ref.U32 * b.abs().max(), k        # (a few hundred roundings, see `piled`)
    only = i['h'].clone().requires_grad_()
    s, y = norm_residual(only, i['residual'], gate=i['gate'], post_weight=i['post_weight'], pre_weight=i['pre_weight'])
    (s.sum() + y.sum()).backward()
    assert only.grad is not None


def test_norm_gradients_match_differences():
    """difference quotients of the kernel's own forward; their truncation error is that of the same quotients in 64 bits"""
    i = norm_inputs((4, 33), F32, 'layer', 'both', 'full', True)
    g, step = gen(9), 2.0 ** -6
    cs, cy = randn(g, 4, 33).double(), randn(g, 4, 33).double()

    def loss(v, fn):
        s, y = fn(v)
        return (s.double() * cs).sum() + (y.double() * cy).sum()
    kernel = lambda v: run_norm(v, 0.5, 'layer', 'both', 1e-3, 'tanh')  # noqa: E731
    wide = lambda v: ref.norm_residual(*[0.5 if k == 'scale' else v[k] for k in ORDER], 'layer', 'both', 1e-3, 'tanh')  # noqa: E731
    leaves = {k: v.clone().requires_grad_() for k, v in i.items()}
    got = dict(zip(leaves, torch.autograd.grad(loss(leaves, kernel), list(leaves.values()))))
    mag = norm_case(i, 0.5, 'layer', 'both', 1e-3, 'tanh')
    noise = piled(33) * ref.U32 * ((mag['stream'] * cs.abs()).sum() + (mag['normed'] * cy.abs()).sum()).item()
    for k in i:
        d = randn(g, *i[k].shape)
        at = lambda sign, t: {**{n: v.to(t) for n, v in i.items()}, k: i[k].to(t) + sign * step * d.to(t)}  # noqa: E731
        quotient = ((loss(at(1, F32), kernel) - loss(at(-1, F32), kernel)) / (2 * step)).item()
        exact = ((loss(at(1, torch.float64), wide) - loss(at(-1, torch.float64), wide)) / (2 * step)).item()
        slope = (got[k].double() * d.double()).sum().item()
        w = {n: v.double().requires_grad_(n == k) for n, v in i.items()}
        true = (torch.autograd.grad(loss(w, wide), w[k])[0] * d.double()).sum().item()
        # (moving fp32 inputs by step * d rounds them: at most one rounding of each input, counted as one more of the forward's)
        assert abs(quotient - slope) <= abs(exact - true) + 2 * noise / step, (k, quotient, slope, exact, true, noise)


def test_norm_quantized_rows():
    for dtype, shape in ((F32, (5, 512)), (BF16, (2, 3, 1003)), (F16, (4, 2050))):
        i = norm_inputs(shape, dtype, 'rms', 'both', 'channel', False)
        s, (q, scale) = run_norm(i, 0.1, 'rms', 'both', 1e-6, 'linear', quantize=True)
        s2, y = run_norm({k: (v.float() if v is not None and k in ('h', 'residual') else v) for k, v in i.items()}, 0.1, 'rms', 'both', 1e-6, 'linear')
        assert torch.equal(s, s2.to(dtype)) and q.shape == i['h'].shape and scale.shape == shape[:-1]
        assert q.stride(-2) % 16 == 0 and q.data_ptr() % 16 == 0
        rq, rscale = ref.quantize(y)               # of the rows in 32 bits, which have the same values
        if dtype == F32:                           # (the other types' fp32 rows are summed by other threads: a few roundings apart)
            assert torch.equal(q.double(), rq) and torch.equal(scale.double(), rscale)
        assert (scale.double() / rscale - 1).abs().max() <= piled(shape[-1]) * ref.U32
        assert (q.double() - rq).abs().max() <= 1 and (q.double() != rq).double().mean() < 1e-3


def test_norm_rows_stand_alone():
    """infinities and NaN stay in their rows, rows of zeros are finite, and the largest finite values do not overflow the stream"""
    i = norm_inputs((6, 256), F32, 'rms', 'both', 'full', False)
    clean = run_norm(i, 0.1, 'rms', 'both', 1e-6, 'linear')
    bad = {k: v.clone() if v is not None else None for k, v in i.items()}
    bad['h'][1, 3], bad['residual'][2, 255], bad['gate'][3, 0] = float('nan'), float('inf'), float('-inf')
    bad['h'][4], bad['residual'][4] = 0, 0
    s, y = run_norm(bad, 0.1, 'rms', 'both', 1e-6, 'linear')
    for k in (0, 5):
        assert torch.equal(s[k], clean[0][k]) and torch.equal(y[k], clean[1][k])
    assert torch.isnan(y[1]).all() and torch.isnan(y[2, 255]) and not torch.isfinite(y[3, 0])
    assert torch.equal(s[4], torch.zeros_like(s[4])) and torch.equal(y[4], torch.zeros_like(y[4]))
    _, (q, scale) = run_norm(bad, 0.1, 'rms', 'both', 1e-6, 'linear', quantize=True)
    assert torch.isnan(scale[1:4]).all() and torch.isfinite(scale[[0, 4, 5]]).all() and scale[4] == 0 and not q[1:5].any()


def test_norm_gradients_of_rows_with_nan():
    """a NaN row spoils its own gradients and the sums over rows that it is part of, and no other sample's"""
    i = norm_inputs((3, 5, 200), F32, 'rms', 'both', 'sample', False)
    i['h'][0, 0, 7] = float('nan')                                  # (the first row: what rows that a block has too few of read their statistics from)
    leaves = {k: v.clone().requires_grad_() for k, v in i.items() if v is not None}
    s, y = run_norm({k: leaves.get(k) for k in i}, 0.1, 'rms', 'both', 1e-6, 'linear')
    ds, dy = randn(gen(1), 3, 5, 200), randn(gen(2), 3, 5, 200)
    got = dict(zip(leaves, torch.autograd.grad([s, y], list(leaves.values()), [ds, dy])))
    clean = {k: (v[1:].clone() if v.ndim == 3 else v.clone()).requires_grad_() for k, v in i.items() if v is not None}
    s, y = run_norm({k: clean.get(k) for k in i}, 0.1, 'rms', 'both', 1e-6, 'linear')
    want = dict(zip(clean, torch.autograd.grad([s, y], list(clean.values()), [ds[1:], dy[1:]])))
    for k in ('h', 'residual', 'gate'):
        assert torch.isnan(got[k][0]).any() and torch.equal(got[k][1:], want[k]), k
    assert torch.isfinite(got['h'][0, 1:]).all() and torch.isfinite(got['residual'][0, 1:]).all() and torch.isnan(got['pre_weight']).any()


def test_norm_strides_empty_and_repeat():
    i = norm_inputs((8, 12, 64), BF16, 'layer', 'both', 'full', True)
    want = run_norm(i, 0.1, 'layer', 'both', 1e-6, 'linear')
    strange = {k: (v.transpose(0, 1).contiguous().transpose(0, 1) if v is not None and v.ndim == 3 else v) for k, v in i.items()}
    strange['pre_weight'] = torch.stack([i['pre_weight'], i['pre_weight']], 1)[:, 0]
    assert not strange['h'].is_contiguous() and not strange['pre_weight'].is_contiguous()
    for a, b in zip(run_norm(strange, 0.1, 'layer', 'both', 1e-6, 'linear'), want):
        assert torch.equal(a, b)
    odd = {k: (torch.cat([v.flatten()[:1], v.flatten()])[1:].view_as(v) if v is not None else None) for k, v in i.items()}      # rows that begin on odd places
    assert odd['h'].data_ptr() % 16
    for a, b in zip(run_norm(odd, 0.1, 'layer', 'both', 1e-6, 'linear'), want):
        assert torch.equal(a, b)
    e = norm_inputs((0, 64), F32, 'rms', 'both', 'channel', False)
    leaves = {k: v.clone().requires_grad_() for k, v in e.items() if v is not None}
    s, y = run_norm({k: leaves.get(k) for k in e}, 0.1, 'rms', 'both', 1e-6, 'linear')
    (s.sum() + y.sum()).backward()
    assert s.shape == y.shape == (0, 64) and all(not v.grad.any() for v in leaves.values())
    grads = []
    for _ in range(2):
        leaves = {k: v.clone().requires_grad_() for k, v in norm_inputs((900, 300), F32, 'rms', 'both', 'channel', False).items() if v is not None}
        s, y = run_norm({k: leaves.get(k) for k in e}, 0.1, 'rms', 'both', 1e-6, 'linear')
        grads.append(torch.autograd.grad((s * s).sum() + (y * y * y).sum(), list(leaves.values())))
    assert all(torch.equal(a, b) for a, b in zip(*grads))          # the sums over rows have one order


def test_norm_rows_behind_32_bits():
    rows, width = 540_000, 4096                                     # 2.2e9 values
    g = gen(3)
    h = torch.zeros(rows, width, device=DEV, dtype=BF16)
    r = torch.zeros(rows, width, device=DEV, dtype=BF16)
    h[-3:], r[-3:] = randn(g, 3, width, dtype=BF16), randn(g, 3, width, dtype=BF16)
    w = torch.ones(width, device=DEV)
    i = dict(h=h, residual=r, gate=None, post_weight=w, post_bias=None, pre_weight=w, pre_bias=None)
    s, y = run_norm(i, 0.5, 'rms', 'both', 1e-6, 'linear')
    last = run_norm({**i, 'h': h[-3:].clone(), 'residual': r[-3:].clone()}, 0.5, 'rms', 'both', 1e-6, 'linear')
    assert torch.equal(s[-3:], last[0]) and torch.equal(y[-3:], last[1]) and not s[:-3].any() and not y[:-3].any()


def test_more_narrow_rows_than_a_launch_has_threads():
    from spi_amd.torch_utils.ops.linear_int8 import quantize_rows
    rows = (1 << 26) + 5                                            # a wave each: more than 2^32 lanes
    x = torch.zeros(rows, 2, device=DEV, dtype=F16)
    x[-7:], x[:3] = randn(gen(4), 7, 2, dtype=F16), 1
    w = torch.ones(2, device=DEV)
    i = dict(h=x, residual=x, gate=None, post_weight=w, post_bias=None, pre_weight=w, pre_bias=None)
    s, y = run_norm(i, 0.5, 'rms', 'both', 1e-6, 'linear')
    q, scale = quantize_rows(x)
    for part in (slice(0, 9), slice(rows - 9, rows)):
        few = x[part].clone()
        fs, fy = run_norm({**i, 'h': few, 'residual': few}, 0.5, 'rms', 'both', 1e-6, 'linear')
        fq, fscale = quantize_rows(few)
        assert torch.equal(s[part], fs) and torch.equal(y[part], fy) and torch.equal(q[part], fq) and torch.equal(scale[part], fscale) and fs.any()
    assert not s[3:-7].any() and not y[3:-7].any() and not scale[3:-7].any()


# ---- 8-bit integers ----------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize('dtype', TYPES, ids=ids)
@pytest.mark.parametrize('rows,width', [(1, 1), (3, 15), (7, 512), (2, 1003), (33, 2048), (5, 8192), (2, 100_001)])
def test_quantize_rows(rows, width, dtype):
    from spi_amd.torch_utils.ops.linear_int8 import quantize_rows
    x = randn(gen(1), rows, width, dtype=dtype) * torch.logspace(-3, 3, rows, device=DEV)[:, None].to(dtype)
    if rows > 2:
        x[1] = 0
        x[2, width // 2] = float('nan')
    q, scale = quantize_rows(x)
    rq, rscale = ref.quantize(x)
    assert torch.equal(q.double(), rq)
    assert torch.equal(torch.isnan(scale.double()), torch.isnan(rscale)) and torch.equal(scale.double().nan_to_num(1e9), rscale.nan_to_num(1e9))
    pitch = q.stride(0) if rows > 1 else width
    if rows > 1:
        assert pitch % 16 == 0
        buf = q.as_strided((rows, pitch), (pitch, 1))
        assert not buf[:, width:].any()


def test_quantize_rows_extremes():
    from spi_amd.torch_utils.ops.linear_int8 import quantize_rows
    x = torch.zeros(5, 40, device=DEV)
    x[0, :3] = torch.tensor([1e-45, 2e-45, -3e-45], device=DEV)      # subnormal
    x[1, :2] = torch.tensor([3.4e38, -1.0], device=DEV)
    x[2, :4] = torch.tensor([127.0, 0.5, 1.5, -2.5], device=DEV)     # ties go to the even number
    x[3, 0] = float('inf')
    q, scale = quantize_rows(x)
    rq, rscale = ref.quantize(x)
    assert torch.equal(q.double(), rq) and torch.isnan(scale[3]) and scale[4] == 0
    assert q[2, :4].tolist() == [127, 0, 2, -2] and q[1, :2].tolist() == [127, 0]


def int8_weights(g, n, k):
    from spi_amd.torch_utils.ops.linear_int8 import quantize_rows
    return quantize_rows(randn(g, n, k))


def int8_reference(q, scale, wq, ws, bias, act, gain, clamp):
    acc = q.double() @ wq.double().T
    pre = acc * (scale.double()[..., None] * ws.double())
    mag = pre.abs()
    if bias is not None:
        pre, mag = pre + bias.double(), mag + bias.double().abs()
    y = ref.activation(act, pre) * gain
    mag = (mag + ref.activation(act, pre).abs()) * gain            # every activation's slope is at most 1.76 (selu); counted in n
    if clamp is not None:
        y = y.clamp(-clamp, clamp)
    return y, mag


@pytest.mark.parametrize('m,n,k', [(1, 512, 512), (1, 1, 1), (2, 33, 17), (14, 512, 2048), (16, 100, 64), (4, 40, 4001), (3, 4099, 33), (17, 4096, 512), (64, 65, 300), (65, 64, 4100), (100, 333, 1003),
                                   (257, 512, 129), (600, 512, 512), (1111, 770, 1031)])
def test_linear_int8_sizes(m, n, k):
    from spi_amd.torch_utils.ops.linear_int8 import linear_int8
    g = gen(m + n + k)
    wq, ws = int8_weights(g, n, k)
    bias = randn(g, n)
    for dtype in TYPES:
        x = randn(g, m, k, dtype=dtype)
        y = linear_int8(x, wq, ws, bias=bias, act='lrelu')
        r, mag = int8_reference(*ref.quantize(x), wq, ws, bias, 'lrelu', 2 ** 0.5, None)
        assert y.dtype == dtype
        ref.check(y, r, mag, 8, f'{m} x {n} x {k}')


@pytest.mark.parametrize('act', ['linear', 'relu', 'lrelu', 'tanh', 'sigmoid', 'elu', 'selu', 'softplus', 'swish'])
def test_linear_int8_activations(act):
    from spi_amd.torch_utils.ops.linear_int8 import linear_int8, quantize_rows
    from spi_amd.torch_utils.ops.bias_act import def_gain
    g = gen(4)
    wq, ws = int8_weights(g, 48, 100)
    x = randn(g, 2, 9, 100) * 0.3
    q, s = quantize_rows(x)
    for clamp in (None, 0.7):
        a = linear_int8(q, wq, ws, x_scale=s, act=act, clamp=clamp)
        assert torch.equal(a, linear_int8(x, wq, ws, act=act, clamp=clamp)) and a.shape == (2, 9, 48)
        r, mag = int8_reference(q, s, wq, ws, None, act, def_gain(act), clamp)
        ref.check(a, r, mag + def_gain(act), 24, act)              # exp and log of the device library: within a few roundings of values up to 1
    a = linear_int8(q, wq, ws, x_scale=s, act='lrelu', alpha=0.01, gain=3.0, out_dtype=BF16)
    r = torch.where((p := int8_reference(q, s, wq, ws, None, 'linear', 1.0, None)[0]) > 0, p, 0.01 * p) * 3
    ref.check(a, r, r.abs(), 8, 'alpha and gain')


def test_linear_int8_exact_sums():
    """the largest products and the longest sum that the call takes: the integers stay exact"""
    from spi_amd.torch_utils.ops.linear_int8 import MAX_IN_FEATURES, linear_int8
    k = MAX_IN_FEATURES
    q = torch.full((2, k), 127, device=DEV, dtype=torch.int8)
    q[1, ::2] = -127
    w = torch.full((3, k), 127, device=DEV, dtype=torch.int8)
    w[1] = -127
    w[2, ::2] = -127
    one = torch.ones(3, device=DEV)
    y = linear_int8(q, w, one, x_scale=one[:2])
    r = q.cpu().long() @ w.cpu().long().T
    assert torch.equal(y.cpu(), r.float())


def test_linear_int8_rows_stand_alone_and_strides():
    from spi_amd.torch_utils.ops.linear_int8 import linear_int8, quantize_rows
    g = gen(6)
    for m in (5, 70, 300):
        x = randn(g, m, 96)
        wq, ws = int8_weights(g, 80, 96)
        want = linear_int8(x, wq, ws)
        bad = x.clone()
        bad[1, 5], bad[3, 95] = float('nan'), float('-inf')
        y = linear_int8(bad, wq, ws)
        keep = [i for i in range(m) if i not in (1, 3)]
        assert torch.equal(y[keep], want[keep]) and torch.isnan(y[1]).all() and torch.isnan(y[3]).all()
        wide = torch.cat([x, x], 1)
        assert torch.equal(linear_int8(wide[:, :96], wq, ws), want)                              # rows apart
        assert torch.equal(linear_int8(x.t().contiguous().t(), wq, ws), want)                    # columns adjacent
        loose = torch.cat([wq.new_zeros(80, 3), wq, wq.new_full((80, 2), 7)], 1)[:, 3:99]         # weights that begin on odd bytes, with others behind them
        assert torch.equal(linear_int8(x, loose, ws), want)
        padded = torch.full((80, 112), 99, device=DEV, dtype=torch.int8)
        padded[:, :90] = wq[:, :90]                                                              # aligned rows whose padding is not zero
        assert torch.equal(linear_int8(x[:, :90], padded[:, :90], ws), linear_int8(x[:, :90], wq[:, :90].contiguous(), ws))
        assert torch.equal(linear_int8(x[:1].expand(4, 96), wq, ws), want[:1].expand(4, 80))
        q, s = quantize_rows(x)
        for width, pitch in ((90, 112), (96, 97)):                                               # ... and int8 rows whose padding is not zero, or that begin on odd bytes
            rows = torch.full((m, pitch), 99, device=DEV, dtype=torch.int8)
            rows[:, :width] = q[:, :width]
            assert torch.equal(linear_int8(rows[:, :width], padded[:, :width] if width == 90 else wq, ws, x_scale=s),
                               linear_int8(q[:, :width].contiguous(), wq[:, :width].contiguous(), ws, x_scale=s))
    assert linear_int8(x[:0], wq, ws).shape == (0, 80)


def test_linear_int8_rows_behind_32_bits():
    from spi_amd.torch_utils.ops.linear_int8 import linear_int8
    m, k, n = 540_000, 4096, 16
    g = gen(8)
    q = torch.zeros(m, k, device=DEV, dtype=torch.int8)
    q[-2:] = torch.randint(-127, 128, (2, k), device=DEV, generator=g, dtype=torch.int8)
    wq, ws = int8_weights(g, n, k)
    s = torch.ones(m, device=DEV)
    y = linear_int8(q, wq, ws, x_scale=s)
    assert torch.equal(y[-2:], linear_int8(q[-2:].clone(), wq, ws, x_scale=s[:2])) and not y[:-2].any() and y[-2:].any()


# ---- groups ------------------------------------------------------------------------------------------------------------------------------
def check_grouped(sizes, k, n, dtype, seed=0, head=0, behind=0, bias=True, gain=0.37):
    from spi_amd.torch_utils.ops.grouped_linear import grouped_linear
    g, e = gen(seed), len(sizes)
    offsets = [head]
    for s in sizes:
        offsets.append(offsets[-1] + s)
    t = offsets[-1] + behind
    x, w, dy = randn(g, t, k, dtype=dtype).requires_grad_(), randn(g, e, n, k, dtype=dtype).requires_grad_(), randn(g, t, n, dtype=dtype)
    b = randn(g, e, n, dtype=dtype).requires_grad_() if bias else None
    o = torch.tensor(offsets, device=DEV, dtype=torch.int32)
    y = grouped_linear(x, w, o, bias=b, gain=gain)
    x64, w64 = x.detach().double(), w.detach().double()
    r, mag = ref.grouped(x64, w64, None if b is None else b.detach().double(), offsets, gain)
    what = f'{sizes} {k} -> {n} {dtype}'
    ref.check(y, r, mag, 2 * k + 8, f'{what} y')
    got = torch.autograd.grad(y, [v for v in (x, w, b) if v is not None], dy)
    exact, mags = ref.grouped_gradients(x64, w64, offsets, gain, dy.double())
    longest = max(sizes)
    for v, a, m, c, name in zip(got, exact, mags, (n, longest, longest), ('dx', 'dw', 'db')):
        ref.check(v, a, m, 2 * c + 8, f'{what} {name}')
    assert not y[:head].any() and not y[offsets[-1]:].any() and not got[0][:head].any() and not got[0][offsets[-1]:].any()


@pytest.mark.parametrize('dtype', TYPES, ids=ids)
@pytest.mark.parametrize('sizes,k,n', [([1], 1, 1), ([4, 4, 6], 512, 512), ([0, 3, 0], 64, 48), ([17, 1, 64, 0, 65], 128, 96), ([5, 130, 2], 515, 71), ([300, 257], 200, 264),
                                       ([1000, 24], 136, 520), ([33] * 40, 40, 24), ([600, 3, 700], 1031, 333)])
def test_grouped_sizes(sizes, k, n, dtype):
    check_grouped(sizes, k, n, dtype)


@pytest.mark.parametrize('dtype', TYPES, ids=ids)
def test_grouped_rows_of_no_group(dtype):
    check_grouped([9, 0, 70], 72, 80, dtype, head=67, behind=130, bias=False)
    check_grouped([0, 0], 32, 32, dtype, head=3, behind=4)
    check_grouped([2] * 300, 16, 8, dtype, head=1, behind=1)          # more groups than a wave has lanes


def test_grouped_empty_call_and_no_grad():
    from spi_amd.torch_utils.ops.grouped_linear import grouped_linear
    g = gen(2)
    w, b = randn(g, 2, 8, 16).requires_grad_(), randn(g, 2, 8).requires_grad_()
    x = randn(g, 0, 16).requires_grad_()
    y = grouped_linear(x, w, torch.zeros(3, device=DEV, dtype=torch.int32), bias=b)
    y.sum().backward()
    assert y.shape == (0, 8) and not w.grad.any() and not b.grad.any() and x.grad.shape == (0, 16)
    with torch.no_grad():
        assert not grouped_linear(randn(g, 4, 16), w, torch.tensor([0, 2, 4], device=DEV, dtype=torch.int32)).requires_grad


def test_grouped_reads_offsets_as_running_maximum():
    from spi_amd.torch_utils.ops.grouped_linear import grouped_linear
    g = gen(7)
    x, w, dy = randn(g, 50, 24).requires_grad_(), randn(g, 5, 40, 24).requires_grad_(), randn(g, 50, 40)
    for wild, means in (([-7, 10, 4, 30, 10 ** 9, 20], [0, 10, 10, 30, 50, 50]), ([60, 70, 80, 90, 100, 110], [50] * 6), ([-2 ** 31, -5, -4, -3, -2, -1], [0] * 6)):
        a, b = (grouped_linear(x, w, torch.tensor(o, device=DEV, dtype=torch.int32)) for o in (wild, means))
        assert torch.equal(a, b)
        for u, v in zip(torch.autograd.grad(a, [x, w], dy), torch.autograd.grad(b, [x, w], dy)):
            assert torch.equal(u, v)


@pytest.mark.parametrize('k,n', [(96, 72), (99, 75)])
def test_grouped_strides_and_rows_stand_alone(k, n):
    from spi_amd.torch_utils.ops.grouped_linear import grouped_linear
    g = gen(11)
    for dtype in TYPES:
        x, w = randn(g, 150, k, dtype=dtype), randn(g, 3, n, k, dtype=dtype)
        o = torch.tensor([0, 20, 90, 150], device=DEV, dtype=torch.int32)
        want = grouped_linear(x, w, o)
        assert torch.equal(grouped_linear(x.t().contiguous().t(), w.transpose(1, 2).contiguous().transpose(1, 2), o), want)
        odd = torch.cat([x.flatten()[:1], x.flatten()])[1:].view_as(x), torch.cat([w.flatten()[:1], w.flatten()])[1:].view_as(w)
        assert odd[0].data_ptr() % 16 and odd[1].data_ptr() % 16
        off = grouped_linear(*odd, o)
        r, mag = ref.grouped(x.double(), w.double(), None, o.tolist(), 1.0)
        ref.check(off, r, mag, 2 * k + 8, 'rows on odd places')
        bad = x.clone()
        bad[21, 7], bad[89, 0] = float('nan'), float('inf')
        y = grouped_linear(bad, w, o)
        keep = [i for i in range(150) if i not in (21, 89)]
        assert torch.equal(y[keep], want[keep]) and torch.isnan(y[21]).all() and not torch.isfinite(y[89]).any()
        # ... and in the sums over a group's rows they reach that group's gradients only
        xg, wg = bad.clone().requires_grad_(), w.clone().requires_grad_()
        dy = randn(g, 150, n, dtype=dtype)
        _, dw = torch.autograd.grad(grouped_linear(xg, wg, o), [xg, wg], dy)
        assert torch.isfinite(dw[0]).all() and torch.isfinite(dw[2]).all() and torch.isnan(dw[1, :, 7]).all()
        # a group's own weights, and gradients that come in, stay with their group and row, too
        spoiled = w.clone()
        spoiled[1, 3, 5] = float('nan')
        y = grouped_linear(x, spoiled, o)
        assert torch.equal(y[:20], want[:20]) and torch.equal(y[90:], want[90:]) and torch.isnan(y[20:90, 3]).all()
        xg, wg, bg = x.clone().requires_grad_(), w.clone().requires_grad_(), randn(g, 3, n, dtype=dtype).requires_grad_()
        first = torch.autograd.grad(grouped_linear(xg, wg, o, bias=bg), [xg, wg, bg], dy)
        dy[95, 2] = float('nan')
        second = torch.autograd.grad(grouped_linear(xg, wg, o, bias=bg), [xg, wg, bg], dy)
        assert torch.equal(first[0][:95], second[0][:95]) and torch.equal(first[0][96:], second[0][96:]) and torch.isnan(second[0][95]).all()
        assert all(torch.equal(first[i][:2], second[i][:2]) for i in (1, 2)) and torch.isnan(second[2][2, 2]) and torch.isfinite(second[2][2, 3:]).all()


def test_grouped_rows_behind_32_bits():
    from spi_amd.torch_utils.ops.grouped_linear import grouped_linear
    t, k, n = 540_000, 4096, 16                                       # 2.2e9 values
    g = gen(12)
    x, dy = torch.zeros(t, k, device=DEV, dtype=BF16), torch.zeros(t, n, device=DEV, dtype=BF16)
    x[-300:], dy[-300:] = randn(g, 300, k, dtype=BF16), randn(g, 300, n, dtype=BF16)
    w = randn(g, 2, n, k, dtype=BF16).requires_grad_()
    x.requires_grad_()
    o = torch.tensor([0, t - 200, t], device=DEV, dtype=torch.int32)
    y = grouped_linear(x, w, o, gain=0.1)
    dx, dw = torch.autograd.grad(y, [x, w], dy)
    offsets, xs, ds, ws = [0, 100, 300], x.detach()[-300:].double(), dy[-300:].double(), w.detach().double()
    r, mag = ref.grouped(xs, ws, None, offsets, 0.1)
    ref.check(y[-300:], r, mag, 2 * k + 8, 'y')
    exact, mags = ref.grouped_gradients(xs, ws, offsets, 0.1, ds)
    ref.check(dx[-300:], exact[0], mags[0], 2 * n + 8, 'dx')
    ref.check(dw, exact[1], mags[1], 2 * 300 + 8, 'dw')               # (zeros before, which round nothing)
    assert not y[:-300].any() and not dx[:-300].any()


def test_grouped_gradients_match_differences():
    from spi_amd.torch_utils.ops.grouped_linear import grouped_linear
    g = gen(13)
    x, w, b = randn(g, 40, 20), randn(g, 3, 28, 20), randn(g, 3, 28)
    offsets = [0, 9, 9, 38]
    o = torch.tensor(offsets, device=DEV, dtype=torch.int32)
    c = randn(g, 40, 28).double()
    leaves = [v.clone().requires_grad_() for v in (x, w, b)]
    got = torch.autograd.grad((grouped_linear(leaves[0], leaves[1], o, bias=leaves[2]).double() * c).sum(), leaves)
    mag = ref.grouped(x.double(), w.double(), b.double(), offsets, 1.0)[1]
    noise = (2 * 20 + 9) * ref.U32 * (mag * c.abs()).sum().item()
    for k in range(3):
        d = randn(g, *leaves[k].shape)
        at = lambda sign: [v + (sign * 0.5 * d if j == k else 0) for j, v in enumerate((x, w, b))]  # noqa: E731
        value = lambda v: (grouped_linear(v[0], v[1], o, bias=v[2]).double() * c).sum().item()  # noqa: E731
        quotient = value(at(1)) - value(at(-1))                        # linear in each argument: no truncation error
        assert abs(quotient - (got[k].double() * d.double()).sum().item()) <= 4 * noise, k


# ---- together ----------------------------------------------------------------------------------------------------------------------------
def test_frozen_block_in_8_bits():
    """norm with 8-bit rows -> wide layer -> 8-bit rows -> narrow layer -> norm behind the block: the serving form of a residual block"""
    from spi_amd.torch_utils.ops.linear_int8 import linear_int8, quantize_rows
    from spi_amd.torch_utils.ops.norm_residual import norm_residual
    g = gen(20)
    for rows, dtype in ((1, F32), (14, BF16), (200, F16)):
        i = norm_inputs((rows, 512), dtype, 'rms', 'both', 'channel', False, seed=rows)
        (w1, s1), (w2, s2) = int8_weights(g, 1024, 512), int8_weights(g, 512, 1024)
        stream, (q, qs) = norm_residual(i['h'], i['residual'], gate=i['gate'], scale=0.1, post_weight=i['post_weight'], pre_weight=i['pre_weight'], eps=1e-6, quantize=True)
        hidden = linear_int8(q, w1, s1, x_scale=qs, act='lrelu', gain=512 ** -0.5, out_dtype=dtype)
        out, _ = norm_residual(linear_int8(hidden, w2, s2), stream, scale=0.1, post_weight=i['post_weight'], where='after', eps=1e-6)
        # the same block step by step on the same integers, in 64 bits, each stage from the values that the stage before handed over
        r, mag = int8_reference(q, qs, w1, s1, None, 'lrelu', 512 ** -0.5, None)
        ref.check(hidden, r, mag, 8, 'hidden')
        r2, _ = int8_reference(*ref.quantize(hidden), w2, s2, None, 'linear', 1.0, None)
        y2 = linear_int8(hidden, w2, s2)
        ref.check(y2, r2, r2.abs(), 8, 'narrow')
        j = dict(h=y2, residual=stream, gate=None, post_weight=i['post_weight'], post_bias=None, pre_weight=None, pre_bias=None)
        ref.check(out, norm_case(j, 0.1, 'rms', 'after', 1e-6, 'linear', fn=ref.norm_residual)[0], norm_case(j, 0.1, 'rms', 'after', 1e-6, 'linear')['stream'], piled(512), 'out')
        # ... and the whole of it is the float block to what 8-bit rows and weights leave: each of the four roundings is at most half a step of 1/127 of a row's maximum
        assert quantize_rows(hidden)[0].shape == hidden.shape


def mapper(x, offsets, p, ops):
    """a residual block over rows whose level chooses the mapper: norm, grouped layer, activation, grouped layer, norm and gate"""
    norm, linear, act = ops
    _, y = norm(torch.zeros_like(x), x, None, None, p['n1'], 'before')
    y = linear(act(linear(y, p['w1'], offsets, p['b1'])), p['w2'], offsets, p['b2'])
    s, _ = norm(y, x, p['gate'], p['n2'], None, 'after')
    return s


def hip_ops():
    from spi_amd.torch_utils.ops import bias_act, grouped_linear, norm_residual
    return (lambda h, r, g, pw, qw, where: norm_residual.norm_residual(h, r, gate=g, scale=0.1, post_weight=pw, pre_weight=qw, where=where, eps=1e-6),
            lambda x, w, o, b: grouped_linear.grouped_linear(x, w, o, bias=b, gain=x.shape[1] ** -0.5), lambda x: bias_act.bias_act(x, act='lrelu'))


def wide_ops(offsets):
    return (lambda h, r, g, pw, qw, where: ref.norm_residual(h, r, g, 0.1, pw, None, qw, None, 'rms', where, 1e-6, 'linear'),
            lambda x, w, o, b: ref.grouped(x, w, b, offsets, x.shape[1] ** -0.5)[0], lambda x: torch.where(x > 0, x, 0.2 * x) * 2 ** 0.5)


def mapper_params(g, k, n):
    return dict(w1=randn(g, 3, n, k), b1=randn(g, 3, n), w2=randn(g, 3, k, n), b2=randn(g, 3, k), n1=1 + 0.1 * randn(g, k), n2=1 + 0.1 * randn(g, k), gate=randn(g, k))


def test_mapper_trains_like_its_definition():
    g = gen(21)
    x, p, offsets = randn(g, 14, 512), mapper_params(g, 512, 256), [0, 4, 8, 14]
    o = torch.tensor(offsets, device=DEV, dtype=torch.int32)
    leaves = {**{k: v.clone().requires_grad_() for k, v in p.items()}, 'x': x.clone().requires_grad_()}
    wide = {k: v.detach().double().requires_grad_() for k, v in leaves.items()}
    dy = randn(g, 14, 512)
    got = torch.autograd.grad(mapper(leaves['x'], o, leaves, hip_ops()), list(leaves.values()), dy)
    exact = torch.autograd.grad(mapper(wide['x'], o, wide, wide_ops(offsets)), list(wide.values()), dy.double())
    for k, a, b in zip(leaves, got, exact):
        # sums of 512, 256 and 512 products and two norms on the way, each within its own bound: their sum, times the spread of the largest value over the typical one
        assert (a.double() - b).norm() <= (2 * (512 + 256 + 512) + 4 * piled(512)) * ref.U32 * b.norm(), k


def test_mapper_in_a_captured_graph():
    """forward and backward captured once; replays with other rows, weights and group sizes agree with eager calls bit for bit"""
    g = gen(22)
    x, p = randn(g, 14, 64), mapper_params(g, 64, 128)
    o = torch.tensor([0, 4, 8, 14], device=DEV, dtype=torch.int32)
    dy = randn(g, 14, 64)

    def step():
        leaves = {**{k: v.detach().requires_grad_() for k, v in p.items()}, 'x': x.detach().requires_grad_()}
        out = mapper(leaves['x'], o, leaves, hip_ops())
        return [out.detach()] + list(torch.autograd.grad(out, list(leaves.values()), dy))
    step()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        held = step()
    for sizes in ([0, 4, 8, 14], [0, 0, 14, 14], [2, 3, 5, 11], [0, 14, 14, 14]):
        x.copy_(randn(g, 14, 64))
        dy.copy_(randn(g, 14, 64))
        p['w1'].copy_(randn(g, 3, 128, 64))
        o.copy_(torch.tensor(sizes, device=DEV, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, step()):
            assert torch.equal(a, b)


def test_int8_block_in_two_captured_graphs():
    from spi_amd.torch_utils.ops.linear_int8 import linear_int8
    g = gen(23)
    graphs = []
    for m in (3, 200):
        x, (wq, ws) = randn(g, m, 256), int8_weights(g, 160, 256)
        fn = lambda x=x, wq=wq, ws=ws: linear_int8(x, wq, ws, act='lrelu')  # noqa: E731
        fn()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = fn()
        graphs.append((graph, x, y, fn))
    for _ in range(3):
        for _, x, _, _ in graphs:
            x.copy_(torch.randn_like(x))
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        for (graph, *_), s in zip(graphs, streams):                     # both at once: neither uses the other's workspace
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for _, _, y, fn in graphs:
            assert torch.equal(y, fn())


def test_other_streams():
    from spi_amd.torch_utils.ops.linear_int8 import linear_int8
    g = gen(24)
    x, p, o = randn(g, 300, 64), mapper_params(g, 64, 96), torch.tensor([0, 100, 100, 300], device=DEV, dtype=torch.int32)
    wq, ws = int8_weights(g, 50, 64)
    want = mapper(x, o, p, hip_ops()), linear_int8(x, wq, ws)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = mapper(x, o, p, hip_ops()), linear_int8(x, wq, ws)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
