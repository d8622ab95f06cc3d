"""GPU tests of the row operators (norm_residual, quantize_rows / linear_int8, grouped_linear) at the edges of what their calls take: the largest launches, every tile of the
product kernels, empty and tiny operands, partial gradients.  The 64-bit statements and bounds are those of row_ops_ref."""
import ctypes

import pytest
import torch

import row_ops_ref as ref
from test_hip_row_ops_gpu import ORDER, check_grouped, int8_reference, norm_case, norm_inputs, piled, run_norm

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


# ---- gradients of a part of the results, for a part of the leaves ------------------------------------------------------------------------
def check_part(inputs, norm, where, act, use, wanted, scale=-0.7, eps=1e-6):
    """gradients of the results in ``use`` ('stream', 'normed') for the leaves in ``wanted``, against the 64-bit statement's.  A result without a use counts as one whose
    gradient is 0; a leaf that is only behind such a result gets none."""
    h = inputs['h']
    v = {k: t if t is None else t.clone().requires_grad_(k in wanted) for k, t in inputs.items()}
    results = dict(zip(('stream', 'normed'), run_norm(v, scale, norm, where, eps, act)))
    ct = {k: randn(gen(i), *h.shape, dtype=h.dtype) if k in use else torch.zeros_like(h) for i, k in enumerate(('stream', 'normed'))}
    leaves = [k for k in inputs if k in wanted and inputs[k] is not None]
    got = torch.autograd.grad([results[k] for k in use], [v[k] for k in leaves], [ct[k] for k in use], allow_unused=True)
    wide = {k: t if t is None else t.detach().double().requires_grad_() for k, t in inputs.items()}
    exact = dict(zip(('stream', 'normed'), ref.norm_residual(*[scale if k == 'scale' else wide[k] for k in ORDER], norm, where, eps, act)))
    exact = torch.autograd.grad([exact[k] for k in use], [wide[k] for k in leaves], [ct[k].double() for k in use], allow_unused=True)
    mag = norm_case(inputs, scale, norm, where, eps, act, ct['stream'], None if where == 'after' else ct['normed'])
    for k, a, e in zip(leaves, got, exact):
        what = f'{norm} {where} {use} d_{k} of {wanted}'
        if e is None:
            assert a is None, what
            continue
        m, add = mag[k], 0
        if a.shape != h.shape:                                        # a sum over rows
            m = m.sum((0, 1)) if a.ndim == 1 else m.sum(1, keepdim=a.ndim == 3)
            add = h.numel() // h.shape[-1]
        assert a.shape == inputs[k].shape and a.dtype == inputs[k].dtype, what
        ref.check(a, e, m, 4 * piled(h.shape[-1]) + add, what)


@pytest.mark.parametrize('gate,act', [(None, 'linear'), ('channel', 'tanh'), ('sample', 'sigmoid'), ('sample2', 'linear'), ('full', 'tanh')])
@pytest.mark.parametrize('where', ['both', 'before', 'after'])
def test_norm_gradients_of_one_result(where, gate, act):
    """the last block of a stack hands on its stream alone, a head reads the normed rows alone"""
    for norm, dtype, wdtype in (('rms', F32, F32), ('layer', F16, F16), ('layer', BF16, F32)):
        i = norm_inputs((3, 5, 200), dtype, norm, where, gate, True, wdtype=wdtype)
        for use in (('stream',), ('normed',), ('stream', 'normed')):
            if where != 'after' or 'normed' not in use:
                check_part(i, norm, where, act, use, tuple(i))


@pytest.mark.parametrize('shape', [(2, 3, 7), (1, 1, 512), (2, 700, 64), (2, 2, 2048), (1, 3, 4101), (2, 2, 8192)])
def test_norm_gradients_of_the_stream_in_every_width(shape):
    for dtype in (F32, BF16):
        check_part(norm_inputs(shape, dtype, 'rms', 'before', 'sample', False), 'rms', 'before', 'linear', ('stream',), ('h', 'residual', 'gate'))


@pytest.mark.parametrize('where', ['both', 'before', 'after'])
def test_norm_gradients_of_one_leaf(where):
    for norm, gate, act, dtype in (('rms', 'channel', 'tanh', F32), ('layer', 'sample', 'sigmoid', BF16), ('layer', 'full', 'linear', F16)):
        i = norm_inputs((4, 9, 136), dtype, norm, where, gate, True)
        for leaf in (k for k, t in i.items() if t is not None):
            check_part(i, norm, where, act, ('stream',) if where == 'after' else ('stream', 'normed'), (leaf,))


@pytest.mark.parametrize('h,gate', [((0, 5, 64), (0, 1, 64)), ((0, 5, 64), (0, 64)), ((0, 5, 64), (0, 5, 64)), ((0, 5, 64), (64,)), ((2, 0, 64), (2, 1, 64)), ((0, 64), (0, 64))])
def test_norm_of_an_empty_batch_with_every_gate(h, gate):
    from spi_amd.torch_utils.ops.norm_residual import norm_residual
    leaves = [torch.ones(s, device=DEV, requires_grad=True) for s in (h, h, gate, 64, 64)]
    for kw in (dict(), dict(norm='layer', gate_act='tanh')):
        s, y = norm_residual(leaves[0], leaves[1], gate=leaves[2], post_weight=leaves[3], pre_weight=leaves[4], **kw)
        assert s.shape == y.shape == h
        for v, g in zip(leaves, torch.autograd.grad(s.sum() + y.sum(), leaves)):
            assert g.shape == v.shape and not g.any()
        with torch.no_grad():
            s, (q, scale) = norm_residual(leaves[0], leaves[1], gate=leaves[2], post_weight=leaves[3], pre_weight=leaves[4], quantize=True, **kw)
        assert q.shape == h and scale.shape == h[:-1]


def test_forward_mode_tangents_are_refused():
    """no operator has a forward-mode derivative: a call on a tensor with a tangent raises, as bias_act's does, with and without gradients recorded, and loses nothing silently"""
    from torch.autograd import forward_ad
    from spi_amd.torch_utils.ops import bias_act, grouped_linear, linear_int8, norm_residual
    g = gen(30)
    x, w, vec = randn(g, 6, 16), randn(g, 2, 8, 16), randn(g, 16)
    o = torch.tensor([0, 2, 6], device=DEV, dtype=torch.int32)
    wq, ws = linear_int8.quantize_rows(randn(g, 8, 16))
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        calls = [lambda: bias_act.bias_act(dual(x), act='lrelu'), lambda: norm_residual.norm_residual(dual(x), x, post_weight=vec, pre_weight=vec),
                 lambda: norm_residual.norm_residual(x, x, gate=dual(vec), post_weight=vec, pre_weight=vec, quantize=True),
                 lambda: norm_residual.norm_residual(x, x, pre_weight=dual(vec), where='before'), lambda: grouped_linear.grouped_linear(dual(x), w, o),
                 lambda: grouped_linear.grouped_linear(x, dual(w), o), lambda: linear_int8.linear_int8(dual(x), wq, ws), lambda: linear_int8.quantize_rows(dual(x))]
        for call in calls + [torch.no_grad()(c) for c in calls]:
            with pytest.raises(RuntimeError):                          # (NotImplementedError, where an autograd function has no such rule, is one)
                call()
        want = norm_residual.norm_residual(x, x, post_weight=vec, pre_weight=vec)       # ... and tensors without one are served as ever
    for a, b in zip(want, norm_residual.norm_residual(x, x, post_weight=vec, pre_weight=vec)):
        assert torch.equal(a, b)


# ---- every tile of the product kernels -----------------------------------------------------------------------------------------------------
# Small whole numbers: every product and every partial sum is exact in 32 bits, so a result is the exact one rounded once, whatever the order of the sum -- the tolerance is 0, and a
# value that is lost, taken twice or from a wrong place shows.
COPY, WIDE, EACH = range(3)


def whole(g, *shape, dtype=F32, most=2):
    return torch.randint(-most, most + 1, shape, device=DEV, generator=g).to(dtype)


def grouped_tiles(x, w, dy, offsets):
    from spi_amd import hip
    t, k = x.shape
    e, n = w.shape[:2]
    tiles = []
    for which, ptrs in enumerate(((x, w, None), (None, w, dy), (x, None, dy))):
        px, pw, pd = (None if v is None else v.data_ptr() for v in ptrs)
        d = hip.GroupedLinearDesc(t, e, n, k, hip.ROW_DTYPES[x.dtype], 1.0, px, pw, None, offsets.data_ptr())
        d.dy = pd
        code = hip.lib().spi_grouped_linear_tile(ctypes.byref(d), which)
        tiles.append((code & 0xffff, code >> 16))
    return tiles


def check_grouped_whole(sizes, k, n, dtype, tiles, head=0, behind=0, odd=False):
    from spi_amd.torch_utils.ops.grouped_linear import grouped_linear
    g, offsets = gen(k + n), [head]
    for s in sizes:
        offsets.append(offsets[-1] + s)
    t, e = offsets[-1] + behind, len(sizes)
    place = lambda v: torch.cat([v.flatten()[:1], v.flatten()])[1:].view_as(v) if odd else v  # noqa: E731  (begins one value behind an aligned place)
    x, w, dy = place(whole(g, t, k, dtype=dtype)), place(whole(g, e, n, k, dtype=dtype)), place(whole(g, t, n, dtype=dtype))
    b, o = whole(g, e, n, dtype=dtype), torch.tensor(offsets, device=DEV, dtype=torch.int32)
    assert grouped_tiles(x, w, dy, o) == tiles
    leaves = [v.requires_grad_() for v in (x, w, b)]
    y = grouped_linear(*leaves[:2], o, bias=b, gain=0.5)
    dx, dw, db = torch.autograd.grad(y, leaves, dy)
    covered = torch.zeros(t, 1, device=DEV, dtype=torch.bool)
    covered[head:offsets[-1]] = True
    for v in (y, dx):
        assert not v[:head].any() and not v[offsets[-1]:].any()
    for i in range(e):
        s = slice(offsets[i], offsets[i + 1])
        xs, ws, ds = x[s].detach().double(), w[i].detach().double(), dy[s].double()
        for name, got, exact in (('y', y[s], 0.5 * (xs @ ws.t()) + b[i].detach().double()), ('dx', dx[s], 0.5 * (ds @ ws)), ('dw', dw[i], 0.5 * (ds.t() @ xs)), ('db', db[i], ds.sum(0))):
            same = got == exact.to(dtype)
            assert same.all(), f'{name} of group {i}: {(~same).sum().item()} values, the first at {(~same).nonzero()[0].tolist()}'


@pytest.mark.parametrize('dtype', [F32, F16, BF16])
@pytest.mark.parametrize('sizes,k,n,tiles,kw', [
    ([70, 0, 131], 136, 264, [(64, COPY)] * 3, {}),
    ([70, 0, 131], 137, 263, [(64, WIDE)] * 3, {}),
    ([2, 0, 1], 1, 1, [(64, EACH)] * 3, {}),
    ([1311, 789], 2056, 2040, [(128, COPY)] * 3, {}),
    ([1, 1408, 640], 2048, 2176, [(128, COPY)] * 3, dict(head=5, behind=140)),
    ([1500, 1501], 2045, 2047, [(128, WIDE)] * 3, {}),
    ([2999, 1], 2048, 2056, [(128, WIDE)] * 3, dict(head=1, odd=True)),                            # rows of whole 16 bytes on odd places
    ([2001, 0, 2999], 3320, 3320, [(256, COPY)] * 3, {}),                                          # 260 tiles a pass: the last four cut into quarters
    ([3000, 4000], 3320, 3320, [(256, COPY)] * 3, {}),                                             # 364 tiles, 108 of them cut; the weight gradient 338, 82 cut
    ([4000, 0, 4000], 3312, 3320, [(256, COPY)] * 3, dict(head=300, behind=1)),                    # 34 x 13 = 442 tiles, none cut
    ([256] * 16 + [512], 4096, 4096, [(256, COPY)] * 3, {}),                                       # tiles without an edge
], ids=lambda v: None if not isinstance(v, list) else '-'.join(map(str, v)) if not isinstance(v[0], tuple) else f'{v[0][0]}')
def test_grouped_tiles(sizes, k, n, tiles, kw, dtype):
    check_grouped_whole(sizes, k, n, dtype, tiles, **kw)


@pytest.mark.parametrize('m,n,k,padded,tiles', [
    # (edge, loader) of int8 rows that begin on 16 bytes if `padded`, and of rows of floats, which the call lays out on 16 bytes
    (100, 333, 1040, True, [(64, COPY), (64, COPY)]), (100, 333, 1031, True, [(64, WIDE), (64, COPY)]), (100, 333, 1031, False, [(64, WIDE), (64, WIDE)]),
    (17, 1, 3, False, [(64, EACH), (64, EACH)]), (2100, 2090, 1040, True, [(128, COPY), (128, COPY)]), (2100, 2090, 1031, True, [(64, WIDE), (128, COPY)]),
    (2600, 2500, 1031, True, [(128, WIDE), (128, COPY)]), (2600, 2500, 1031, False, [(128, WIDE), (128, WIDE)]), (4100, 4000, 1040, True, [(256, COPY), (256, COPY)]),
    (4100, 4003, 1031, True, [(128, WIDE), (256, COPY)]), (4096, 4352, 2048, True, [(256, COPY), (256, COPY)])])
def test_linear_int8_tiles(m, n, k, padded, tiles):
    from spi_amd import hip
    from spi_amd.torch_utils.ops.linear_int8 import linear_int8
    g, pitch = gen(m + n + k), (k + 15) // 16 * 16 if padded else k

    def rows(count):                                                  # what stands behind a row is not 0
        full = torch.full((count, pitch), 99, device=DEV, dtype=torch.int8)
        full[:, :k] = whole(g, count, k, dtype=torch.int8, most=127)
        full[:, 0] = 127                                              # so that rows of floats have the scale 1, and quantise to themselves
        return full[:, :k]
    q, w, one = rows(m), rows(n), torch.ones(max(m, n), device=DEV)
    exact = (q.double() @ w.double().t()).float()                     # integers: exact in 64 bits, rounded once
    for x, scale, tile in zip((q, q.float()), (one[:m], None), tiles):
        d = hip.LinearInt8Desc(m, n, k, hip.DTYPE_I8 if scale is not None else 0, 0, x.stride(0), w.stride(0), w.untyped_storage().nbytes(), x.data_ptr(), one.data_ptr(), w.data_ptr(),
                               one.data_ptr(), None, one.data_ptr(), 1, 0.0, 1.0, -1.0)
        code = hip.lib().spi_linear_int8_tile(ctypes.byref(d))
        assert (code & 0xffff, code >> 16) == tile
        for dtype in (F32, BF16):
            same = linear_int8(x, w, one[:n], x_scale=scale, out_dtype=dtype) == exact.to(dtype)
            assert same.all(), f'{(~same).sum().item()} values, the first at {(~same).nonzero()[0].tolist()}'


# ---- a block in 8 bits against the block in floats -----------------------------------------------------------------------------------------
def test_block_in_8_bits_is_the_float_block_within_its_roundings():
    """norm -> 8-bit layer -> 8-bit layer -> norm and residual, against the same block in 64 bits with the weights as they were.

    The four roundings to 8 bits (of both layers' rows and weights) are at most half a step each and independent: uniform, of variance step^2 / 12.  A product's error is a sum of 512
    or 1024 of them with known factors, so its deviation follows; an activation of slope <= 1 does not widen it, and eight deviations are asked for (one value in 1e15 lies outside).
    The rounding of the hidden rows to their type adds half a step, u |hidden|.  Through the norm, x -> x / sigma(x): |d| / sigma + |x| |1/sigma' - 1/sigma|, and sigma, a root mean square,
    moves by at most the root mean square of d (allowed here: twice its deviation)."""
    from spi_amd.torch_utils.ops.linear_int8 import linear_int8, quantize_rows
    from spi_amd.torch_utils.ops.norm_residual import norm_residual
    g = gen(40)
    for rows, dtype in ((1, F32), (14, BF16), (200, F16)):
        i = norm_inputs((rows, 512), dtype, 'rms', 'both', 'channel', False, seed=rows)
        w1, w2 = randn(g, 1024, 512), randn(g, 512, 1024)
        (q1, s1), (q2, s2) = quantize_rows(w1), quantize_rows(w2)
        stream, (q, qs) = norm_residual(i['h'], i['residual'], gate=i['gate'], scale=0.1, post_weight=i['post_weight'], pre_weight=i['pre_weight'], eps=1e-6, quantize=True)
        hidden = linear_int8(q, q1, s1, x_scale=qs, act='lrelu', gain=512 ** -0.5, out_dtype=dtype)
        y2 = linear_int8(hidden, q2, s2)
        out, _ = norm_residual(y2, stream, scale=0.1, post_weight=i['post_weight'], where='after', eps=1e-6)
        # the float block
        s64, y64 = norm_case(i, 0.1, 'rms', 'both', 1e-6, 'linear', fn=ref.norm_residual)
        w1, w2, u = w1.double(), w2.double(), ref.half_step(dtype)
        h64 = ref.activation('lrelu', y64 @ w1.t()) * 512 ** -0.5
        x64 = h64 @ w2.t()
        sigma = torch.sqrt((x64 ** 2).mean(-1, keepdim=True) + 1e-6)
        o64 = s64 + 0.1 * x64 / sigma * i['post_weight'].double()

        def variance(step, q, s, x, before):                          # of a product's error: (step^2 / 12 + before) through the weights, and the weights' own roundings
            w = q.double() * s.double()[:, None]
            return (step ** 2 / 12 + before) @ (w ** 2).t() + s.double() ** 2 / 12 * (x ** 2).sum(-1, keepdim=True)
        one = torch.ones_like(y64)
        v1 = variance(qs.double()[:, None] * one, q1, s1, y64, 0 * one) / 512
        t2 = hidden.double().abs().amax(-1, keepdim=True) / 127
        v2 = variance(t2 * torch.ones_like(h64), q2, s2, h64, v1 + (u * h64) ** 2) + (u * x64) ** 2
        d, moved = 8 * v2.sqrt(), 2 * v2.mean(-1, keepdim=True).sqrt()
        through = (d + (x64.abs() + d) * moved / (sigma - moved)) / sigma * i['post_weight'].double().abs()
        bound = 0.1 * through + 2 * u * (s64.abs() + o64.abs()) + piled(512) * ref.U32 * o64.abs()
        worst = ((out.double() - o64).abs() / bound).max().item()
        assert worst <= 1, (rows, dtype, worst)
        # The bound means something, about a fifth of the 0.1 that the block adds to a value: with the largest of a row at four deviations, a rounding is 4 / 127 / 12^0.5 = 0.0091 of the
        # rows (0.0126 of the hidden ones, whose root mean square the activation takes to 0.72), 0.0091 of either weight; with bf16's two of 2^-8, 0.021 together.  Eight of it, and
        # twice of it times 0.8 + 8 * 0.021 for the deviation that divides, over 1 - 2 * 0.021: 0.218.
        assert (0.1 * through).mean() < 0.022
