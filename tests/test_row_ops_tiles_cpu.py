"""The choice of a product's matrix tile and loader (spi_linear_int8_tile, spi_grouped_linear_tile): a host decision, made here without a GPU.

What a loader asks of its operands: _COPY wants rows that begin and end on 16 bytes, _WIDE reads 16 bytes wherever a chunk would pass the tensor's end -- so the tensor has to have
them, whatever the tile's edge -- and _EACH asks nothing."""
import ctypes
import itertools

import pytest

from spi_amd import hip

COPY, WIDE, EACH = range(3)
F32, F16, BF16, I8 = 0, 1, 3, 4
FWD, DGRAD, WGRAD = range(3)
P = 0x100000                                                           # never read


def grouped_tile(t, e, n, k, dtype, which, odd=0):
    at = lambda on, size: (P + odd if size else None) if on else None   # noqa: E731  (an empty tensor has no address)
    d = hip.GroupedLinearDesc(t, e, n, k, dtype, 1.0, at(which != DGRAD, t * k), at(which != WGRAD, e * n * k), None, P)
    d.dy = at(which != FWD, t * n)
    code = hip.lib().spi_grouped_linear_tile(ctypes.byref(d), which)
    return None if code < 0 else (code & 0xffff, code >> 16)


def int8_tile(m, n, k, x_dtype, x_stride=None, w_stride=None, tail=0, odd=0):
    xs, ws = x_stride or k, w_stride or k
    d = hip.LinearInt8Desc(m, n, k, x_dtype, F32, xs, ws, (n - 1) * ws + k + tail, P, P if x_dtype == I8 else None, P + odd, P, None, P, 1, 0.0, 1.0, -1.0)
    d.workspace, d.workspace_bytes = P, 1 << 60
    code = hip.lib().spi_linear_int8_tile(ctypes.byref(d))
    return None if code < 0 else (code & 0xffff, code >> 16)


@pytest.mark.parametrize('which', [FWD, DGRAD, WGRAD], ids=['forward', 'rows', 'weights'])
@pytest.mark.parametrize('dtype', [F32, F16, BF16])
def test_grouped_operands_have_what_their_loader_reads(dtype, which):
    size, seen = 4 if dtype == F32 else 2, set()
    for t, e, n, k, odd in itertools.product((0, 1, 2, 3, 7, 100, 4099, 50_000, 1 << 30), (1, 3, 8, 24, 400, 65535), (1, 2, 3, 5, 7, 8, 15, 16, 771, 1003, 2048, 1 << 20),
                                             (1, 2, 3, 5, 7, 8, 15, 16, 515, 1003, 2048, 1 << 20), (0, size)):
        tile = grouped_tile(t, e, n, k, dtype, which, odd)
        if tile is None:                                               # (more tiles than a launch has blocks)
            continue
        if t == 0 and which != WGRAD:
            assert tile == (0, 0)                                      # nothing is launched
            continue
        edge, load = tile
        rows = {FWD: (t * k, e * n * k), DGRAD: (t * n, e * n * k), WGRAD: (t * n, t * k)}[which]
        assert edge in (64, 128, 256) and load in (COPY, WIDE, EACH)
        if load == WIDE:
            assert min(rows) * size >= 16, (t, e, n, k)
        if load == COPY:
            assert n * size % 16 == 0 and k * size % 16 == 0 and (odd == 0 or not min(rows)), (t, e, n, k)
        else:
            assert edge != 256
        if load == EACH:
            assert edge == 64 and min(rows) * size < 16                # and it is not taken where it need not be
        seen.add((edge, load))
    assert seen == {(64, COPY), (128, COPY), (256, COPY), (64, WIDE), (128, WIDE), (64, EACH)}


@pytest.mark.parametrize('x_dtype', [I8, F32, F16, BF16])
def test_int8_operands_have_what_their_loader_reads(x_dtype):
    seen = set()
    for m, n, k, pad, tail, odd in itertools.product((1, 16, 17, 100, 4099, 50_000, 1 << 30), (1, 2, 3, 5, 15, 16, 17, 771, 4096, 1 << 20), (1, 2, 3, 5, 15, 16, 17, 1003, 2048, 131071),
                                                     (0, 1, 16), (0, 15), (0, 1)):
        stride = k if pad == 0 else k + 1 if pad == 1 else (k + 15) // 16 * 16
        tile = int8_tile(m, n, k, x_dtype, stride, stride, tail, odd)
        if tile is None:
            continue
        if tile == (0, 0):
            assert m <= 16                                             # the kernel for few rows
            continue
        edge, load = tile
        q_stride = stride if x_dtype == I8 else (k + 15) // 16 * 16    # rows of floats are quantised into rows of whole 16 bytes
        smallest = min((m - 1) * q_stride, (n - 1) * stride) + k
        assert edge in (64, 128, 256)
        if load == WIDE:
            assert smallest >= 16 and edge != 256, (m, n, k)
        elif load == EACH:
            assert smallest < 16 and edge == 64, (m, n, k)
        else:
            assert odd == 0 and q_stride % 16 == 0 and stride % 16 == 0 and (k % 16 == 0 or (x_dtype != I8 and (n - 1) * stride + k + tail >= (n - 1) * stride + (k + 15) // 16 * 16))
        seen.add((edge, load))
    assert seen == {(64, COPY), (128, COPY), (256, COPY), (64, WIDE), (128, WIDE), (64, EACH)}


def test_the_calls_that_used_to_read_in_front_of_a_tensor():
    """no rows, hardly any rows, and one short row of weights, at sizes that fill the chip with tiles of 128"""
    assert grouped_tile(0, 8, 1003, 1003, F32, WGRAD) == (64, EACH) == grouped_tile(0, 8, 771, 1003, F32, WGRAD)
    assert grouped_tile(1, 100, 1003, 5, F16, WGRAD) == (64, EACH)
    assert grouped_tile(1, 400, 3, 5, F16, WGRAD) == (64, EACH) == grouped_tile(1, 400, 3, 5, F16, FWD)
    assert grouped_tile(5, 5, 1 << 20, 1, F16, FWD) == (64, EACH)
    assert int8_tile(50_000, 1, 15, I8) == (64, EACH) == int8_tile(50_000, 1, 15, F32)


def test_tiles_of_wrong_calls_are_errors():
    assert int8_tile(4, 0, 4, I8) is None and grouped_tile(4, 0, 8, 8, F32, FWD) is None and grouped_tile(4, 2, 8, 8, F32, 3) is None and grouped_tile(4, 2, 8, 8, F32, -1) is None
    assert hip.lib().spi_linear_int8_tile(None) == -1 == hip.lib().spi_grouped_linear_tile(None, 0)
