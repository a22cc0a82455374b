"""mxfp4_linear through every kernel it has (mxfp4_shapes.SHAPES), against the
64-bit product of the dequantised weight on the device; scale bytes at the ends
of the format, split products in graphs and on several streams.

Tolerance.  The operands are exact in bf16, products and sums of K terms fp32:
off by at most (K + 8) 2^-24 sum |x w|; one rounding to bf16, at most 2^-8 of
the value.  With silu(g) * u the errors dg, du of the two products enter by the
derivative, |silu'| <= 1.1 and |silu(g)| <= |g|, and expf, the division and the
products add 8 * 2^-24 of the value."""
import numpy as np
import pytest
import torch

import oracle.ops as O
from fp4_cases import as_codes, as_scales
from mxfp4_shapes import SHAPES

pytestmark = pytest.mark.gpu


def _weight(dev, n, k, seed, low=117, high=122):
    g = torch.Generator(device=dev).manual_seed(seed)
    return (torch.randint(0, 256, (n, k // 2), generator=g, device=dev, dtype=torch.uint8),
            torch.randint(low, high + 1, (n, k // 32), generator=g, device=dev, dtype=torch.uint8))


def _values(w, s):
    """The weight in 64 bits (scale 255: NaN), from the definition."""
    table = torch.from_numpy(np.concatenate([O.FP4_MAGNITUDES, -O.FP4_MAGNITUDES])).to(w.device)
    pair = torch.stack((w & 15, w >> 4), dim=-1).flatten(1)
    unit = torch.where(s == 255, torch.nan, torch.exp2(s.double() - 127))
    return (table[pair.int()].unflatten(1, (-1, 32)) * unit[..., None]).flatten(1)


def _bounds(x, w, s, silu):
    """(the product in 64 bits, how far its bf16 may be off)."""
    x, k = x.double(), x.shape[1]
    half = w.shape[0] // 2 if silu else w.shape[0]
    ys, mags = [], []
    for i in range(0, w.shape[0], 4096):
        v = _values(w[i : i + 4096], s[i : i + 4096])
        ys.append(x @ v.t().contiguous())
        mags.append(x.abs() @ v.abs().t().contiguous() * (k + 8) * 2.0 ** -24)
    y, mag = torch.cat(ys, 1), torch.cat(mags, 1)
    if silu:
        g, u, dg, du = y[:, :half], y[:, half:], mag[:, :half], mag[:, half:]
        y = g * torch.sigmoid(g) * u
        mag = 1.1 * dg * (u.abs() + du) + g.abs() * du + 8 * 2.0 ** -24 * y.abs()
    return y, 2.0 ** -8 * y.abs() + 1.01 * mag + 1e-37


def _check(got, x, w, s, silu):
    y, tol = _bounds(x, w, s, silu)
    assert got.shape == y.shape and torch.isfinite(got).all()
    worst = float(((got.double() - y).abs() - tol).max())
    assert worst <= 0, f"excess {worst:.4g}"


def _product(x, w, s, silu=False):
    from xvllm.layers.linear import mxfp4_linear

    return mxfp4_linear(x, as_codes(w), as_scales(s), silu_mul=silu)


def _rows(dev, m, k, seed):
    return torch.randn(m, k, generator=torch.Generator(device=dev).manual_seed(seed), device=dev).to(torch.bfloat16)


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_every_kernel(dev, m, n, k):
    w, s = _weight(dev, n, k, m + n + k)
    x = _rows(dev, m, k, m * n)
    for silu in (False, True):
        got = _product(x, w, s, silu)
        torch.cuda.synchronize()
        _check(got, x, w, s, silu)


# one of each size of kernel, K whole and in parts
FORMS = [(3, 40, 128), (12, 40, 4128), (40, 512, 4128), (33, 16, 8192), (64, 514, 8224), (200, 96, 512), (100, 320, 2080), (193, 3000, 6144)]


@pytest.mark.parametrize("m,n,k", FORMS)
def test_scales_at_the_ends_of_the_format(dev, m, n, k):
    """Bytes 0, 1 and 254 in the first, a middle and the last block of a row; 255 makes its row NaN, alone."""
    w, s = _weight(dev, n, k, 9)
    x = _rows(dev, m, k, 10)
    x[:, :32] *= 2.0 ** -60
    last = k // 32 - 1
    s[3], s[4, last // 2], s[5, 0], s[6, last], s[n - 1, 1] = 1, 0, 254, 0, 0
    w[5, :16] = 0x11  # 0.5 * 2^127
    _check(_product(x, w, s), x, w, s, False)
    for at in {0, last // 2, last}:
        row = 7 + at % 5
        t = s.clone()
        t[row, at] = 255
        got = _product(x, w, t)
        nan = torch.zeros_like(got, dtype=torch.bool)
        nan[:, row] = True
        assert torch.equal(got.isnan(), nan)
        _check(torch.where(nan, 0, got), x, torch.where(torch.arange(n, device=dev)[:, None] == row, 0, w), s, False)


@pytest.mark.parametrize("m,n,k", [(40, 512, 8224), (33, 16, 8192), (64, 514, 8224), (200, 96, 2080), (100, 320, 2080), (193, 3000, 6144)])
@pytest.mark.parametrize("silu", [False, True])
def test_split_products_on_two_streams(dev, m, n, k, silu):
    """Two graphs, replayed at once on two streams beside eager calls on a third, over new inputs: each has parts of
    its own and gives the eager result."""
    from xvllm import _C

    assert _C.lib().xv_mxfp4_gemm_workspace_size(m, n, k, silu) > 0
    weights = [_weight(dev, n, k, 20 + i) for i in (0, 1)]
    xs = [torch.zeros(m, k, dtype=torch.bfloat16, device=dev) for _ in (0, 1)]
    _product(xs[0], *weights[0], silu)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for x, ws in zip(xs, weights):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(_product(x, *ws, silu))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(3)]
    for turn in range(4):
        new = [_rows(dev, m, k, 30 + 2 * turn + i) for i in (0, 1)]
        want = [_product(x, *ws, silu) for x, ws in zip(new, weights)]
        for x, y in zip(xs, new):
            x.copy_(y)
        torch.cuda.synchronize()
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        with torch.cuda.stream(streams[2]):
            eager = _product(new[0], *weights[0], silu)
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1]) and torch.equal(eager, want[0])
        _check(want[1], new[1], *weights[1], silu)
