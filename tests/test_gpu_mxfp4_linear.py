"""mxfp4_linear against the 64-bit product of the oracle's dequantised weight.

Tolerance.  The operands are exact in bf16 (code * 2^e), products exact in
fp32 up to its rounding, K terms summed in fp32: an error of at most
(K + 8) 2^-24 sum |x w|, far above what a sum of random signs shows; then one
rounding to bf16, at most 2^-8 of the value (8 significant bits: half a step is
2^(e-8) for a value of at least 2^e).  With silu(g) * u the errors dg, du of the
two products enter through the derivative, |silu'| <= 1.1 and |silu(g)| <=
|g|, and expf, the division and the products add 8 * 2^-24 of the value."""
import numpy as np
import pytest
import torch

import oracle.ops as O
from fp4_cases import as_codes, as_scales

pytestmark = pytest.mark.gpu


def _weight(rng, n, k, low=117, high=122):
    return (rng.integers(0, 256, (n, k // 2), dtype=np.uint8), rng.integers(low, high + 1, (n, k // 32)).astype(np.uint8))


def _run(dev, x, w, s, **kw):
    from xvllm.layers.linear import mxfp4_linear

    return mxfp4_linear(x, as_codes(torch.from_numpy(w).to(dev)), as_scales(torch.from_numpy(s).to(dev)), **kw)


def _check(got, x, w, s, silu):
    x = x.double().cpu().numpy()
    k = x.shape[-1]
    full = O.dequantize_fp4(w, s)
    y, mag = x @ full.T, np.abs(x) @ np.abs(full).T * (k + 8) * 2.0 ** -24
    if silu:
        i = w.shape[0] // 2
        g, u, dg, du = y[:, :i], y[:, i:], mag[:, :i], mag[:, i:]
        y = g / (1 + np.exp(-g)) * u
        mag = 1.1 * dg * (np.abs(u) + du) + np.abs(g) * du + 8 * 2.0 ** -24 * np.abs(y)
    got = got.double().cpu().numpy()
    assert got.shape == y.shape and np.isfinite(got).all()
    excess = np.abs(got - y) - (2.0 ** -8 * np.abs(y) + 1.01 * mag + 1e-37)
    assert (excess <= 0).all(), f"max excess {excess.max():.4g} at {np.unravel_index(excess.argmax(), excess.shape)}"


@pytest.mark.parametrize("silu", [False, True])
@pytest.mark.parametrize("m,n,k", [
    (1, 16, 32), (1, 4096, 4096), (3, 34, 64), (16, 130, 96), (17, 1000, 416), (33, 258, 2080), (64, 512, 1024),
    (65, 20, 160), (200, 96, 512), (256, 514, 288), (100, 320, 2080), (160, 1026, 1024), (190, 200, 4000), (225, 66, 3200), (8, 2, 12288), (300, 18, 32), (15, 6000, 224), (130, 1538, 1056),
    (64, 514, 8224), (40, 512, 4128), (33, 66, 12288), (20, 48, 9024), (17, 4096, 4096), (48, 1000, 5152),
])
def test_product_matches_oracle(dev, m, n, k, silu):
    rng = np.random.default_rng(m * 7 + n + k)
    w, s = _weight(rng, n, k)
    x = torch.from_numpy(rng.standard_normal((m, k)).astype(np.float32)).to(torch.bfloat16).to(dev)
    got = _run(dev, x, w, s, silu_mul=silu)
    torch.cuda.synchronize()
    _check(got, x, w, s, silu)


@pytest.mark.parametrize("m,n,k", [(5, 77, 4096), (1, 1, 32), (40, 333, 992)])
def test_odd_column_counts(dev, m, n, k):
    rng = np.random.default_rng(n)
    w, s = _weight(rng, n, k)
    x = torch.from_numpy(rng.standard_normal((m, k)).astype(np.float32)).to(torch.bfloat16).to(dev)
    got = _run(dev, x, w, s)
    torch.cuda.synchronize()
    _check(got, x, w, s, False)


def test_layouts_of_x_and_w(dev):
    """x as a strided, an unaligned, an expanded and a three-dimensional view;
    a weight and its scales as rows of wider ones; no rows."""
    from xvllm.layers.linear import mxfp4_linear

    rng = np.random.default_rng(4)
    n, k = 50, 256
    w, s = _weight(rng, n, k)
    wide, swide = torch.zeros(n, k // 2 + 32, dtype=torch.uint8, device=dev), torch.zeros(n, k // 32 + 3, dtype=torch.uint8, device=dev)
    wide[:, 16 : 16 + k // 2] = torch.from_numpy(w).to(dev)
    swide[:, 1 : 1 + k // 32] = torch.from_numpy(s).to(dev)
    wv, sv = as_codes(wide)[:, 16 : 16 + k // 2], as_scales(swide)[:, 1 : 1 + k // 32]
    base = torch.from_numpy(rng.standard_normal((6, 2, k + 9)).astype(np.float32)).to(torch.bfloat16).to(dev)
    for x in (base[:, 0, :k], base[:, 1, 3 : 3 + k], base[:1, 0, :k].expand(6, k), base[:, 0, :k].t().contiguous().t()):
        got = mxfp4_linear(x, wv, sv)
        _check(got, x, w, s, False)
    got = mxfp4_linear(base[:, :, :k], wv, sv)
    assert got.shape == (6, 2, n)
    _check(got.view(12, n), base[:, :, :k].reshape(12, k), w, s, False)
    assert mxfp4_linear(base[:0, 0, :k], wv, sv).shape == (0, n)


def test_special_scales(dev):
    """Scale bytes at both ends of the format; 255 makes its row NaN and leaves the others."""
    rng = np.random.default_rng(9)
    n, k, m = 40, 128, 3
    w, s = _weight(rng, n, k)
    s[3], s[4, 1], s[5, 2] = 1, 0, 254
    w[5, 32:48] = 0x11  # 0.5 * 2^127
    x = torch.from_numpy(rng.standard_normal((m, k)).astype(np.float32)).to(torch.bfloat16).to(dev)
    x[:, 64:96] = 2.0 ** -60
    _check(_run(dev, x, w, s), x, w, s, False)
    s[7, 3] = 255
    got = _run(dev, x, w, s).cpu()
    assert got[:, 7].isnan().all() and not got[:, :7].isnan().any() and not got[:, 8:].isnan().any()


def test_graph_and_stream(dev):
    from xvllm.layers.linear import mxfp4_linear

    rng = np.random.default_rng(2)
    n, k = 512, 2048
    w, s = _weight(rng, n, k)
    wd, sd = as_codes(torch.from_numpy(w).to(dev)), as_scales(torch.from_numpy(s).to(dev))
    x = torch.zeros(9, k, dtype=torch.bfloat16, device=dev)
    mxfp4_linear(x, wd, sd)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = mxfp4_linear(x, wd, sd)
        z = mxfp4_linear(x, wd, sd, silu_mul=True)
    for i in range(4):
        x.normal_(generator=torch.Generator(device=dev).manual_seed(i))
        graph.replay()
        torch.cuda.synchronize()
        got = y.clone(), z.clone()
        assert torch.equal(got[0], mxfp4_linear(x, wd, sd)) and torch.equal(got[1], mxfp4_linear(x, wd, sd, silu_mul=True))
        _check(got[0], x, w, s, False)
        _check(got[1], x, w, s, True)


def test_refusals(dev):
    from xvllm.layers.linear import mxfp4_linear

    w = as_codes(torch.zeros(8, 64, dtype=torch.uint8, device=dev))
    s = as_scales(torch.zeros(8, 4, dtype=torch.uint8, device=dev))
    x = torch.zeros(2, 128, dtype=torch.bfloat16, device=dev)
    with pytest.raises(TypeError):
        mxfp4_linear(x, w.view(torch.uint8), s)
    with pytest.raises(TypeError):
        mxfp4_linear(x.float(), w, s)
    for bad in ((x[:, :64], w, s), (x, w, s[:, :3]), (x, w[:7], s), (x[:, :48], w[:, :24], s[:, :1])):
        with pytest.raises(ValueError):
            mxfp4_linear(*bad)
    with pytest.raises(ValueError):
        mxfp4_linear(x, w[:7], s[:7], silu_mul=True)
    with pytest.raises(ValueError):
        mxfp4_linear(x, w.view(torch.uint8).t().contiguous().t().view(w.dtype), s)
    with pytest.raises(RuntimeError):
        mxfp4_linear(x.requires_grad_(), w, s)


@pytest.mark.parametrize("silu", [False, True])
def test_product_in_a_compiled_function(dev, silu):
    """A compiler's trace holds the product as one op, with the eager result."""
    from xvllm.layers.linear import mxfp4_linear

    rng = np.random.default_rng(31)
    w, s = _weight(rng, 64, 96)
    w, s = as_codes(torch.from_numpy(w).to(dev)), as_scales(torch.from_numpy(s).to(dev))
    x = torch.from_numpy(rng.standard_normal((2, 5, 96)).astype(np.float32)).to(torch.bfloat16).to(dev)
    f = torch.compile(lambda t: mxfp4_linear(t * 2, w, s, silu_mul=silu) + 1, backend="eager", fullgraph=True)
    with torch.no_grad():
        got, want = f(x), mxfp4_linear(x * 2, w, s, silu_mul=silu) + 1
    torch.cuda.synchronize()
    assert torch.equal(got, want)


def test_product_op_registration(dev):
    import xvllm.layers.linear  # noqa: F401  (registers the op)

    rng = np.random.default_rng(32)
    w, s = (torch.from_numpy(a).to(dev) for a in _weight(rng, 32, 64))
    x = torch.zeros((3, 64), dtype=torch.bfloat16, device=dev)
    torch.library.opcheck(torch.ops.xv.mxfp4_linear, (x, w, s, False), test_utils=("test_schema", "test_faketensor"))
