"""Decode attention over 4-bit pages to more than the output's own rounding, and
at the ends of its number formats: V scale bytes from 0 to 252, whole caches of
the largest and smallest values, weights that few tokens share, queries whose
32-value blocks differ widely in size.

Tolerance, by element: one rounding of the output to bf16, at most 2^-8 of the
value (2^-134 where the result is subnormal); the weights, held in two bf16
terms (the second rounds what the first left, 2^-8 of the weight at most, by
at most 2^-8 of itself), off by at most 2^-16 of A, the weighted mean magnitude
of the column; the exponent of a weight off by the score's own error E (absolute,
in units of the exponent), which moves weights and their sum by E each: 2 E A.
fp32 sums and exp2 add less than 2^-13 A.  Weights times a V scale are off by
2^-134 where they are subnormal, times 6 at most, n tokens of them over a sum of
weights of at least 1, or 2^-40 with V scales of 2^65 and more (whose weights are
kept that much lower): 6 n 2^-134, or 2^-94.  E is 2^-24 (128 + 8) sum |q k| scale
for the 128-term sums, plus what q's two e4m3 terms leave: nothing of a value
within 2^-10 of its block's largest, at most 2^-21 of the largest otherwise."""
import numpy as np
import pytest
import torch

import oracle.ops as O
from fp4_cases import as_codes, as_scales, on_device, random_pages, tables

pytestmark = pytest.mark.gpu

D = 128


def _reference(q, kc, ks, vc, vs, bt, ctx):
    """(outputs, tolerances) [B, Hq, D] in 64 bits."""
    hq, hkv, page = q.shape[1], kc.shape[2], kc.shape[1]
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    for b, n in enumerate(ctx):
        ids = bt[b, : -(-n // page)]
        k, v = (O.dequantize_fp4(c[ids], s[ids]).reshape(-1, hkv, D)[:n] for c, s in ((kc, ks), (vc, vs)))
        for h in range(hq):
            x, kh, vh = q[b, h], k[:, h // (hq // hkv)], v[:, h // (hq // hkv)]
            s = kh @ x * D ** -0.5
            top = np.abs(x).reshape(-1, 32).max(1).repeat(32)
            left = np.where(np.abs(x) >= 2.0 ** -10 * top, 0.0, 2.0 ** -21 * top)
            e = ((136 * 2.0 ** -24 * np.abs(kh * x).sum(1) + np.abs(kh) @ left) * D ** -0.5).max()
            w = np.exp(s - s.max())
            w /= w.sum()
            a = w @ np.abs(vh)
            out[b, h] = w @ vh
            small = 6 * n * 2.0 ** (-94 if (vs[ids][..., h // (hq // hkv), :] >= 192).any() else -134)
            tol[b, h] = 2.0 ** -8 * np.abs(out[b, h]) + (2.0 ** -16 + 2.0 ** -13 + 2 * e) * a + 2.0 ** -134 + small
    return out, tol


def _call(dev, q, kc, ks, vc, vs, bt, ctx, hkv):
    from xvllm.layers.attention import paged_decode_attention

    k, v, s1, s2 = (on_device(a, dev, "hnd") for a in (kc, vc, ks, vs))
    out = paged_decode_attention(q.to(dev).flatten(1), as_codes(k), as_codes(v), torch.from_numpy(bt).to(dev),
                                 torch.tensor(ctx, dtype=torch.int32, device=dev), q.shape[1], hkv, D,
                                 k_block_scale=as_scales(s1), v_block_scale=as_scales(s2))
    torch.cuda.synchronize()
    return out.double().cpu().numpy().reshape(q.shape)


def _check(got, want, tol):
    assert np.isfinite(got).all()
    excess = np.abs(got - want) - tol
    worst = float(excess.max())
    assert worst <= 0, f"excess {worst:.4g} at {np.unravel_index(excess.argmax(), excess.shape)}"


def _inputs(rng, ctx, hq, hkv, page=16, v=(120, 130), k=(120, 124)):
    bt, nb = tables(rng, ctx, page)
    kc, ks = random_pages(rng, nb, page, hkv, D, *k)
    vc, vs = random_pages(rng, nb, page, hkv, D, *v)
    q = torch.from_numpy(rng.standard_normal((len(ctx), hq, D)).astype(np.float32)).to(torch.bfloat16)
    return q, kc, ks, vc, vs, bt


GROUPS = [(8, 1), (8, 2), (4, 2), (3, 3)]


@pytest.mark.parametrize("hq,hkv", GROUPS)
def test_few_tokens_share_the_weight(dev, hq, hkv):
    """Contexts of 1 .. 9 tokens, where a weight's rounding is not averaged out."""
    rng = np.random.default_rng(hq)
    ctx = rng.integers(1, 10, 60).tolist()
    case = _inputs(rng, ctx, hq, hkv)
    q, *rest = case
    _check(_call(dev, *case, ctx, hkv), *_reference(q.double().numpy(), *rest, ctx))


@pytest.mark.parametrize("hq,hkv", GROUPS)
@pytest.mark.parametrize("low,high", [(0, 0), (0, 3), (1, 40), (0, 130), (100, 252), (192, 215), (245, 252), (0, 252)])
def test_v_scale_bytes_of_any_size(dev, hq, hkv, low, high):
    """Short, cut and ragged sequences whose V scales span a part of the format."""
    rng = np.random.default_rng(low * 256 + high + hq)
    ctx = [1, 5, 64, 65, 700, 130, 33, 2100]
    case = _inputs(rng, ctx, hq, hkv, v=(low, high))
    q, *rest = case
    _check(_call(dev, *case, ctx, hkv), *_reference(q.double().numpy(), *rest, ctx))


@pytest.mark.parametrize("hq,hkv", GROUPS)
def test_v_scales_that_change_along_the_sequence(dev, hq, hkv):
    """Units of 64 tokens of tiny, ordinary and huge V in turn, with scores that climb, fall or stay."""
    rng = np.random.default_rng(hq + 50)
    ctx, page = [900, 901, 902], 16
    q, kc, ks, vc, vs, bt = _inputs(rng, ctx, hq, hkv)
    for b in range(3):
        for j, p in enumerate(bt[b, : -(-ctx[b] // page)]):
            vs[p] = rng.integers(*[(0, 30), (118, 130), (230, 253)][(j // 4 + b) % 3], vs[p].shape)
            ks[p] = [110 + j // 4, 124 - j // 4, 122][b]
    case = q, kc, ks, vc, vs, bt
    _check(_call(dev, *case, ctx, hkv), *_reference(q.double().numpy(), *case[1:], ctx))


@pytest.mark.parametrize("hq,hkv", [(8, 1), (1, 1)])
@pytest.mark.parametrize("byte,code", [(252, 0x77), (252, 0xff), (0, 0x11), (1, 0x77)])
def test_the_largest_and_smallest_values_alone(dev, hq, hkv, byte, code):
    """One value everywhere in V: the weighted mean is that value, exactly, also where many waves' partials are joined."""
    rng = np.random.default_rng(3)
    ctx = [9000, 1, 64]
    q, kc, ks, vc, vs, bt = _inputs(rng, ctx, hq, hkv)
    vc[:], vs[:] = code, byte
    got = _call(dev, q, kc, ks, vc, vs, bt, ctx, hkv)
    want = O.dequantize_fp4(vc[0, 0, 0, :16], vs[0, 0, 0, :1])[0]
    # the sum of the weights times one value over the sum of the weights: exact to about 2^-14, far below half a bf16
    # step, and the value is a bf16
    assert got.min() == got.max() == want


@pytest.mark.parametrize("hq,hkv", GROUPS)
@pytest.mark.parametrize("kind", ["mixed", "loud", "subnormal", "large"])
def test_query_blocks_of_any_size(dev, hq, hkv, kind):
    """mixed: the 32-value blocks of q differ by up to 2^24, K's scales the other way; loud: within a block, values
    down to 2^-24 of its largest; subnormal and large: q at the ends of bf16."""
    rng = np.random.default_rng(hq + len(kind))
    ctx = [1, 40, 64, 300, 77]
    q, kc, ks, vc, vs, bt = _inputs(rng, ctx, hq, hkv)
    x = rng.standard_normal((len(ctx), hq, D))
    if kind == "mixed":
        e = rng.integers(-12, 13, 4)
        x *= np.exp2(e.astype(np.float64)).repeat(32)
        ks[:] = rng.integers(118, 124, ks.shape) - e
    elif kind == "loud":
        x *= np.exp2(rng.integers(-24, 1, x.shape).astype(np.float64)) * 16
    else:
        e = -128 if kind == "subnormal" else 124
        x = np.clip(x, -4, 4) * 2.0 ** e * 0.9
        ks[:] = np.clip(rng.integers(118, 124, ks.shape) - e, 0, 254)
    q = torch.from_numpy(x).to(torch.bfloat16)
    case = q, kc, ks, vc, vs, bt
    assert np.isfinite(q.double().numpy()).all()
    _check(_call(dev, *case, ctx, hkv), *_reference(q.double().numpy(), *case[1:], ctx))


def test_queries_that_are_not_finite(dev):
    """An infinity or NaN in a head's q makes that head NaN and leaves the others as they were."""
    rng = np.random.default_rng(8)
    ctx, hq, hkv = [70, 3], 8, 2
    q, *rest = _inputs(rng, ctx, hq, hkv)
    want = _call(dev, q, *rest, ctx, hkv)
    q[0, 1, 5], q[0, 6, 127], q[1, 3, 64] = float("inf"), float("nan"), -float("inf")
    got = _call(dev, q, *rest, ctx, hkv)
    nan = np.zeros((2, hq, D), bool)
    nan[0, 1] = nan[0, 6] = nan[1, 3] = True
    assert np.array_equal(np.isnan(got), nan) and np.array_equal(got[~nan], want[~nan])
