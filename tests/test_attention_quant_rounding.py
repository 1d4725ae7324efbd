"""The rounding that attention over a cache in codes promises for 16-bit queries: softmax weights, and for more than 16 query rows to a key/value head keys and
values too, to fp16's 11 bits (half a step: 2^-11 of each); all else in fp32.  Queries with a single feature that is not 0 and small scores keep the
errors of the scores far below that, and the features whose values cancel show the weights' rounding beside the output's own.

That the bounds can tell fp16 from bf16 is shown on the CPU, with roundings planted in the formula."""
import numpy as np
import pytest
import torch

import recurrent_drafting as rd
from quant_helpers import fill, host, scale_zero, values, wide

FP16 = 2.0 ** -11


def to_bits(x, bits):
    m, e = np.frexp(x)
    return np.ldexp(np.rint(m * 2.0 ** bits), e - bits)


def exact(cache, q, new, base, scale, many, plant=None):
    """(out, bound) [tokens, heads, dim] of one row with `new` causal tokens on `base`.  plant: significant bits that the weights are rounded to.

    Scores: products with one feature and with zero * sum q, 5 roundings of 2^-23 of at most 2 |x| (2^bits - 1) scale_k; 2^-22 of the score for the
    exponent's argument; where keys are rounded, 2^-11 |x k|.  They count twice, in a weight and in the sum.  e^x: 2^-20.  Sums of n weights: n 2^-23.
    Weights (few rows: p s / r 2^14) and values (many rows) in fp16: 2^-11 of each product p |v|, the sum of weights is that of the unrounded ones.
    fp16's smallest step: see quant_helpers.attention.  What W code and W zero come to apart (few rows) is at most r = R (2^bits - 1) times the weights' share;
    a tensor core cuts each addend of a product of 16 keys at 2^-24 of the largest, all n of them, and the two sums and their difference round."""
    l = cache.layers[0]
    hd, bits = cache.head_dim, cache.bits
    k, v = (values(host(c), host(p), bits)[0] for c, p in ((l.k_codes, l.k_params), (l.v_codes, l.v_params)))
    ks, vs = scale_zero(host(l.k_params))[0][0], scale_zero(host(l.v_params))[0][0]
    m, nh = q.shape[:2]
    out, bound = np.zeros((m, nh, hd)), np.zeros((m, nh, hd))
    top = 2 ** bits - 1
    for i in range(m):
        n = base + i + 1
        for h in range(nh):
            g = h // (nh // k.shape[0])
            x = q[i, h]
            assert np.count_nonzero(x) == 1
            s = k[g, :n] @ x * scale
            p = np.exp(s - s.max())
            total = p.sum()
            if plant is not None:
                p = to_bits(p * vs[g, :n], plant) / vs[g, :n] if not many else to_bits(p, plant)
            p /= total
            out[i, h] = p @ v[g, :n]
            err = 5 * 2.0 ** -23 * np.abs(x).sum() * 2 * top * ks[g, :n].max() * scale + 2.0 ** -22 * np.abs(s).max()
            if many:
                err += FP16 * np.abs(s).max()
            both = 2.0 ** -20 + 2 * err + n * 2.0 ** -23
            weight = both + FP16 * (2.001 if many else 1.0)
            r = vs[g, : base + new].max() * top
            bound[i, h] = weight * (p @ np.abs(v[g, :n])) + both * np.abs(out[i, h]) + (n * 2.0 ** -32 + (0.0 if many else n * 2.0 ** -24 + 2.0 ** -21)) * r
    return out, bound + 2.0 ** -8 * np.abs(out)


def case(bits, dim, new, base, device):
    cache = rd.kv_cache.QuantizedCache(1, base + new, 1, 2, dim, bits, torch.device(device))
    fill(cache, 0, 10 * new + bits)
    rng = np.random.default_rng(dim)
    q = np.zeros((new, 4, dim))
    at = rng.integers(0, dim, (new, 4))
    np.put_along_axis(q, at[..., None], to_bits(rng.uniform(0.5, 2.0, (new, 4, 1)) * rng.choice([-1, 1], (new, 4, 1)), 8), -1)
    return cache, q


SIZES = [(1, 3), (1, 7), (2, 20), (8, 1), (24, 4), (40, 1)]  # new tokens, keys before them; 2 query heads to a key/value head


def scale_of(many):
    """Scores of some 2, or where keys are rounded of some 0.4."""
    return 1 / 48 if many else 0.125


@pytest.mark.parametrize("bits, dim", [(4, 64), (8, 128)])
@pytest.mark.parametrize("new, base", SIZES)
def test_the_bounds_tell_fp16_from_bf16(bits, dim, new, base):
    cache, q = case(bits, dim, new, base, "cpu")
    many = 2 * new > 16
    want, bound = exact(cache, q, new, base, scale_of(many), many)
    assert (np.abs(exact(cache, q, new, base, scale_of(many), many, plant=11)[0] - want) <= bound).all()
    off = np.abs(to_bits(exact(cache, q, new, base, scale_of(many), many, plant=8)[0], 8) - want) / bound
    assert off.max() > 1.2, off.max()


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new, base", SIZES)
def test_rounding(bits, dim, new, base):
    cache, q = case(bits, dim, new, base, "cuda")
    want, bound = exact(cache, q, new, base, scale_of(2 * new > 16), 2 * new > 16)
    rows = torch.from_numpy(q.reshape(new, -1)).to("cuda", torch.bfloat16)
    out = torch.empty_like(rows)
    i32 = dict(dtype=torch.int32, device="cuda")
    cache.attend(0, rows, out, torch.tensor([0, new], **i32), torch.tensor([0], **i32), torch.tensor([base], **i32), new, base + new, scale=scale_of(2 * new > 16))
    off = np.abs(wide(out).reshape(want.shape) - want) / bound
    assert off.max() <= 1.0, off.max()
