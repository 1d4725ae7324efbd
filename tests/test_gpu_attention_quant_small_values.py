"""Attention over a cache in codes whose values are near the smallest that bf16 holds: what has few query rows and what has many, alike."""
import numpy as np
import pytest
import torch

import recurrent_drafting as rd
from quant_helpers import attention, fill, i32, starts, wide

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def check(bits, dim, new, base, factors):
    """factors: [slots], what the value scales of a slot are multiplied with (powers of two: exact while they stay above 2^-126)."""
    B, heads, kv, slots = len(base), 4, 2, factors.numel()
    cache = rd.kv_cache.QuantizedCache(B, slots, 1, kv, dim, bits, torch.device("cuda"))
    fill(cache, 0, dim + new)
    l = cache.layers[0]
    scales = l.v_params[..., 0].contiguous().view(BF16).double() * factors.cuda()
    assert float(scales[scales > 0].min()) >= 2.0 ** -126
    l.v_params[..., 0] = scales.to(BF16).view(torch.int16)
    q = torch.randn(B * new, heads * dim, generator=torch.Generator(device="cuda").manual_seed(new), device="cuda").to(BF16)
    out, status = torch.empty_like(q), torch.zeros(1, dtype=torch.int32, device="cuda")
    counts = [new] * B
    cache.attend(0, q, out, i32(starts(counts)), i32([0] * B), i32(base), new, max(base) + new, status=status)
    assert int(status.item()) == 0
    want, bound = attention(cache, 0, wide(q), starts(counts), [0] * B, base, 0, None, dim ** -0.5, 2.0 ** -8)
    # Beside what quant_helpers says: few rows, weights p s / r 2^14 with r at least 2^-112, half of fp16's smallest step for each key;
    # many rows, values s (code - zero) 2^(100 + 6) or more in fp16, half a smallest step again, and the weights add up to 1; the output's own.
    top = 2 ** bits - 1
    small = slots * 2.0 ** -25 * 2.0 ** -14 * 2.0 ** -112 * top + 2.0 ** -25 * 2.0 ** -106 + 2.0 ** -134
    off = np.abs(wide(out) - want) / (bound + 2.0 ** -8 * np.abs(want) + small)
    assert np.abs(want).max() > 2.0 ** -124 and off.max() <= 1.0, off.max()


@pytest.mark.parametrize("bits, dim", [(4, 128), (8, 128), (4, 64), (8, 64)])
@pytest.mark.parametrize("exponent", [-98, -104, -110, -116])
@pytest.mark.parametrize("new, base", [(1, [100, 300]), (1, [3000, 5]), (24, [100, 300])])
def test_small_values(bits, dim, exponent, new, base):
    slots = (max(base) + new + 63) // 64 * 64
    check(bits, dim, new, base, torch.full((slots,), 2.0 ** exponent, dtype=torch.float64))


@pytest.mark.parametrize("bits, dim", [(4, 128), (8, 64)])
@pytest.mark.parametrize("new", [1, 24])
def test_values_that_grow_from_tile_to_tile(bits, dim, new):
    exponent = torch.linspace(-116, -102, 1088).round()
    check(bits, dim, new, [1000, 700], 2.0 ** exponent.double())
