"""Attention over a cache in codes whose bounds of new tokens and keys are those of a capacity, as captured steps have them, and not of the rows that are there."""
import numpy as np
import pytest
import torch

import recurrent_drafting as rd
from quant_helpers import attention, fill, i32, starts, trees, wide

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits, dim", [(4, 128), (8, 64), (8, 40)])
@pytest.mark.parametrize("max_new, max_kv", [(0, 3000), (5, 0), (225, 4096)])  # beyond what is needed
@pytest.mark.parametrize("new, base", [([1, 1, 0], [300, 5, 70]), ([3, 14, 1], [0, 129, 600]), ([60, 1, 33], [90, 0, 411])])
@pytest.mark.parametrize("tree", [False, True])
def test_bounds_of_a_capacity(bits, dim, max_new, max_kv, new, base, tree):
    max_new, max_kv = max_new + max(new), max_kv + max(b + n for b, n in zip(base, new))
    cache = rd.kv_cache.QuantizedCache(3, 700, 1, 2, dim, bits, torch.device("cuda"))
    fill(cache, 0, dim)
    m = sum(new)
    q = torch.randn(m, 4 * dim, generator=torch.Generator(device="cuda").manual_seed(m), device="cuda").to(torch.bfloat16)
    mask = trees(new, m, words=(max_new + 31) // 32) if tree else None
    out, status = torch.full_like(q, 9.0), torch.zeros(1, dtype=torch.int32, device="cuda")
    cache.attend(0, q, out, i32(starts(new)), i32([0, 7, 19]), i32(base), max_new, max_kv, rd._lib.ATTN_TREE if tree else rd._lib.ATTN_CAUSAL,
                 None if mask is None else torch.from_numpy(mask).cuda(), status=status)
    want, bound = attention(cache, 0, wide(q), starts(new), [0, 7, 19], base, int(tree), mask, dim ** -0.5, 2.0 ** -8)
    assert int(status.item()) == 0 and (np.abs(wide(out) - want) <= bound + 2.0 ** -8 * np.abs(want) + 1e-30).all()
