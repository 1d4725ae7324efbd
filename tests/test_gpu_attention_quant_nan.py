"""NaN in queries and keys of an attention over a cache in codes: whoever sees it is NaN, also where no score is a number."""
import numpy as np
import pytest
import torch

import recurrent_drafting as rd
from quant_helpers import attention, fill, i32, starts, wide

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
NAN_SCALE = 0x7FFF


def run(dim, dtype, new, base, spoil):
    """Two rows of `new` tokens on base keys, 4 heads on 2; spoil(layer, q) plants NaN.  Returns (out, want, bound), [tokens, heads, dim]."""
    cache = rd.kv_cache.QuantizedCache(2, max(base) + new, 1, 2, dim, 8, torch.device("cuda"))
    fill(cache, 0, dim)
    g = torch.Generator(device="cuda").manual_seed(new)
    q = torch.randn(2 * new, 4, dim, generator=g, device="cuda").to(dtype)
    clean = wide(q).reshape(2 * new, -1)
    want, bound = attention(cache, 0, clean, starts([new, new]), [0, 0], base, 0, None, dim ** -0.5, 2.0 ** -8)
    spoil(cache.layers[0], q)
    out = torch.full((2 * new, 4 * dim), 4.0, dtype=dtype, device="cuda")
    cache.attend(0, q.view(2 * new, -1), out, i32(starts([new, new])), i32([0, 0]), i32(base), new, max(base) + new)
    return (x.reshape(2 * new, 4, dim) for x in (wide(out), want, bound))


def check(odd, got, want, bound):
    assert np.array_equal(np.isnan(got), np.broadcast_to(odd[..., None], got.shape))
    assert (np.abs(got - want) <= bound + 2.0 ** -8 * np.abs(want) + 1e-30)[~odd].all()


KINDS = [(128, BF16), (64, BF16), (40, BF16), (64, F32)]


@pytest.mark.parametrize("dim, dtype", KINDS)
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("new, base", [(1, [0, 50]), (1, [300, 4000]), (3, [0, 17]), (40, [0, 100]), (40, [3000, 2000])])
def test_queries(dim, dtype, value, new, base):
    """One head's query of one token: all its scores are NaN (or infinite), so its output is, whatever its keys; nobody else's."""
    odd = np.zeros((2 * new, 4), bool)
    odd[0, 1] = odd[2 * new - 1, 2] = True

    def spoil(layer, q):
        # a key has features of both signs, so every score is inf - inf or inf * 0
        q[torch.from_numpy(odd).cuda()] = value

    check(odd, *run(dim, dtype, new, base, spoil))


@pytest.mark.parametrize("dim, dtype", KINDS)
@pytest.mark.parametrize("new, base", [(1, [0, 70]), (1, [16, 128]), (1, [1000, 4000]), (20, [0, 2000])])
@pytest.mark.parametrize("kind", ["keys", "values"])
def test_keys_all_of_them(dim, dtype, new, base, kind):
    """Every key (or value) of a head is NaN: no score is a number."""
    odd = np.zeros((2 * new, 4), bool)
    odd[:, :2] = True

    def spoil(layer, q):
        params = layer.k_params if kind == "keys" else layer.v_params
        params[:, 0, :, 0], params[:, 0, :, 1] = NAN_SCALE, 0

    check(odd, *run(dim, dtype, new, base, spoil))


@pytest.mark.parametrize("dim, dtype", KINDS)
@pytest.mark.parametrize("new, base, at", [(1, [16, 16], 16), (1, [128, 128], 128), (1, [1024, 1500], 1024), (1, [4000, 4000], 7), (20, [2100, 2100], 63)])
def test_one_key(dim, dtype, new, base, at):
    """One key of one row and head, alone in its tile or one among many."""
    odd = np.zeros((2 * new, 4), bool)
    odd[new:, 2:] = True

    def spoil(layer, q):
        layer.k_params[1, 1, at, 0], layer.k_params[1, 1, at, 1] = NAN_SCALE, 0

    check(odd, *run(dim, dtype, new, base, spoil))
