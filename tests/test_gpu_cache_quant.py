"""A cache in codes: rows as they are quantised, read back, moved, against numpy in 64 bits.  Codes and parameters are compared exactly."""
import numpy as np
import pytest
import torch

import recurrent_drafting as rd
from quant_helpers import fill, host, i32, pack, parameters, quantise, values, wide

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")


def new(batch, length, layers, heads, dim, bits):
    return rd.kv_cache.QuantizedCache(batch, length, layers, heads, dim, bits, DEV)


def planes(cache, layer=0):
    l = cache.layers[layer]
    return (l.k_codes, l.k_params), (l.v_codes, l.v_params)


def expect(cache, x, kind):
    """(codes, params) of rows x as the definition has them."""
    c, s, z = quantise(wide(x), cache.bits)
    return pack(c, cache.bits), parameters(s, z)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads, dim", [(1, 8), (3, 24), (2, 64), (5, 96), (8, 128), (2, 256)])
def test_append_and_read(bits, dtype, heads, dim):
    g = torch.Generator(device="cuda").manual_seed(dim + bits)
    B, base, counts = 3, [0, 7, 61], [5, 0, 40]
    cache = new(B, 101, 2, heads, dim, bits)
    m = sum(counts)
    both = (torch.randn(m, 2, heads, dim, generator=g, device=DEV) * torch.logspace(-6, 6, m, device=DEV)[:, None, None, None]).to(dtype)
    k, v = both[:, 0], both[:, 1]  # rows of a projection: strided
    row = [b for b, c in enumerate(counts) for _ in range(c)]
    slot = [base[b] + i for b, c in enumerate(counts) for i in range(c)]
    order = np.random.default_rng(1).permutation(m)  # tokens in any order
    cache.append(1, k[torch.from_numpy(order).cuda()], v[torch.from_numpy(order).cuda()], i32(np.array(row)[order]), i32(np.array(slot)[order]))
    for (codes, params), x in zip(planes(cache, 1), (k, v)):
        want_c, want_p = np.zeros(codes.shape, np.uint8), np.zeros(params.shape, np.int16)
        c, p = expect(cache, x, dtype)
        want_c[row, :, slot], want_p[row, :, slot] = c, p
        assert np.array_equal(host(params), want_p)
        assert np.array_equal(host(codes), want_c)
    assert not any(t.any() for pair in planes(cache, 0) for t in pair)  # the other layer
    # the same through strides of their own
    again = new(B, 101, 2, heads, dim, bits)
    again.append(1, k, v, i32(row), i32(slot))
    assert all(torch.equal(a, b) for p, q in zip(planes(cache, 1), planes(again, 1)) for a, b in zip(p, q))
    for out_dtype in (torch.bfloat16, torch.float32):
        k_out, v_out = (torch.full((B, heads, 45, dim), 7.0, dtype=out_dtype, device=DEV) for _ in range(2))
        cache.read(1, i32(base), i32(counts), k_out, v_out)
        for out, (codes, params) in zip((k_out, v_out), planes(cache, 1)):
            full = values(host(codes), host(params), bits)
            want = torch.full((B, heads, 45, dim), 7.0, dtype=torch.float64)
            for b in range(B):
                want[b, :, : counts[b]] = torch.from_numpy(full[b, :, base[b] : base[b] + counts[b]])
            assert torch.equal(out.cpu(), want.float().to(out_dtype))  # scale * (code - zero) has 17 bits: exact in fp32, rounded once


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_half_steps_go_to_even(bits, dtype):
    """Values exactly half way between two codes, and their neighbours."""
    q = 2 ** bits - 1
    scale = 0.0390625  # 5 / 128
    half = (np.arange(q) + 0.5) * scale
    x = np.zeros((3, 1, 256))
    x[:, 0, 0] = q * scale  # the row's largest: its scale is the one above
    n = min(255, q)
    x[0, 0, 1 : n + 1] = half[:n]
    up = torch.from_numpy(half).to(dtype)
    x[1, 0, 1 : n + 1] = torch.nextafter(up, torch.full_like(up, 1e9)).double().numpy()[:n]
    x[2, 0, 1 : n + 1] = torch.nextafter(up, torch.full_like(up, -1e9)).double().numpy()[:n]
    t = torch.from_numpy(x).to(dtype).cuda()
    cache = new(1, 3, 1, 1, 256, bits)
    cache.append(0, t, -t, i32([0, 0, 0]), i32([0, 1, 2]))
    for (codes, params), r in zip(planes(cache), (t, -t)):
        c, p = expect(cache, r.transpose(0, 1), dtype)
        assert np.array_equal(host(params)[0, :, :3], p) and np.array_equal(host(codes)[0, :, :3], c)


@pytest.mark.parametrize("bits", [4, 8])
def test_odd_rows(bits):
    """Zeros, constants, one sign only, the smallest and the largest numbers, NaN and infinities."""
    tiny, huge = 2.0 ** -149, 3.0e38
    rows = np.zeros((12, 64), np.float32)
    rows[1] = 5.0
    rows[2] = -5.0
    rows[3] = np.linspace(1, 2, 64)
    rows[4] = -np.linspace(1, 2, 64)
    rows[5, 3] = tiny
    rows[6, 3] = huge
    rows[7, 3], rows[7, 4] = huge, -huge  # a range past fp32
    rows[8, 3], rows[9, 3], rows[10, 3] = np.nan, np.inf, -np.inf
    rows[11] = np.random.default_rng(0).standard_normal(64) * 1e30
    t = torch.from_numpy(rows).cuda()[:, None]
    cache = new(1, 12, 1, 1, 64, bits)
    cache.append(0, t, t, i32([0] * 12), i32(range(12)))
    out = torch.empty(1, 1, 12, 64, device=DEV)
    cache.read(0, i32([0]), i32([12]), out, torch.empty_like(out))
    got = wide(out)[0, 0]
    assert np.isnan(got[7:11]).all()
    assert (got[0] == 0).all() and (got[5] == 0).all()  # a scale of tiny / Q is 0
    for i in (1, 2, 3, 4, 6, 11):
        c, s, z = quantise(rows[i].astype(np.float64), bits)
        assert np.array_equal(got[i], (s * (c - z)).astype(np.float32).astype(np.float64)), i
        # half a step, the scale's own rounding over all Q of them, and zero's
        assert np.abs(got[i] - rows[i]).max() <= s[0] * (1.0 + (2 ** bits - 1) * 2.0 ** -8), i


def test_places_outside_are_left_out():
    cache = new(2, 64, 1, 2, 64, 8)
    x = torch.ones(6, 2, 64, device=DEV)
    cache.append(0, x, x, i32([0, -1, 2, 1, 1, 1]), i32([3, 0, 0, -1, 64, 63]))
    want = np.zeros((2, 2, 64), bool)
    want[0, :, 3] = want[1, :, 63] = True
    assert np.array_equal(host(cache.layers[0].k_codes).any(-1), want) and np.array_equal(host(cache.layers[0].v_params).any(-1), want)


def test_live_count_on_the_device():
    cache = new(1, 64, 1, 2, 64, 4)
    x = torch.ones(6, 2, 64, device=DEV)
    cache.append(0, x, x, i32([0] * 6), i32(range(6)), m_dev=i32([4]))
    assert host(cache.layers[0].k_codes).any(-1)[0, 0].tolist() == [True] * 4 + [False] * 60


@pytest.mark.parametrize("bits", [4, 8])
def test_read_bounds(bits):
    """Rows of no length, longer than the output, past the cache's end, with a negative begin."""
    cache = new(5, 64, 1, 3, 72, bits)
    fill(cache, 0, 5)
    begin, length = [0, 10, 60, -3, 63], [0, 50, 50, 4, 1]
    out = [torch.full((5, 3, 7, 72), 3.0, device=DEV) for _ in range(2)]
    cache.read(0, i32(begin), i32(length), *out)
    counts = [0, 7, 4, 0, 1]
    for o, (codes, params) in zip(out, planes(cache)):
        full, want = values(host(codes), host(params), bits), np.full((5, 3, 7, 72), 3.0)
        for b, n in enumerate(counts):
            want[b, :, :n] = full[b, :, begin[b] : begin[b] + n]
        assert np.array_equal(wide(o), want.astype(np.float32).astype(np.float64))


@pytest.mark.parametrize("bits, dim", [(4, 64), (8, 128), (4, 8), (8, 256)])
def test_commit_moves_the_accepted_path(bits, dim):
    B, W, L, heads = 3, 4, 3, 2
    cache = new(B, 70, 2, heads, dim, bits)
    fill(cache, 0, 1)
    fill(cache, 1, 2)
    before = [[(host(c), host(p)) for c, p in planes(cache, layer)] for layer in range(2)]
    rng = np.random.default_rng(3)
    unpacker = np.stack([np.sort(rng.permutation(W * L)[: W * L]).reshape(W, L) for _ in range(B)])
    seq, acc, base, begin = [1, 3, 0], [2, 0, 1], [5, 20, 0], [0, 3, 50]

    class Pack:
        pass

    fp = Pack()
    fp.base_len, fp.unpacker = i32(base), i32(unpacker)
    cache.commit_draft(fp, i32(acc), i32(seq), rd.modeling_drafter.BeamShape(W, L), i32(begin))
    for layer in range(2):
        for (c, p), (c0, p0) in zip(planes(cache, layer), before[layer]):
            c0, p0 = c0.copy(), p0.copy()
            for b in range(B):
                s = begin[b] + base[b]
                for j in range(acc[b] + 1):
                    c0[b, :, s + j], p0[b, :, s + j] = c0[b, :, s + unpacker[b, seq[b], j]], p0[b, :, s + unpacker[b, seq[b], j]]
            assert np.array_equal(host(c), c0) and np.array_equal(host(p), p0)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_read_of_long_rows(bits, dtype):
    """Rows that take many steps of a thread block, next to short and empty ones."""
    B, heads, dim, length, begin = 4, 8, 64, [6000, 1, 0, 4097], [3, 0, 9, 1900]
    cache = new(B, 6016, 1, heads, dim, bits)
    fill(cache, 0, 5)
    k, v = (torch.full((B, heads, 6001, dim), 7.0, dtype=dtype, device="cuda") for _ in range(2))
    cache.read(0, i32(begin), i32(length), k, v)
    layer = cache.layers[0]
    for codes, params, got in ((layer.k_codes, layer.k_params, k), (layer.v_codes, layer.v_params, v)):
        c = codes if bits == 8 else torch.stack([codes & 15, codes >> 4], dim=-1).flatten(-2)
        want = params[..., 0:1].contiguous().view(torch.bfloat16).float() * (c.float() - params[..., 1:2].float())  # exact
        for b in range(B):
            assert torch.equal(got[b, :, : length[b]], want[b, :, begin[b] : begin[b] + length[b]].to(dtype))
            assert (got[b, :, length[b] :] == 7.0).all()


def test_commit_stays_inside_the_cache():
    """A path whose tokens would lie past the last slot, and a sequence that there is not: nothing moves."""
    cache = new(2, 64, 1, 2, 64, 8)
    fill(cache, 0, 1)
    before = [(host(c), host(p)) for c, p in planes(cache, 0)]

    class Pack:
        pass

    fp = Pack()
    fp.base_len, fp.unpacker = i32([62, 5]), i32(np.tile([0, 3, 6], (2, 2, 1)).reshape(-1).tolist())
    cache.commit_draft(fp, i32([2, 2]), i32([1, 2]), rd.modeling_drafter.BeamShape(2, 3), i32([0, 0]))
    for (c, p), (c0, p0) in zip(planes(cache, 0), before):
        assert np.array_equal(host(c), c0) and np.array_equal(host(p), p0)
