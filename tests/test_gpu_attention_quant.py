"""Attention over a cache in codes against 64 bits, at the sizes, layouts and masks where it can go wrong."""
import numpy as np
import pytest
import torch

import recurrent_drafting as rd
from quant_helpers import HALF_STEP, attention, fill, host, i32, starts, trees, wide

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
CAUSAL, TREE = rd._lib.ATTN_CAUSAL, rd._lib.ATTN_TREE
# the softmax weights' rounding: bf16 at most for 16-bit queries; 32-bit ones keep theirs in fp32, with e^x and sums to 2^-21
WEIGHT = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -21}


def run(bits, dtype, heads, kv, dim, new, base, begin=None, mode=CAUSAL, seed=0, scale=None, capacity=None, ldq=None, slack=0, q=None, mutate=None):
    B = len(new)
    begin = [0] * B if begin is None else begin
    cache = rd.kv_cache.QuantizedCache(B, capacity or max(a + b + n for a, b, n in zip(begin, base, new)), 2, kv, dim, bits, DEV)
    fill(cache, 1, seed)
    if mutate is not None:
        mutate(cache.layers[1])
    m = sum(new)
    g = torch.Generator(device="cuda").manual_seed(seed)
    width = heads * dim
    full = torch.randn(m + slack, ldq or width, generator=g, device=DEV).to(dtype) if q is None else q
    rows = full[:, :width]
    mask = trees(new, seed + 1) if mode == TREE else None
    out = torch.full((m + slack, width), 9.0, dtype=dtype, device=DEV)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    cache.attend(1, rows, out, i32(starts(new)), i32(begin), i32(base), max(new), max(b + n for b, n in zip(base, new)), mode,
                 None if mask is None else torch.from_numpy(np.pad(mask, ((0, slack), (0, 0)))).cuda(), scale, status)
    assert int(status.item()) == 0
    assert (out[m:] == 9.0).all()
    want, bound = attention(cache, 1, wide(rows[:m]), starts(new), begin, base, mode, mask, scale or 1 / np.sqrt(dim), WEIGHT[dtype])
    return wide(out[:m]), want, bound + HALF_STEP[dtype] * np.abs(want) + 1e-30


def check(*a, **kw):
    got, want, bound = run(*a, **kw)
    off = np.abs(got - want) / bound
    assert np.isfinite(got).all() and off.max() <= 1.0, (off.max(), np.unravel_index(off.argmax(), off.shape))


BF16, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("heads, kv, dim", [(1, 1, 8), (3, 3, 40), (4, 2, 64), (8, 1, 64), (8, 8, 128), (12, 4, 128), (16, 2, 128), (5, 1, 128), (2, 1, 96), (4, 4, 256)])
def test_steps(bits, dtype, heads, kv, dim):
    """One new token a row, rows of every length, one row without a new token."""
    check(bits, dtype, heads, kv, dim, [1, 1, 1, 0, 1, 1], [0, 1, 15, 40, 64, 333], seed=dim)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("base", [31, 32, 33, 127, 128, 255, 256, 257, 511, 512, 1023, 2049, 5000])
def test_step_lengths(bits, dim, base):
    check(bits, BF16, 4, 2, dim, [1, 1], [base, base // 2], begin=[0, 3], seed=base)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("heads, kv, dim", [(4, 4, 128), (8, 2, 128), (4, 1, 64), (6, 2, 64), (3, 3, 24)])
@pytest.mark.parametrize("new, base", [([2, 3, 1], [0, 17, 100]), ([5, 16, 17], [63, 0, 200]), ([33, 64, 1, 65], [0, 31, 5, 190]), ([130, 200], [1, 77])])
def test_several_causal_tokens(bits, heads, kv, dim, new, base):
    check(bits, BF16, heads, kv, dim, new, base, begin=[7 * i for i in range(len(new))], seed=sum(new))


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("heads, kv, dim", [(4, 4, 128), (8, 2, 128), (4, 1, 64), (3, 1, 48)])
@pytest.mark.parametrize("new, base", [([1, 2], [0, 9]), ([7, 0, 31], [30, 5, 64]), ([60, 97, 140], [500, 1, 77]), ([225], [333])])
def test_draft_trees(bits, heads, kv, dim, new, base):
    check(bits, BF16, heads, kv, dim, new, base, mode=TREE, seed=sum(new))


@pytest.mark.parametrize("mode", [CAUSAL, TREE])
def test_fp32_rows(mode):
    check(8, F32, 4, 2, 64, [3, 9, 40], [0, 33, 100], begin=[1, 0, 5], mode=mode)


@pytest.mark.parametrize("new", [1, 20])
def test_strides_slack_and_scale(new):
    check(4, BF16, 4, 2, 128, [new, new], [70, 5], ldq=4 * 128 + 24, slack=3, scale=0.3)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("new, dim", [(1, 128), (1, 64), (4, 128), (40, 128), (40, 64), (1, 40)])
def test_what_lies_outside_does_not_show(bits, new, dim):
    """Rows past a row's end, before its begin and, in a tree, those a token does not see may stand for anything: NaN scales, all bits set."""
    base, begin = [50, 129], [5, 18]

    def mutate(l):
        for b in range(2):
            for params, codes in ((l.k_params, l.k_codes), (l.v_params, l.v_codes)):
                for part in (slice(0, begin[b]), slice(begin[b] + base[b] + new, None)):
                    params[b, :, part] = -1
                    codes[b, :, part] = 255

    check(bits, BF16, 4, 2, dim, [new, new], base, begin=begin, mutate=mutate, capacity=300)


@pytest.mark.parametrize("new, dim", [(1, 128), (3, 64), (40, 128), (2, 40)])
@pytest.mark.parametrize("what", ["k", "v"])
def test_nan_rows(new, dim, what):
    """A row of NaN scale among the keys makes the outputs of those that see it NaN, and no others."""
    base = 70

    def mutate(l):
        params = l.k_params if what == "k" else l.v_params
        params[0, 0, base + new - 1, 0] = 0x7FFF  # seen by the last new token of row 0 alone, in the first head's group
        params[0, 0, base + new - 1, 1] = 0

    got, want, bound = run(8, BF16, 4, 2, dim, [new, new], [base, base], mutate=mutate)
    got, want, bound = (x.reshape(2 * new, 4, dim) for x in (got, want, bound))
    odd = np.zeros((2 * new, 4, dim), bool)
    odd[new - 1, :2] = True
    assert np.array_equal(np.isnan(got), odd)
    assert (np.abs(got - want)[~odd] <= bound[~odd]).all()


@pytest.mark.parametrize("dim", [128, 64, 40])
@pytest.mark.parametrize("n", [3, 30])
def test_a_token_that_sees_nothing_is_zero(dim, n):
    cache = rd.kv_cache.QuantizedCache(1, 64, 1, 1, dim, 4, DEV)
    fill(cache, 0, 3)
    mask = np.zeros((n, 1), np.uint32)
    mask[0, 0], mask[2, 0] = 1, 5
    q = torch.randn(n, dim, device=DEV).to(BF16)
    out = torch.full_like(q, 4.0)
    cache.attend(0, q, out, i32([0, n]), i32([0]), i32([0]), n, n, TREE, torch.from_numpy(mask.view(np.int32)).cuda())
    want, bound = attention(cache, 0, wide(q), [0, n], [0], [0], TREE, mask, 1 / np.sqrt(dim), 2.0 ** -8)
    assert (out[1] == 0).all() and (np.abs(wide(out) - want) <= bound + 2.0 ** -8 * np.abs(want)).all()


@pytest.mark.parametrize("bits, dim", [(4, 128), (8, 64)])
@pytest.mark.parametrize("factor", [2.0 ** -60, 2.0 ** -20, 2.0 ** 20, 2.0 ** 60])
@pytest.mark.parametrize("new", [1, 24])
def test_queries_and_values_of_any_size(bits, dim, factor, new):
    """Queries and values far from 1 (scores kept near it): powers of two change nothing but the exponents."""
    g = torch.Generator(device="cuda").manual_seed(5)
    q = torch.randn(2 * new, 4 * dim, generator=g, device=DEV).to(BF16)

    def mutate(l):
        l.v_params[..., 0] = (l.v_params[..., 0].contiguous().view(torch.bfloat16) * factor).view(torch.int16)

    plain = run(bits, BF16, 4, 2, dim, [new, new], [100, 300], q=q, scale=0.1)[0]
    got = run(bits, BF16, 4, 2, dim, [new, new], [100, 300], q=q * factor, scale=0.1 / factor, mutate=mutate)[0]
    assert np.array_equal(got, plain * factor)


def test_peaked_and_wide_scores():
    """Large queries: the maximum moves often, most weights vanish."""
    g = torch.Generator(device="cuda").manual_seed(9)
    for new in (1, 30):
        q = (torch.randn(new, 4 * 128, generator=g, device=DEV) * 30).to(BF16)
        check(8, BF16, 4, 2, 128, [new], [1000], q=q)


def test_long_step_of_one_row():
    """Offsets past 2^31 bytes: the second of two rows of 140000 slots, 64 heads of 128 in 8 bits."""
    heads, dim, base = 64, 128, 139000
    cache = rd.kv_cache.QuantizedCache(2, 140000, 1, heads, dim, 8, DEV)
    l = cache.layers[0]
    g = torch.Generator(device="cuda").manual_seed(2)
    for codes, params in ((l.k_codes, l.k_params), (l.v_codes, l.v_params)):
        codes.copy_(torch.randint(0, 256, codes.shape, generator=g, device=DEV, dtype=torch.uint8))
        params[..., 0] = torch.full((1,), 0.01, dtype=BF16, device=DEV).view(torch.int16)
        params[..., 1] = 127
    q = torch.randn(2, heads * dim, generator=g, device=DEV).to(BF16)
    out = torch.zeros_like(q)
    cache.attend(0, q, out, i32([0, 1, 2]), i32([0, 0]), i32([5, base]), 1, base + 1)
    for h in (0, 63):  # one head at a time, in 64 bits on the device
        k = (l.k_codes[1, h, : base + 1].double() - 127) * float(torch.tensor(0.01, dtype=BF16))
        v = (l.v_codes[1, h, : base + 1].double() - 127) * float(torch.tensor(0.01, dtype=BF16))
        x = q[1, h * dim : (h + 1) * dim].double()
        p = torch.softmax(k @ x / dim ** 0.5, 0)
        # weights off by 2^-8 at most, scores by (dim + 4) 2^-23 of their absolute sum, twice; 2^-20 for e^x; the output's half step
        err = 2.0 ** -8 + 2.0 ** -20 + 4 * (dim + 4) * 2.0 ** -23 * float(x.abs().sum()) * 255 * 0.01 / dim ** 0.5
        want = p @ v
        bound = err * (p @ v.abs()) + (err + 2.0 ** -8) * want.abs()
        assert ((out[1, h * dim : (h + 1) * dim].double() - want).abs() <= bound).all()


def test_results_do_not_change_between_calls():
    a, b = (run(4, BF16, 8, 2, 128, [1, 1, 1], [3000, 5, 700])[0] for _ in range(2))
    assert np.array_equal(a, b)


def test_captured_calls_side_by_side():
    """Two captured graphs and an eager call, replayed in turn on different streams: each has its own workspace."""
    def make(seed, base):
        cache = rd.kv_cache.QuantizedCache(2, 4096, 1, 2, 128, 4, DEV)
        fill(cache, 0, seed)
        q = torch.randn(2, 8 * 128, generator=torch.Generator(device="cuda").manual_seed(seed), device=DEV).to(BF16)
        args = (q, torch.empty_like(q), i32([0, 1, 2]), i32([0, 0]), i32(base), 1, 4096)
        cache.attend(0, *args)
        torch.cuda.synchronize()
        return cache, args, args[1].clone()

    one, two = make(1, [3000, 100]), make(2, [64, 2222])
    graphs = []
    for cache, args, _ in (one, two):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            cache.attend(0, *args)
        graphs.append(graph)
    one[1][1].zero_(), two[1][1].zero_()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(10):
        for stream, graph in zip(streams, graphs):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(one[1][1], one[2]) and torch.equal(two[1][1], two[2])


@pytest.mark.parametrize("heads, kv, dim, new", [(4, 2, 128, 1), (4, 2, 64, 2), (4, 2, 128, 40), (2, 2, 40, 3)])
@pytest.mark.parametrize("most", [0, 1, 63, 200])
def test_keys_past_the_bound_are_left_out(heads, kv, dim, new, most):
    """Rows with more keys than max_kv says: the first max_kv are seen; without any the output is zero."""
    base = [300, 250]
    cache = rd.kv_cache.QuantizedCache(2, 400, 1, kv, dim, 4, DEV)
    fill(cache, 0, most)
    q = torch.randn(2 * new, heads * dim, device=DEV).to(BF16)
    out = torch.full_like(q, 4.0)
    cache.attend(0, q, out, i32(starts([new, new])), i32([0, 5]), i32(base), new, most)
    if most == 0:
        assert (out == 0).all()
        return
    nothing = np.zeros((2 * new, 1 + (new - 1) // 32), np.int32)
    want, bound = attention(cache, 0, wide(q), starts([new, new]), [0, 5], [most, most], TREE, nothing, 1 / np.sqrt(dim), 2.0 ** -8)
    assert (np.abs(wide(out) - want) <= bound + 2.0 ** -8 * np.abs(want)).all()


@pytest.mark.parametrize("new, dim", [(1, 128), (3, 64), (40, 128), (2, 40)])
def test_rows_that_begin_past_the_cache_have_no_keys(new, dim):
    cache = rd.kv_cache.QuantizedCache(2, 128, 1, 2, dim, 8, DEV)
    fill(cache, 0, 1)
    q = torch.randn(2 * new, 4 * dim, device=DEV).to(BF16)
    out = torch.full_like(q, 4.0)
    cache.attend(0, q, out, i32(starts([new, new])), i32([128, 100000]), i32([7, 0]), new, 100)
    assert (out == 0).all()


@pytest.mark.parametrize("new, dim", [(3, 128), (40, 128), (40, 64), (3, 40)])
def test_tokens_past_the_bound_are_left_alone(new, dim):
    cache = rd.kv_cache.QuantizedCache(1, 128, 1, 2, dim, 8, DEV)
    fill(cache, 0, 1)
    q = torch.randn(new, 4 * dim, device=DEV).to(BF16)
    some, all_ = torch.full_like(q, 4.0), torch.full_like(q, 4.0)
    cache.attend(0, q, all_, i32([0, new]), i32([0]), i32([70]), new, 128)
    cache.attend(0, q, some, i32([0, new]), i32([0]), i32([70]), new - 1, 128)
    assert (some[new - 1] == 4.0).all() and (some[: new - 1] != 4.0).any()
    assert (wide(some[: new - 1]) - wide(all_[: new - 1])).__abs__().max() <= 2.0 ** -6 * np.abs(wide(all_)).max()


@pytest.mark.parametrize("bits, dim", [(4, 128), (8, 64)])
@pytest.mark.parametrize("mode", [CAUSAL, TREE])
def test_more_chains_than_multiprocessors(bits, dim, mode):
    """An odd number of (row, head) chains, many of them without new tokens or with a second tile of query rows."""
    rng = np.random.default_rng(dim)
    new = [int(x) for x in rng.choice([0, 1, 17, 60, 128, 140, 150], 33)]
    base = [int(x) for x in rng.integers(0, 200, 33)]
    check(bits, BF16, 5, 5, dim, new, base, mode=mode, seed=4)


def test_no_tokens():
    cache = rd.kv_cache.QuantizedCache(2, 128, 1, 2, 64, 8, DEV)
    q = torch.empty(0, 256, dtype=BF16, device=DEV)
    cache.attend(0, q, torch.empty_like(q), i32([0, 0, 0]), i32([0, 0]), i32([7, 0]), 0, 100)
