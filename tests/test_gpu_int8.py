"""Rows as 8-bit integers and their products, against numpy in 64 bits.  The codes and the sums are exact."""
import numpy as np
import pytest
import torch

import recurrent_drafting as rd
from quant_helpers import HALF_STEP, host, i32, int8_rows, wide

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
BF16, F32 = torch.bfloat16, torch.float32
Int8Linear, quantize_rows = rd.modeling_common.Int8Linear, rd.modeling_common.quantize_rows
EPI = {"none": rd._lib.EPI_NONE, "residual": rd._lib.EPI_RES, "swiglu": rd._lib.EPI_SWIGLU}


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("m, k", [(1, 1), (2, 7), (3, 16), (5, 100), (17, 256), (4, 1000), (2, 4096), (3, 11008), (2, 20001)])
def test_rows(dtype, m, k):
    g = torch.Generator(device="cuda").manual_seed(k)
    x = (torch.randn(m, k + 3, generator=g, device=DEV) * torch.logspace(-5, 5, m, device=DEV)[:, None]).to(dtype)[:, :k]
    ld = (k + 15) // 16 * 16 + 16
    codes, scales = torch.full((m, ld), 77, dtype=torch.int8, device=DEV), torch.empty(m, device=DEV)
    quantize_rows(x, codes, scales)
    c, s = int8_rows(wide(x))
    assert np.array_equal(wide(scales), s)
    assert np.array_equal(host(codes)[:, :k], c) and (host(codes)[:, k:] == 0).all()


def test_odd_rows():
    x = torch.zeros(7, 40, device=DEV)
    x[1, 3], x[2, 0], x[3, 39] = float("nan"), float("inf"), -float("inf")
    x[4, 5] = 2.0 ** -149
    x[5, 5] = 3.3e38
    x[6] = torch.arange(40) * (-127.0 / 39)
    codes, scales = torch.empty(7, 48, dtype=torch.int8, device=DEV), torch.empty(7, device=DEV)
    quantize_rows(x, codes, scales)
    s = wide(scales)
    assert s[0] == 0 and np.isnan(s[1:4]).all() and s[4] == 0 and (host(codes)[:5] == 0).all()
    c, want = int8_rows(wide(x[5:]))
    assert np.array_equal(s[5:], want) and np.array_equal(host(codes)[5:, :40], c)


def test_half_steps_go_to_even():
    scale = 0.03125
    half = (np.arange(-127, 127) + 0.5) * scale
    x = np.concatenate([[127 * scale], half])[None]
    rows = []
    for dtype in (BF16, F32):
        t = torch.from_numpy(x).to(dtype)
        up, down = (torch.nextafter(t, torch.full_like(t, e)) for e in (1e9, -1e9))
        up[:, 0], down[:, 0] = 127 * scale, 127 * scale
        for r in (t, up, down, -t, -up):
            codes, scales = torch.empty(1, 256, dtype=torch.int8, device=DEV), torch.empty(1, device=DEV)
            quantize_rows(r.cuda(), codes, scales)
            c, s = int8_rows(wide(r))
            assert wide(scales)[0] == s[0] and np.array_equal(host(codes)[:, :255], c)
            rows.append(c)
    assert len(rows) == 10


def check(m, n, k, out, epilogue, dtype=BF16, seed=0, m_dev=None, pad=0, alias=False):
    g = torch.Generator(device="cuda").manual_seed(seed + 1000 * m + k)
    w = torch.randn(n, k, generator=g, device=DEV) * 0.05
    a = (torch.randn(m, k + pad, generator=g, device=DEV) * 2).to(dtype)[:, :k]
    lin = Int8Linear(w)
    wide_n = n // 2 if epilogue == "swiglu" else n
    c = torch.full((m, wide_n + pad), 5.0, dtype=out, device=DEV)[:, :wide_n]
    res = None
    if epilogue == "residual":
        res = torch.randn(m, wide_n, generator=g, device=DEV).to(out)
        if alias:
            c.copy_(res)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    keep = None if res is None else wide(res)
    lin(a, c, EPI[epilogue], residual=c if alias else res, m_dev=None if m_dev is None else i32([m_dev]), status=status)
    assert int(status.item()) == 0
    live = m if m_dev is None else m_dev
    got = wide(c)
    if live < m:
        assert np.array_equal(got[live:], np.full_like(got[live:], 5.0) if not alias else keep[live:])
    ca, sa = int8_rows(wide(a))
    cw, sw = int8_rows(wide(w))
    assert np.array_equal(wide(lin.scales), sw) and np.array_equal(host(lin.codes)[:, :k], cw)
    acc = (torch.from_numpy(ca).cuda() @ torch.from_numpy(cw).cuda().t()).cpu().numpy()  # whole numbers below 2^31: exact in 64 bits
    v = acc * sa[:, None] * sw[None, :]
    eps = 2.0 ** -24
    bound = 3 * eps * np.abs(v)  # the sum as fp32, the scales' product (exact: 8 bits each), their product
    if epilogue == "residual":
        want = v + keep
        bound = bound + eps * np.abs(want)
    elif epilogue == "swiglu":
        gate, up = v[:, 0::2], v[:, 1::2]
        sig = 1 / (1 + np.exp(-gate))
        want = gate * sig * up
        # |d(g sig g)/dg| <= 1.1, so the gate's error counts up to 1.1 |up| of itself; e^-g and the division: 2^-20 of what e^-g weighs in
        # the sum (fast forms, bf16 outputs), 2^-21 with the exact ones
        bound = 1.1 * bound[:, 0::2] * np.abs(up) + (3 * eps + (2.0 ** -20 if out == BF16 else 2.0 ** -21) * (2 + np.abs(gate))) * np.abs(want)
    else:
        want = v
    off = np.abs(got - want)[:live] / (bound + HALF_STEP[out] * np.abs(want) + 1e-35)[:live]
    assert live == 0 or off.max() <= 1.0, (off.max(), np.unravel_index(off.argmax(), off.shape))


@pytest.mark.parametrize("epilogue", ["none", "residual", "swiglu"])
@pytest.mark.parametrize("out", [BF16, F32])
@pytest.mark.parametrize("m, n, k", [(1, 2, 1), (1, 64, 16), (3, 70, 40), (1, 1000, 512), (16, 130, 256), (17, 4096, 128), (33, 258, 1040), (64, 256, 4096), (129, 514, 144)])
def test_products(m, n, k, out, epilogue):
    check(m, n, k, out, epilogue)


@pytest.mark.parametrize("m", [1, 2, 15, 16, 31, 32, 63, 65, 96, 127, 128, 130, 191, 192, 193, 255, 256, 257, 300, 511, 513, 1000])
@pytest.mark.parametrize("n, k, epilogue", [(384, 320, "none"), (6144, 256, "residual"), (1030, 640, "swiglu")])
def test_row_counts(m, n, k, epilogue):
    check(m, n, k, BF16, epilogue)


@pytest.mark.parametrize("m, n, k, epilogue", [(1, 12288, 4096, "none"), (110, 4096, 11008, "residual"), (777, 5632, 2048, "swiglu"), (2050, 4096, 1024, "none")])
def test_sizes_of_models(m, n, k, epilogue):
    check(m, n, k, BF16, epilogue)


@pytest.mark.parametrize("m, live", [(40, 0), (40, 1), (40, 33), (300, 17), (300, 260), (600, 5)])
@pytest.mark.parametrize("epilogue", ["none", "residual"])
def test_live_rows(m, live, epilogue):
    check(m, 512, 256, BF16, epilogue, m_dev=live)


@pytest.mark.parametrize("m", [1, 50, 300])
def test_strided_rows_and_aliased_residual(m):
    check(m, 200, 96, F32, "none", dtype=F32, pad=5)
    check(m, 200, 96, BF16, "none", pad=8)
    check(m, 201, 96, BF16, "none", pad=3)
    check(m, 256, 96, BF16, "residual", alias=True)
    check(m, 250, 96, F32, "residual", alias=True)


@pytest.mark.parametrize("m", [1, 200])
def test_largest_sums(m):
    """K = 131072 products of 127 * 127: 2.11e9, below 2^31."""
    k, n = 131072, 256
    codes = torch.full((n, k), 127, dtype=torch.int8, device=DEV)
    codes[1::2] = -127
    lin = Int8Linear.from_codes(codes, torch.ones(n, device=DEV))
    c = torch.empty(m, n, device=DEV)
    lin(torch.full((m, k), 127.0, device=DEV), c)
    want = np.where(np.arange(n) % 2, -1.0, 1.0) * 127 * 127 * k
    assert np.array_equal(wide(c), np.broadcast_to(want, (m, n)))  # 127^2 2^17 has 14 bits


def test_nan_rows_stay_in_their_rows():
    for m in (3, 300):
        x = torch.randn(m, 128, device=DEV).to(BF16)
        x[1, 5] = float("nan")
        w = torch.randn(64, 128, device=DEV)
        w[7, 1] = float("inf")
        c = torch.empty(m, 64, dtype=BF16, device=DEV)
        Int8Linear(w)(x, c)
        odd = torch.zeros(m, 64, dtype=torch.bool, device=DEV)
        odd[1], odd[:, 7] = True, True
        assert torch.equal(c.isnan(), odd)


def test_captured_products_and_another_stream():
    g = torch.Generator(device="cuda").manual_seed(3)
    lin = Int8Linear(torch.randn(512, 256, generator=g, device=DEV))
    x = torch.randn(20, 256, generator=g, device=DEV).to(BF16)
    c, want = torch.empty(20, 512, dtype=BF16, device=DEV), torch.empty(20, 512, dtype=BF16, device=DEV)
    lin(x, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        lin(x, c)
    c.zero_()
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(c, want)
    x.mul_(-1)  # the captured call reads its input anew
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(c, -want)
