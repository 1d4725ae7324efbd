"""What the operators of a cache in codes and of 8-bit products refuse, before anything is launched: runs without a GPU."""
import ctypes

import pytest
import torch

import recurrent_drafting as rd
from recurrent_drafting import _lib

P = 1 << 20  # an aligned address; nothing reads it


def order(a, names):
    """The fields of a struct, None as the null pointer."""
    assert sorted(names.split()) == sorted(a)
    return [0 if a[n] is None else a[n] for n in names.split()]


def append(**kw):
    a = dict(dtype=1, bits=4, k=P, v=P, ts=64, hs=64, kc=P, kp=P, vc=P, vp=P, row=P, slot=P, m=2, m_dev=None, B=1, nkv=2, hd=64, max_len=16)
    a.update(kw)
    return _lib.load().rd_cache_quant_append(_lib.CACHE_APPEND.pack(*order(a, "k v ts hs kc kp vc vp row slot m_dev dtype bits m B nkv hd max_len")), None)


def read(**kw):
    a = dict(dtype=1, bits=4, kc=P, kp=P, vc=P, vp=P, begin=P, length=P, B=1, nkv=2, hd=64, max_len=16, ko=P, vo=P, out_len=4)
    a.update(kw)
    return _lib.load().rd_cache_quant_read(_lib.CACHE_READ.pack(*order(a, "kc kp vc vp begin length ko vo dtype bits B nkv hd max_len out_len")), None)


def commit(**kw):
    a = dict(bits=4, codes=P, params=P, planes=2, B=1, nkv=2, max_len=16, hd=64, begin=P, base=P, unpacker=P, W=2, Lb=2, acc=P, seq=P)
    a.update(kw)
    return _lib.load().rd_cache_quant_commit(*a.values(), None)


def attend(**kw):
    a = dict(dtype=1, bits=4, q=P, ldq=128, kc=P, kp=P, vc=P, vp=P, out=P, rs=P, kb=P, bl=P, m=2, B=1, nh=2, nkv=2, hd=64, max_len=16, max_new=1, max_kv=16,
             mode=0, mask=None, words=0, scale=0.125, ws=None, ws_bytes=0, status=None)
    a.update(kw)
    return _lib.load().rd_attention_quant(_lib.ATTENTION_QUANT.pack(*order(
        a, "q ldq kc kp vc vp out rs kb bl mask ws ws_bytes status dtype bits m B nh nkv hd max_len max_new max_kv mode words scale")), None)


def rows(**kw):
    a = dict(dtype=1, x=P, ldx=64, codes=P, ld=64, scales=P, m=2, m_dev=None, K=64)
    a.update(kw)
    return _lib.load().rd_quant_rows(*a.values(), None)


def product(**kw):
    a = dict(out=1, A=P, lda=64, sa=P, W=P, ldw=64, sw=P, C=P, ldc=8, R=None, ldr=0, m=2, m_dev=None, N=8, K=64, epi=0, status=None)
    a.update(kw)
    return _lib.load().rd_gemm_int8(*a.values(), None)


def linear(**kw):
    a = dict(x=P, ldx=64, codes=P, ld=64, scales=P, W=P, ldw=64, sw=P, C=P, ldc=8, R=None, ldr=0, m_dev=None, status=None, dtype=1, out=1, m=2, N=8, K=64, epi=0)
    a.update(kw)
    return _lib.load().rd_linear_int8(_lib.LINEAR_INT8.pack(*order(a, "x ldx codes ld scales W ldw sw C ldc R ldr m_dev status dtype out m N K epi")), None)


ARG, DTYPE, SIZE, ALIGN, UNSUPPORTED = -1, -2, -3, -5, -6


@pytest.mark.parametrize("call, kw, want", [
    (append, dict(dtype=2), DTYPE), (append, dict(bits=2), UNSUPPORTED), (append, dict(hd=12), SIZE), (append, dict(hd=264), SIZE), (append, dict(hd=0), SIZE),
    (append, dict(k=None), ARG), (append, dict(slot=None), ARG), (append, dict(m=-1), ARG), (append, dict(nkv=0), ARG), (append, dict(k=P + 2), ALIGN),
    (append, dict(ts=63), ALIGN), (append, dict(kc=P + 4), ALIGN), (append, dict(vp=P + 4), ALIGN), (append, dict(dtype=0, hs=2), ALIGN),
    (read, dict(dtype=3), DTYPE), (read, dict(bits=16), UNSUPPORTED), (read, dict(hd=20), SIZE), (read, dict(length=None), ARG), (read, dict(out_len=-1), ARG),
    (read, dict(ko=P + 8), ALIGN),
    (commit, dict(bits=5), UNSUPPORTED), (commit, dict(seq=None), ARG), (commit, dict(planes=0), SIZE), (commit, dict(B=70000), SIZE),
    (attend, dict(dtype=5), DTYPE), (attend, dict(bits=3), UNSUPPORTED), (attend, dict(mode=2), UNSUPPORTED), (attend, dict(nh=3), ARG), (attend, dict(hd=10), SIZE),
    (attend, dict(max_len=20), SIZE), (attend, dict(q=None), ARG), (attend, dict(ldq=64), ARG), (attend, dict(mode=1), ARG), (attend, dict(mode=1, mask=P, words=0), ARG),
    (attend, dict(out=P + 2), ALIGN), (attend, dict(ldq=129), ALIGN), (attend, dict(scale=0.0), ARG), (attend, dict(scale=float("nan")), ARG),
    (attend, dict(B=70000), SIZE),
    (rows, dict(dtype=2), DTYPE), (rows, dict(K=0), ARG), (rows, dict(ld=48), ARG), (rows, dict(x=None), ARG), (rows, dict(codes=P + 8), ALIGN), (rows, dict(ld=72), ALIGN),
    (product, dict(out=2), DTYPE), (product, dict(epi=1), UNSUPPORTED), (product, dict(K=40), SIZE), (product, dict(K=131088, lda=131088, ldw=131088), SIZE),
    (product, dict(epi=5, N=7), SIZE), (product, dict(A=None), ARG), (product, dict(epi=4), ARG), (product, dict(lda=48), ARG), (product, dict(ldc=7), ARG),
    (linear, dict(dtype=7), DTYPE), (linear, dict(out=7), DTYPE), (linear, dict(epi=2), UNSUPPORTED), (linear, dict(K=65), ARG), (linear, dict(K=60, ld=48), ARG),
    (linear, dict(x=None), ARG), (linear, dict(W=None), ARG), (linear, dict(codes=P + 8), ALIGN), (linear, dict(ldw=72), ALIGN), (linear, dict(epi=5, N=9), SIZE),
    (product, dict(A=P + 8), ALIGN), (product, dict(ldw=72), ALIGN), (product, dict(C=P + 1), ALIGN),
])
def test_refused(call, kw, want):
    assert call(**kw) == want


@pytest.mark.parametrize("call, kw", [(append, dict(m=0)), (append, dict(B=0)), (read, dict(out_len=0)), (read, dict(B=0)), (attend, dict(m=0)), (attend, dict(B=0)),
                                      (attend, dict(max_new=0)), (rows, dict(m=0)), (product, dict(m=0)), (linear, dict(m=0))])
def test_nothing_to_do(call, kw):
    assert call(**kw) == 0


def test_cpu_tensors_and_shapes_are_refused():
    cache = rd.kv_cache.QuantizedCache(2, 20, 1, 2, 64, 4, torch.device("cpu"))
    assert cache.max_length == 20 and cache.layers[0].k_codes.shape == (2, 2, 64, 32) and cache.layers[0].v_params.shape == (2, 2, 64, 2)
    assert cache.bytes_per_token() == 2 * 2 * (32 + 4)
    x, i = torch.zeros(3, 2, 64), torch.zeros(3, dtype=torch.int32)
    with pytest.raises(rd._lib.RedrafterError, match="CPU"):
        cache.append(0, x, x, i, i)
    with pytest.raises(rd._lib.RedrafterError, match="one type"):
        cache.append(0, x, x.double(), i, i)
    with pytest.raises(rd._lib.RedrafterError, match="strides"):
        cache.append(0, x, torch.zeros(2, 3, 64).transpose(0, 1), i, i)
    with pytest.raises(rd._lib.RedrafterError, match="strides"):
        cache.append(0, torch.zeros(3, 64, 2).transpose(1, 2), torch.zeros(3, 64, 2).transpose(1, 2), i, i)
    out = torch.zeros(2, 2, 5, 64)
    with pytest.raises(rd._lib.RedrafterError, match="rows"):
        cache.read(0, i, i, out[:1], out[:1])
    with pytest.raises(rd._lib.RedrafterError, match="contiguous"):
        cache.read(0, i, i, out.transpose(1, 2).contiguous().transpose(1, 2), out)
    q = torch.zeros(3, 2 * 64)
    with pytest.raises(rd._lib.RedrafterError, match="queries"):
        cache.attend(0, q[:, :64], q[:, :64], i, i, i, 1, 4)
    with pytest.raises(rd._lib.RedrafterError, match="queries"):
        cache.attend(0, q, q[:2], i, i, i, 1, 4)
    for bad in (dict(bits=3), dict(head_dim=20)):
        kw = dict(batch_size=1, max_length=8, n_layers=1, n_heads=1, head_dim=64, bits=4, device=torch.device("cpu"))
        with pytest.raises(rd._lib.RedrafterError):
            rd.kv_cache.QuantizedCache(**{**kw, **bad})


def test_int8_linear_refuses_on_the_host():
    Int8Linear = rd.modeling_common.Int8Linear
    with pytest.raises(rd._lib.RedrafterError, match="CPU"):
        Int8Linear(torch.zeros(4, 16))
    lin = Int8Linear.from_codes(torch.zeros(4, 24, dtype=torch.int8), torch.ones(4))
    assert lin.codes.shape == (4, 32) and lin.in_features == 24
    with pytest.raises(rd._lib.RedrafterError, match="wanted"):
        lin(torch.zeros(2, 16), torch.zeros(2, 4))
    with pytest.raises(rd._lib.RedrafterError, match="residual"):
        lin(torch.zeros(2, 24), torch.zeros(2, 4), rd._lib.EPI_RES, residual=torch.zeros(2, 3))
    with pytest.raises(rd._lib.RedrafterError, match="codes"):
        Int8Linear.from_codes(torch.zeros(4, 16), torch.ones(4))
    with pytest.raises(rd._lib.RedrafterError, match="codes"):
        rd.modeling_common.quantize_rows(torch.zeros(2, 20), torch.zeros(2, 20, dtype=torch.int8), torch.zeros(2))


def test_structs_agree_with_the_header():
    sizes = [x.size for x in (_lib.CACHE_APPEND, _lib.CACHE_READ, _lib.ATTENTION_QUANT, _lib.LINEAR_INT8)]
    assert [_lib.load().rd_quant_desc_bytes(i) for i in range(4)] == sizes
    assert _lib.load().rd_quant_desc_bytes(4) < 0
    for call in ("rd_cache_quant_append", "rd_cache_quant_read", "rd_attention_quant", "rd_linear_int8"):
        assert getattr(_lib.load(), call)(None, None) == ARG


def test_workspace_sizes_are_host_calls():
    lib = _lib.load()
    assert lib.rd_attention_quant_workspace_bytes(1, 4, 1, 1, 32, 8, 128, 1, 100000) >= 0
    assert ctypes.c_int64(lib.rd_attention_quant_workspace_bytes(1, 7, 1, 1, 32, 8, 128, 1, 100000)).value < 0


def test_counts_and_status_are_int32():
    """Said before the device is looked at."""
    cache = rd.kv_cache.QuantizedCache(1, 16, 1, 2, 64, 8, torch.device("cpu"))
    k, index, wrong = torch.zeros(3, 2, 64), torch.zeros(3, dtype=torch.int32), torch.zeros(1, dtype=torch.int64)
    with pytest.raises(_lib.RedrafterError, match="int32"):
        cache.append(0, k, k, index, index, wrong)
    with pytest.raises(_lib.RedrafterError, match="int32"):
        cache.attend(0, k.reshape(3, 128), torch.zeros(3, 128), index, index, index, 3, 16, status=wrong)
    linear = rd.modeling_common.Int8Linear.from_codes(torch.zeros(16, 64, dtype=torch.int8), torch.ones(16))
    for kw in (dict(m_dev=wrong), dict(status=wrong)):
        with pytest.raises(_lib.RedrafterError, match="int32"):
            linear(torch.zeros(2, 64), torch.zeros(2, 16), **kw)
