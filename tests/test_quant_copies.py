"""Copies of a cache in codes and of 8-bit linear layers: their calls go by addresses, which have to be the copy's own."""
import copy
import pickle

import pytest
import torch

import recurrent_drafting as rd

COPIES = [copy.deepcopy, copy.copy, lambda x: pickle.loads(pickle.dumps(x))]


@pytest.mark.parametrize("how", COPIES)
def test_linear(how):
    one = rd.modeling_common.Int8Linear.from_codes(torch.arange(64, dtype=torch.int8).view(4, 16), torch.ones(4))
    two = how(one)
    assert torch.equal(two.codes, one.codes) and torch.equal(two.scales, one.scales) and (two.in_features, two.out_features) == (16, 4)
    assert (two._codes_ptr, two._scales_ptr, two._device) == (two.codes.data_ptr(), two.scales.data_ptr(), -1)


@pytest.mark.parametrize("how", COPIES)
def test_cache(how):
    one = rd.kv_cache.QuantizedCache(2, 20, 3, 2, 64, 4, torch.device("cpu"))
    one.layers[1].k_codes.fill_(7)
    one.set_length(5)
    two = how(one)
    assert two.length == 5 and two.bytes_per_token() == one.bytes_per_token() and int(two.layers[1].k_codes.min()) == 7
    assert two._planes == [tuple(t.data_ptr() for t in l) for l in two.layers]
    assert two.layers[1].k_codes.data_ptr() - two._codes.data_ptr() == one.layers[1].k_codes.data_ptr() - one._codes.data_ptr()
    two.layers[1].k_codes.fill_(9)  # the layers are the storage, also in the copy
    assert int(two._codes[1, 0].max()) == 9 and int(one._codes[1, 0].max()) == (9 if how is copy.copy else 7)


@pytest.mark.gpu
@pytest.mark.parametrize("how", [copy.deepcopy, lambda x: pickle.loads(pickle.dumps(x))])
def test_calls_of_copies(how):
    """A copy answers as the original did, and goes on when that has changed."""
    g = torch.Generator(device="cuda").manual_seed(0)
    i32 = dict(dtype=torch.int32, device="cuda")
    cache = rd.kv_cache.QuantizedCache(1, 64, 2, 2, 64, 8, torch.device("cuda"))
    x = torch.randn(20, 2, 64, generator=g, device="cuda")
    cache.append(1, x, x, torch.zeros(20, **i32), torch.arange(20, **i32))
    lin = rd.modeling_common.Int8Linear(torch.randn(32, 128, generator=g, device="cuda"))
    q = torch.randn(1, 128, generator=g, device="cuda").to(torch.bfloat16)

    def answers(cache, lin):
        out, c = torch.empty_like(q), torch.empty(1, 32, device="cuda")
        cache.attend(1, q, out, torch.tensor([0, 1], **i32), torch.zeros(1, **i32), torch.tensor([19], **i32), 1, 20)
        lin(q, c)
        return out, c

    want = answers(cache, lin)
    copies = how(cache), how(lin)
    cache._codes.zero_(), lin.codes.zero_()
    assert all(torch.equal(a, b) for a, b in zip(answers(*copies), want))
