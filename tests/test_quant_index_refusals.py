"""Indices and counts of the operators in codes that would be read past their end, or as other numbers: refused on the host.  Runs without a GPU."""
import types

import pytest
import torch

import recurrent_drafting as rd

B, W, L = 2, 3, 4
SHAPE = rd.modeling_drafter.BeamShape(W, L)


def commit(**kw):
    cache = rd.kv_cache.QuantizedCache(B, 64, 1, 2, 64, 8, torch.device("cpu"))
    i = torch.zeros(B, dtype=torch.int32)
    a = dict(unpacker=torch.zeros(B, W, L, dtype=torch.int32), base_len=i, kv_begin=i, n_accepted=i, seq_in_beam=i)
    a.update(kw)
    fp = types.SimpleNamespace(unpacker=a["unpacker"], base_len=a["base_len"])
    cache.commit_draft(fp, a["n_accepted"], a["seq_in_beam"], SHAPE, a["kv_begin"])


@pytest.mark.parametrize("name", ["base_len", "kv_begin", "n_accepted", "seq_in_beam", "unpacker"])
@pytest.mark.parametrize("spoil", [lambda t: t.long(), lambda t: t[:1], lambda t: torch.stack([t, t], -1)[..., 0]])
def test_commit(name, spoil):
    good = torch.zeros(B, W, L, dtype=torch.int32) if name == "unpacker" else torch.zeros(B, dtype=torch.int32)
    with pytest.raises(rd._lib.RedrafterError, match=f"{name} is a contiguous int32"):
        commit(**{name: spoil(good)})


def test_commit_on_the_cpu():
    with pytest.raises(rd._lib.RedrafterError, match="CPU"):
        commit()


@pytest.mark.parametrize("count", [torch.zeros(1, dtype=torch.int64), torch.zeros(0, dtype=torch.int32), torch.zeros(1)])
def test_row_quantiser(count):
    with pytest.raises(rd._lib.RedrafterError, match="m_dev is an int32 count"):
        rd.modeling_common.quantize_rows(torch.zeros(2, 16), torch.zeros(2, 16, dtype=torch.int8), torch.zeros(2), count)


@pytest.mark.parametrize("name", ["m_dev", "status"])
def test_empty_counts(name):
    """An empty tensor has no count in it."""
    none = torch.zeros(0, dtype=torch.int32)
    cache = rd.kv_cache.QuantizedCache(1, 16, 1, 2, 64, 8, torch.device("cpu"))
    k, i = torch.zeros(3, 2, 64), torch.zeros(3, dtype=torch.int32)
    linear = rd.modeling_common.Int8Linear.from_codes(torch.zeros(16, 64, dtype=torch.int8), torch.ones(16))
    with pytest.raises(rd._lib.RedrafterError, match="int32"):
        linear(torch.zeros(2, 64), torch.zeros(2, 16), **{name: none})
    with pytest.raises(rd._lib.RedrafterError, match="int32"):
        if name == "m_dev":
            cache.append(0, k, k, i, i, none)
        else:
            cache.attend(0, k.view(3, 128), torch.zeros(3, 128), i, i, i, 3, 16, status=none)
