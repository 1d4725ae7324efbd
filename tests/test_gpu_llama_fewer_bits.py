"""A Llama model whose cache is held in codes and whose projections are 8-bit integers: the operators as a decode runs them, one after another."""
import numpy as np
import pytest
import torch

import recurrent_drafting as rd
from gpu_helpers import llama_config
from quant_helpers import HALF_STEP, attention, host, int8_rows, pack, parameters, quantise, wide

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
SMALL = dict(hidden_size=256, num_attention_heads=4, num_key_value_heads=2, num_hidden_layers=1, intermediate_size=352, vocab_size=320, rms_norm_eps=1e-6,
             rope_theta=10000.0)
WIDE = dict(SMALL, hidden_size=512)  # heads of 128


def build(cfg, dtype, seed=0, **kw):
    llm = rd.modeling_llama.LlamaForCausalLM(llama_config(dict(cfg, **kw))).to("cuda", dtype)
    return llm.init_random(0.05, seed)


def planted(cfg, dtype, **kw):
    """The token after t is t + 1 by a clear margin, whatever the layers add."""
    llm = build(cfg, dtype, **kw)
    g = torch.Generator(device="cuda").manual_seed(1)
    V, H = llm.config.vocab_size, llm.config.hidden_size
    e = torch.randn(V, H, generator=g, device="cuda")
    llm.model.embed_tokens.weight.copy_(e * 4)
    llm.lm_head.weight.copy_(torch.roll(e, 1, 0))
    return llm


def extend(llm, counts, seed=3, begin=None, batch=None):
    session = rd.session.Session(llm, batch or len(counts), 200, begin=begin)
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(3, llm.config.vocab_size, (sum(counts),), generator=g).cuda()
    hidden = session.extend(ids, counts)
    session.check()
    return session, hidden


@pytest.mark.parametrize("cfg, dtype", [(SMALL, F32), (SMALL, BF16), (WIDE, BF16), (WIDE, F32)])
@pytest.mark.parametrize("bits", [4, 8])
def test_a_layer_on_a_cache_in_codes(cfg, dtype, bits):
    """The first layer's keys and values do not depend on the cache: their codes are those of the plain cache's rows, and the attention is
    that over what the codes stand for."""
    counts, begin = [70, 1, 33], [2, 0, 5]
    plain, _ = extend(build(cfg, dtype), counts, begin=begin)
    llm = build(cfg, dtype).hold_cache_in(bits)
    session, _ = extend(llm, counts, begin=begin)
    cache = session.cache
    assert isinstance(cache, rd.kv_cache.QuantizedCache) and cache.max_length == 200
    l = cache.layers[0]
    for kind, (codes, params) in enumerate(((l.k_codes, l.k_params), (l.v_codes, l.v_params))):
        for b, n in enumerate(counts):
            rows = wide(plain.cache.storage[0, kind, b, :, begin[b] : begin[b] + n])
            c, s, z = quantise(rows, bits)
            assert np.array_equal(host(codes)[b, :, begin[b] : begin[b] + n], pack(c, bits))
            assert np.array_equal(host(params)[b, :, begin[b] : begin[b] + n], parameters(s, z))
    M = sum(counts)
    ws = llm.workspace(M, 1)
    starts = np.concatenate([[0], np.cumsum(counts)])
    hd = llm.head_dim
    want, bound = attention(cache, 0, wide(ws["q"]), starts, begin, [0] * 3, 0, None, 1 / np.sqrt(hd), {BF16: 2.0 ** -8, F32: 2.0 ** -21}[dtype])
    assert (np.abs(wide(ws["attn"]) - want) <= bound + HALF_STEP[dtype] * np.abs(want) + 1e-30).all()


@pytest.mark.parametrize("cfg", [SMALL, WIDE])
def test_projections_in_8_bit_integers(cfg):
    """Each projection of a layer against integers in 64 bits, from the rows that it was given."""
    counts = [40, 7]
    plain = build(cfg, BF16, seed=5)
    gu = wide(plain.wgu[0])
    llm = build(cfg, BF16, seed=5).hold_weights_in_int8()
    assert llm.wqkv[0].numel() == 0
    _, hidden = extend(llm, counts)
    ws = llm.workspace(sum(counts), 1)
    a, sa = int8_rows(wide(ws["xn"]))  # the norm before gate and up: nothing writes it after
    w, sw = int8_rows(gu)
    v = (a @ w.T) * sa[:, None] * sw[None, :]
    gate, up = v[:, 0::2], v[:, 1::2]
    want = gate / (1 + np.exp(-gate)) * up
    # three roundings of 2^-24 each in gate (counted up to 1.1 times) and up, e^x and the division, the output's half step
    bound = (1.1 * 3 + 3 + 3) * 2.0 ** -24 * np.abs(gate * up) + 2.0 ** -20 * (2 + np.abs(gate)) * np.abs(want) + 2.0 ** -8 * np.abs(want)
    assert (np.abs(wide(ws["act"]) - want) <= bound + 1e-30).all()
    assert hidden.isfinite().all()
    for refused in (llm.reference_state_dict, lambda: llm.to(F32), lambda: llm.load_state_dict({})):
        with pytest.raises(rd._lib.RedrafterError, match="8-bit"):
            refused()
    assert llm.hold_weights_in_int8() is llm  # a second time changes nothing


@pytest.mark.parametrize("cfg, dtype, bits, int8", [(SMALL, F32, 8, False), (SMALL, BF16, 4, True), (WIDE, BF16, 4, False), (WIDE, BF16, 8, True), (WIDE, BF16, None, True)])
def test_generation(cfg, dtype, bits, int8):
    """Autoregressive and speculative decoding over codes give the planted tokens, and the same first-layer cache: what a draft's acceptance
    moved is what decoding token by token writes."""
    def model():
        llm = planted(cfg, dtype, num_hidden_layers=2).hold_cache_in(bits)
        return llm.hold_weights_in_int8() if int8 else llm

    prompt = torch.tensor([[0, 0, 5, 6, 7, 8], [20, 40, 60, 61, 62, 63], [0, 9, 11, 13, 100, 101]], device="cuda")
    special, greedy, length = rd.SpecialTokens(0, None), rd.SamplingArgs(1.0, True), 26
    want = torch.cat([prompt, prompt[:, -1:] + torch.arange(1, length - 5, device="cuda")], 1)
    llm = model()
    for out in rd.autoregressive.generate(llm, prompt, length, special, greedy):
        pass
    assert torch.equal(out, want)

    llm = model()
    H, V = llm.config.hidden_size, llm.config.vocab_size
    drafter = rd.modeling_drafter.Drafter(rd.configuration_drafter.DrafterConfig(vocab_size=V, hidden_size=H, exit_dim=2 * H, num_draft_layers=1, rnn=True))
    drafter = drafter.to("cuda", dtype)
    drafter.init_random(0.02, seed=3)
    both = rd.RecurrentDrafting(llm, drafter)
    for out in both.generate(rd.stats.Ledger(), prompt, length, rd.modeling_drafter.BeamShape(4, 3), greedy, special):
        pass
    # rows that accept more than others are longer; the yielded matrix ends with the longest
    for b in range(3):
        row = out[b].tolist()
        row = row[next(i for i, t in enumerate(row) if t):]
        first = [t for t in prompt[b].tolist() if t]
        assert row[: len(first)] == first and row[len(first):] == list(range(first[-1] + 1, first[-1] + 1 + len(row) - len(first)))
    if bits is not None:
        cache, kv_len = both.last_cache, both.last_state.kv_len.tolist()
        l = cache.layers[0]
        # a plain cache of the same tokens, one prompt of them
        again = model()
        session = rd.session.Session(again, 3, 64)
        rows = [out[b][out[b] != 0][: kv_len[b]] for b in range(3)]
        session.extend(torch.cat(rows), [len(x) for x in rows])
        m = session.cache.layers[0]
        for b in range(3):
            for x, y in zip(l, m):
                assert torch.equal(x[b, :, : len(rows[b])], y[b, :, : len(rows[b])])


def test_command_line(capsys):
    from recurrent_drafting.cmd import generate as cli

    args = ["--hf_llm", "random:tiny", "--hf_drafter", "random:1", "--batch_size", "2", "--synthetic_prompts", "2", "--beam_width", "4", "--beam_length", "3",
            "--dtype", "bf16", "--max_prompt_length", "16", "--max_generation_length", "12", "--greedy_search", "--cache_bits", "4", "--int8_weights"]
    assert cli.main(args) == 0 and "Tokens/second" in capsys.readouterr().out
    assert cli.main(args + ["--autoregression"]) == 0


def test_what_a_model_refuses():
    llm = build(SMALL, F32)
    with pytest.raises(rd._lib.RedrafterError, match="4 or 8"):
        llm.hold_cache_in(5)
    llm.hold_cache_in(8)
    session = rd.session.Session(llm, 1, 32)
    i32 = dict(dtype=torch.int32, device="cuda")
    one = torch.zeros(1, **i32)
    with pytest.raises(rd._lib.RedrafterError, match="explicit mask"):
        llm.backbone(llm.workspace(1, 1), session.cache.storage, 1, None, torch.ones(1, dtype=torch.int64, device="cuda"), one, one, one, torch.tensor([0, 1], **i32),
                     one, one, 1, 1, 1, rd._lib.ATTN_DENSE, dense_mask=torch.ones(1, 1, 1, dtype=torch.uint8, device="cuda"))
    assert isinstance(llm.hold_cache_in(None).new_cache(1, 8), rd.kv_cache.Cache)
