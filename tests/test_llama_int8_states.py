"""What a Llama model in 8-bit integers can be asked for, and what is left of one whose conversion fails."""
import pytest
import torch
from gpu_helpers import llama_config

import recurrent_drafting as rd
from recurrent_drafting import modeling_llama

CONFIG = dict(hidden_size=32, num_attention_heads=2, num_key_value_heads=1, num_hidden_layers=2, intermediate_size=48, vocab_size=40, rms_norm_eps=1e-6,
              rope_theta=10000.0)


class Held:
    """In the place of Int8Linear: refuses the calls after the first `left`."""

    left = 0

    def __init__(self, weight):
        if Held.left == 0:
            raise rd._lib.RedrafterError("no memory left")
        Held.left -= 1
        self.sum = float(weight.double().sum())


def model():
    return modeling_llama.LlamaForCausalLM(llama_config(CONFIG)).init_random(0.1, 3)


def sums(llm):
    return {name: [float(w.double().sum()) for w in ws] for name, ws in (("qkv", llm.wqkv), ("o", llm.wo), ("gu", llm.wgu), ("down", llm.wdown))}


def test_a_refused_conversion_changes_nothing():
    llm = model()
    before = sums(llm)
    for _ in range(2):
        with pytest.raises(rd._lib.RedrafterError, match="CPU"):
            llm.hold_weights_in_int8()
    assert sums(llm) == before and len(llm._lin()["qkv"]) == 2
    assert llm.to(torch.bfloat16).wqkv[1].dtype is torch.bfloat16
    assert "model.layers.1.mlp.down_proj.weight" in llm.reference_state_dict()


@pytest.mark.parametrize("first", [1, 3, 5, 7])
def test_a_conversion_goes_on_where_it_failed(monkeypatch, first):
    monkeypatch.setattr(modeling_llama, "Int8Linear", Held)
    llm = model()
    before = sums(llm)
    Held.left = first
    with pytest.raises(rd._lib.RedrafterError, match="memory"):
        llm.hold_weights_in_int8()
    for refused in (llm._lin, llm.reference_state_dict, lambda: llm.to(torch.bfloat16), lambda: llm.load_state_dict({})):
        with pytest.raises(rd._lib.RedrafterError, match="hold_weights_in_int8|8-bit"):
            refused()
    Held.left = 8 - first  # each weight once
    assert llm.hold_weights_in_int8() is llm and Held.left == 0
    assert {name: [lin.sum for lin in lins] for name, lins in llm._lin().items() if name != "head"} == before
    assert all(w.numel() == 0 for w in llm.wqkv) and all(w.numel() == 0 for w in llm.wdown)
    assert llm.hold_weights_in_int8() is llm  # a second time changes nothing


def held(monkeypatch):
    monkeypatch.setattr(modeling_llama, "Int8Linear", Held)
    Held.left = 8
    return model().hold_weights_in_int8()


def test_no_checkpoint_without_projections(monkeypatch):
    """Also as a part of a larger module, and with weights made anew: the projections in integers would stay the old ones."""
    llm = held(monkeypatch)
    embedding = llm.model.embed_tokens.weight.clone()
    both = torch.nn.ModuleDict({"llm": llm})
    for refused in (llm.state_dict, both.state_dict, llm.init_random, lambda: llm.save_pretrained("/nonexistent")):
        with pytest.raises(rd._lib.RedrafterError, match="8-bit"):
            refused()
    assert torch.equal(llm.model.embed_tokens.weight, embedding)
    assert set(torch.nn.ModuleDict({"llm": model()}).state_dict()) >= {"llm.wqkv.0", "llm.lm_head.weight"}


def test_moves_that_change_nothing(monkeypatch):
    """As RecurrentDrafting(llm, drafter).to(device) asks of a model that is there already."""
    llm = held(monkeypatch)
    drafter = rd.modeling_drafter.Drafter(rd.configuration_drafter.DrafterConfig(vocab_size=40, hidden_size=32, exit_dim=64, num_draft_layers=1, rnn=True))
    both = rd.RecurrentDrafting(llm, drafter)
    weights = [p.data_ptr() for p in llm.parameters()]
    assert both.to("cpu") is both and both.float() is both and llm.to("cpu", torch.float32) is llm and llm.cpu() is llm
    assert [p.data_ptr() for p in llm.parameters()] == weights and len(llm._lin()["qkv"]) == 2
    for moved in (lambda: both.to(torch.bfloat16), lambda: llm.to("meta"), llm.double, lambda: llm.to_empty(device="cpu")):
        with pytest.raises(rd._lib.RedrafterError, match="8-bit"):
            moved()
    assert [p.data_ptr() for p in llm.parameters()] == weights and llm.dtype is torch.float32


@pytest.mark.gpu
def test_on_the_device():
    """The same of a real conversion, and the model goes on as before."""
    llm = model().to("cuda", torch.bfloat16).hold_weights_in_int8()
    ids, counts = torch.arange(3, 12, device="cuda"), [9]
    before = rd.session.Session(llm, 1, 32).extend(ids, counts).clone()
    drafter = rd.modeling_drafter.Drafter(rd.configuration_drafter.DrafterConfig(vocab_size=40, hidden_size=32, exit_dim=64, num_draft_layers=1, rnn=True))
    both = rd.RecurrentDrafting(llm, drafter)
    assert both.to("cuda") is both and both.to(torch.device("cuda", 0), torch.bfloat16) is both and llm.cuda() is llm
    for refused in (llm.state_dict, both.state_dict, llm.init_random, llm.cpu, llm.float, llm.reference_state_dict):
        with pytest.raises(rd._lib.RedrafterError, match="8-bit"):
            refused()
    assert torch.equal(rd.session.Session(llm, 1, 32).extend(ids, counts), before)
