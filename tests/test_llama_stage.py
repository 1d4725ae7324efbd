"""Where a Llama model on a cache in codes keeps a step's keys and values before they are quantised."""
import pytest
import torch
from gpu_helpers import llama_config

import recurrent_drafting as rd

CONFIG = dict(hidden_size=256, num_attention_heads=4, num_key_value_heads=2, num_hidden_layers=2, intermediate_size=352, vocab_size=320, rms_norm_eps=1e-6,
              rope_theta=10000.0)


def test_smaller_portions_take_a_part_of_it():
    llm = rd.modeling_llama.LlamaForCausalLM(llama_config(CONFIG))
    first = llm._stage_of(20)
    assert all(llm._stage_of(m) is first for m in (20, 1, 19, 7, 20))
    more = llm._stage_of(33)
    assert more is not first and llm._stage_of(20) is more and more["k"].shape == (1, 2, 33, 64)
    assert more["slot"].tolist() == list(range(33)) and not more["row"].any()
    assert {t.data_ptr() for t in more.values()} <= {t.data_ptr() for t in llm.held_buffers()}  # what captured steps keep alive


@pytest.mark.gpu
@pytest.mark.parametrize("hidden", [256, 512])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("int8", [False, True])
def test_portions_of_other_sizes_between(hidden, dtype, int8):
    """Two sessions, their portions of different sizes in turn: the codes of each are those of a model that serves it alone."""
    def model():
        llm = rd.modeling_llama.LlamaForCausalLM(llama_config(dict(CONFIG, hidden_size=hidden))).to("cuda", dtype).init_random(0.05, 3).hold_cache_in(8)
        return llm.hold_weights_in_int8() if int8 else llm

    g = torch.Generator().manual_seed(1)
    portions = [(0, [9, 3]), (1, [1]), (0, [2, 0]), (1, [40]), (0, [1, 1]), (1, [1]), (0, [1, 1])]
    portions = [(which, counts, torch.randint(3, 320, (sum(counts),), generator=g).cuda()) for which, counts in portions]

    def serve(llms):
        sessions = [rd.session.Session(llm, batch, 64) for llm, batch in zip(llms, (2, 1))]
        hidden = [sessions[which].extend(ids, counts).clone() for which, counts, ids in portions]
        for s in sessions:
            s.check()
        return hidden, [p for s in sessions for layer in s.cache.layers for p in layer]

    one = model()
    got, want = serve([one, one]), serve([model(), model()])
    for a, b in zip(got[0] + got[1], want[0] + want[1]):
        assert torch.equal(a, b)
