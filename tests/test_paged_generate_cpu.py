"""What PagedGenerator refuses, seen without a GPU."""

import pytest
import torch
from torch import nn
from transformers import AutoModelForCausalLM, LlamaConfig

from neuralzip_b200.gpu.generate import PagedCache, PagedGenerator, _rotates_neighbours, _token_ids


def _model(**more):
    config = LlamaConfig(hidden_size=64, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2,
                         intermediate_size=128, vocab_size=97, **more)
    torch.manual_seed(0)
    return AutoModelForCausalLM.from_config(config, dtype=torch.bfloat16).eval()


def test_refuses_a_model_off_the_gpu():
    with pytest.raises(ValueError, match="CUDA device"):
        PagedGenerator(_model(), requests=2, max_length=32)


def test_refuses_length_dependent_rotary():
    model = _model(rope_parameters=dict(rope_type="dynamic", factor=2.0, rope_theta=10000.0))
    with pytest.raises(ValueError, match="dynamic"):
        PagedGenerator(model, requests=2, max_length=32)


def test_refuses_other_attention():
    model = _model()
    model.model.layers[1].self_attn.gate = nn.Linear(4, 4)
    with pytest.raises(ValueError, match="not an attention"):
        PagedGenerator(model, requests=2, max_length=32)
    model = _model()
    model.model.layers[0].self_attn.sinks = nn.Parameter(torch.zeros(4))
    with pytest.raises(ValueError, match="not an attention"):
        PagedGenerator(model, requests=2, max_length=32)
    model = _model()
    model.model.layers[0].self_attn.q_norm = nn.LayerNorm(16)
    with pytest.raises(ValueError, match="root-mean-square"):
        PagedGenerator(model, requests=2, max_length=32)
    model = _model()
    model.config.attn_logit_softcapping = 30.0
    with pytest.raises(ValueError, match="capped"):
        PagedGenerator(model, requests=2, max_length=32)
    with pytest.raises(ValueError, match="multiple of 8"):
        PagedGenerator(_model(head_dim=12), requests=2, max_length=32)
    model = _model()
    del model.model.rotary_emb
    with pytest.raises(ValueError, match="rotary"):
        PagedGenerator(model, requests=2, max_length=32)


def test_reads_the_rotary_pairing_from_the_model():
    assert _rotates_neighbours(_model().model.layers[0].self_attn) is False
    with pytest.raises(ValueError, match="unknown way"):
        _rotates_neighbours(nn.Linear(2, 2))


def test_cache_sizes():
    sizes = dict(requests=3, pages=5, page_size=16, max_length=40, dtype=torch.bfloat16, device="cpu")
    cache = PagedCache(2, 2, 16, **sizes)
    assert cache.block_table.shape == (3, 3) and cache.pages == 5 and cache.pages_for(17) == 2
    for change in (dict(requests=0), dict(requests=4097), dict(pages=0), dict(page_size=12), dict(max_length=0)):
        with pytest.raises(ValueError):
            PagedCache(2, 2, 16, **{**sizes, **change})


def test_refuses_unknown_model_types():
    """Other types' attention may differ in ways that its modules do not show: only where the caller says so."""
    model = _model()
    model.config.model_type = "other"
    with pytest.raises(ValueError, match="other_types"):
        PagedGenerator(model, requests=2, max_length=32)
    with pytest.raises(ValueError, match="CUDA device"):  # as far as a model on the CPU gets
        PagedGenerator(model, requests=2, max_length=32, other_types=True)


def test_refuses_a_window_that_the_attention_does_not_tell():
    model = _model()
    model.config.sliding_window = 16
    with pytest.raises(ValueError, match="sliding window"):
        PagedGenerator(model, requests=2, max_length=32)
    for layer in model.model.layers:
        layer.self_attn.sliding_window = 16
    with pytest.raises(ValueError, match="CUDA device"):
        PagedGenerator(model, requests=2, max_length=32)


def test_refuses_norms_of_different_epsilon():
    """One epsilon goes to the rotary pass: two would give the queries the keys' one."""
    from transformers.models.llama.modeling_llama import LlamaRMSNorm

    model = _model()
    for layer in model.model.layers:
        layer.self_attn.q_norm, layer.self_attn.k_norm = LlamaRMSNorm(16, eps=1e-5), LlamaRMSNorm(16, eps=1e-5)
    with pytest.raises(ValueError, match="CUDA device"):
        PagedGenerator(model, requests=2, max_length=32)
    model.model.layers[1].self_attn.k_norm = LlamaRMSNorm(16, eps=1e-2)
    with pytest.raises(ValueError, match="same epsilon"):
        PagedGenerator(model, requests=2, max_length=32)
    del model.model.layers[1].self_attn.q_norm  # a key norm alone has its own
    with pytest.raises(ValueError, match="CUDA device"):
        PagedGenerator(model, requests=2, max_length=32)


def test_token_ids_are_whole_numbers():
    for tokens in ([1, 2], torch.tensor([1, 2], dtype=torch.int32), torch.tensor([[1], [2]]), (1, 2)):
        assert _token_ids("Prompts", tokens).tolist() == [1, 2]
    assert _token_ids("eos_token_id", 7).tolist() == _token_ids("eos_token_id", torch.tensor(7)).tolist() == [7]
    assert _token_ids("Prompts", []).tolist() == []
    for tokens in ([1.7, 2.2], torch.tensor([3.0]), [True, False], 2.5, True):
        with pytest.raises(TypeError, match="whole numbers"):
            _token_ids("Prompts", tokens)
