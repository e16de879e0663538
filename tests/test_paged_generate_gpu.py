"""Generation over the paged cache: the operators together, as a user has them."""

import copy

import pytest
import torch
from transformers import AutoModelForCausalLM, LlamaConfig, Qwen2Config

from neuralzip_b200.gpu.generate import PagedGenerator
from neuralzip_b200.gpu.inference import NeuralZipRuntime, export_model_for_gpu
from neuralzip_b200.setup import NeuralZipSetup

pytestmark = pytest.mark.gpu
DEVICE = "cuda:0"


def _model(kind="llama", dtype=torch.float32, **more):
    common = dict(hidden_size=256, num_hidden_layers=3, num_attention_heads=4, num_key_value_heads=2,
                  intermediate_size=512, vocab_size=512, max_position_embeddings=4096, **more)
    config = LlamaConfig(**common) if kind == "llama" else Qwen2Config(**common)
    config._attn_implementation = "eager"
    torch.manual_seed(0)
    with torch.device(DEVICE):
        return AutoModelForCausalLM.from_config(config, dtype=dtype).eval()


def _prompts(lengths, seed=1):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(512, (n,), generator=g) for n in lengths]


def _expected(model, prompts, new):
    out = []
    for p in prompts:
        ids = p[None].to(DEVICE)
        with torch.no_grad():
            out.append(model.generate(ids, attention_mask=torch.ones_like(ids), max_new_tokens=new, min_new_tokens=new,
                                      do_sample=False, pad_token_id=0)[0, len(p):].cpu())
    return out


@pytest.mark.parametrize("kind,more", [("llama", {}), ("qwen2", {}),
                                       ("qwen2", dict(use_sliding_window=True, sliding_window=24, max_window_layers=1)),
                                       ("llama", dict(rope_parameters=dict(rope_type="linear", factor=2.0,
                                                                           rope_theta=10000.0)))])
@pytest.mark.parametrize("cuda_graph", [False, True])
def test_generates_transformers_greedy_tokens(kind, more, cuda_graph):
    """In fp32, prompts of ragged lengths give the tokens that Transformers gives each alone."""
    model = _model(kind, **more)
    prompts = _prompts([1, 17, 40, 16])
    want = _expected(model, prompts, 33)
    generator = PagedGenerator(model, requests=6, max_length=96, page_size=16, cuda_graph=cuda_graph)
    for _ in range(2):  # the second call replays the first one's capture over released pages
        got = generator.generate(prompts, max_new_tokens=33)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    # Fewer, other prompts through the same capture.
    other = _prompts([30, 3], seed=5)
    assert all(torch.equal(a, b) for a, b in zip(generator.generate(other, max_new_tokens=20), _expected(model, other, 20)))
    assert int(generator.cache.used) == 0
    # The model itself is as it was.
    assert all(torch.equal(a, b) for a, b in zip(_expected(model, prompts, 33), want))


def test_end_tokens():
    model = _model()
    prompts = _prompts([5, 9, 30])
    full = PagedGenerator(model, requests=3, max_length=80).generate(prompts, max_new_tokens=40)
    eos = [int(full[0][7]), int(full[2][20])]
    got = PagedGenerator(model, requests=3, max_length=80).generate(prompts, max_new_tokens=40, eos_token_id=eos)
    for a, b in zip(got, full):
        ends = [i for i, t in enumerate(b.tolist()) if t in eos]
        assert torch.equal(a, b[:ends[0] + 1] if ends else b)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_compressed_model_gives_the_same_tokens(dtype):
    model = _model(dtype=dtype)
    uncompressed = copy.deepcopy(model)
    runtime = NeuralZipRuntime.attach(model, export_model_for_gpu(model, NeuralZipSetup().build(model)), device=DEVICE,
                                      blocks_per_launch=1)
    prompts = _prompts([12, 50, 1, 33, 8])
    want = PagedGenerator(uncompressed, requests=5, max_length=128, page_size=32).generate(prompts, max_new_tokens=60)
    generator = PagedGenerator(model, requests=5, max_length=128, page_size=32)
    generator.start(prompts, max_new_tokens=60)
    for workspace in runtime.workspaces.values():
        workspace.view(torch.uint8).fill_(0xA5)
    got = generator.generate(prompts, max_new_tokens=60)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    runtime.check_status()


def test_small_cache_is_shared():
    """The cache holds what the requests need together, not the longest times their number; more is refused."""
    model = _model()
    prompts = _prompts([100, 1, 1, 1])
    generator = PagedGenerator(model, requests=4, max_length=128, tokens=176, page_size=16)
    got = generator.generate(prompts, max_new_tokens=12)
    assert all(torch.equal(a, b) for a, b in zip(got, _expected(model, prompts, 12)))
    with pytest.raises(ValueError, match="pages"):
        generator.generate(_prompts([100, 60, 30, 1]), max_new_tokens=12)
    with pytest.raises(ValueError, match="max_length"):
        generator.generate(_prompts([120]), max_new_tokens=12)
    with pytest.raises(ValueError, match="1 to 4 prompts"):
        generator.generate(_prompts([1] * 5), max_new_tokens=2)
    with pytest.raises(ValueError, match="0 to 511"):
        generator.generate([[3, 512]], max_new_tokens=2)
    with pytest.raises(ValueError, match="at least one token"):
        generator.generate([[]], max_new_tokens=2)


@pytest.mark.parametrize("page_size", [4, 16, 64])
def test_default_cache_holds_all_requests_at_max_length(page_size):
    """max_length need not be whole pages: the last page of each request is its own."""
    model = _model()
    prompts = _prompts([10, 17, 3])
    generator = PagedGenerator(model, requests=3, max_length=17, page_size=page_size)
    for prompt_lengths in ((10, 10, 10), (17, 16, 3)):
        new = 18 - max(prompt_lengths)
        batch = [p[:n] if len(p) >= n else torch.cat([p] * 6)[:n] for p, n in zip(prompts, prompt_lengths)]
        got = generator.generate(batch, max_new_tokens=new)
        assert all(torch.equal(a, b) for a, b in zip(got, _expected(model, batch, new)))


def test_advances_no_further_than_max_new_tokens():
    """A step behind the last would write behind the tokens' buffer; it is refused on the host."""
    model = _model()
    generator = PagedGenerator(model, requests=2, max_length=20)
    with pytest.raises(RuntimeError, match="nothing to advance"):
        generator.advance()
    prompts = _prompts([17, 2])
    generator.start(prompts, max_new_tokens=4)
    for _ in range(3):
        generator.advance()
    with pytest.raises(RuntimeError, match="nothing to advance"):
        generator.advance()
    assert all(torch.equal(a.cpu(), b) for a, b in zip(generator._tokens[:, :4], _expected(model, prompts, 4)))
    generator.generate(prompts, max_new_tokens=4, eos_token_id=int(generator._tokens[0, 1]))
    with pytest.raises(RuntimeError, match="nothing to advance"):
        generator.advance()
    with pytest.raises(ValueError, match="power of two"):
        PagedGenerator(model, requests=2, max_length=20, page_size=0)


def test_query_and_key_norms():
    """Attention with a norm of each head of queries and keys goes through the norm of the rotary pass."""
    from transformers.models.llama.modeling_llama import LlamaRMSNorm, apply_rotary_pos_emb

    model = _model()
    for layer in model.model.layers:
        for name in ("q_norm", "k_norm"):
            norm = LlamaRMSNorm(64, eps=1e-5).to(DEVICE)
            with torch.no_grad():
                norm.weight.copy_(1 + 0.3 * torch.randn(64, generator=torch.Generator().manual_seed(len(name))))
            setattr(layer.self_attn, name, norm)
    prompts = _prompts([7, 21])
    got = PagedGenerator(model, requests=2, max_length=64).generate(prompts, max_new_tokens=16)

    def logits(ids):  # the whole sequence at once, no cache
        def forward(attention):
            def run(hidden_states, position_embeddings=None, **_kwargs):
                n = hidden_states.shape[1]
                q, k, v = (p(hidden_states).view(1, n, -1, 64).transpose(1, 2)
                           for p in (attention.q_proj, attention.k_proj, attention.v_proj))
                q, k = apply_rotary_pos_emb(attention.q_norm(q), attention.k_norm(k), *position_embeddings)
                out = torch.nn.functional.scaled_dot_product_attention(q, k, v, is_causal=True, enable_gqa=True)
                return attention.o_proj(out.transpose(1, 2).reshape(1, n, -1)), None
            return run

        for layer in model.model.layers:
            layer.self_attn.forward = forward(layer.self_attn)
        with torch.no_grad():
            out = model(input_ids=ids[None].to(DEVICE), use_cache=False).logits[0]
        for layer in model.model.layers:
            del layer.self_attn.forward
        return out

    for prompt, new in zip(prompts, got):
        ids = torch.cat([prompt, new])
        assert torch.equal(logits(ids)[len(prompt) - 1:-1].argmax(-1).cpu(), new)


@pytest.mark.parametrize("wrong", [dict(prompts=[[1.7, 2.2]]), dict(prompts=[[3], torch.tensor([3.5])]),
                                   dict(prompts=[[True, False]]), dict(prompts=[[3]], eos_token_id=2.5)])
def test_refuses_tokens_that_are_no_whole_numbers(wrong):
    """They are not rounded to tokens that nobody asked for."""
    generator = PagedGenerator(_model(), requests=2, max_length=20)
    with pytest.raises(TypeError, match="whole numbers"):
        generator.generate(**{"max_new_tokens": 2, **wrong})
    assert len(generator.generate([[3], torch.tensor([4], dtype=torch.int32)], max_new_tokens=2, eos_token_id=torch.tensor(511))) == 2


@pytest.mark.parametrize("kind,more", [
    ("llama", {}), ("qwen2", {}), ("qwen2", dict(use_sliding_window=True, sliding_window=24, max_window_layers=1)),
    ("llama", dict(rope_parameters=dict(rope_type="linear", factor=2.0, rope_theta=10000.0))),
    ("llama", dict(rope_parameters=dict(rope_type="llama3", factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0,
                                        original_max_position_embeddings=64, rope_theta=5e5))),
    ("qwen2", dict(rope_parameters=dict(rope_type="yarn", factor=64.0, original_max_position_embeddings=64,
                                        rope_theta=10000.0)))])
@pytest.mark.parametrize("cuda_graph", [False, True])
def test_tokens_that_hang_on_the_attention(kind, more, cuda_graph):
    """With weights of this size hardly two tokens in a row are alike, and each hangs on all that is cached: a cache
    that loses its oldest page gives others."""
    model = _model(kind, initializer_range=0.3, **more)
    prompts = _prompts([1, 17, 40, 16, 150])
    want = _expected(model, prompts, 33)
    assert all(len(set(w.tolist())) > 20 for w in want)
    generator = PagedGenerator(model, requests=6, max_length=200, page_size=16, cuda_graph=cuda_graph)
    assert all(torch.equal(a, b) for a, b in zip(generator.generate(prompts, max_new_tokens=33), want, strict=True))
    assert all(torch.equal(a, b) for a, b in zip(generator.generate(prompts[::-1], max_new_tokens=33), want[::-1], strict=True))
    if "use_sliding_window" not in more:
        generator.start(prompts[4:], max_new_tokens=33)
        for layer in generator.cache.keys:
            layer[generator.cache.block_table[0, 0]] = 0
        for _ in range(32):
            generator.advance()
        assert not torch.equal(generator._tokens[0, :33].cpu(), want[4])
