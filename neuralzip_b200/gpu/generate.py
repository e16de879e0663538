"""Greedy generation over a paged key-value cache.

The reference leaves generation to Transformers' ``generate``, whose cache
pads every request to the longest one. ``PagedGenerator`` runs the same
model (compressed by NeuralZipRuntime or not, sliced for tensor parallelism
or not) for a batch of prompts of any lengths, keeping keys and values in
the pages of neuralzip_b200.gpu.paged, so that the HBM which compressed
weights free holds as many cached tokens as fit, whichever request they
belong to.

Prompts run packed, without padding, through the model once. After that
every step is one token a request: pages reserved, queries and keys rotated
and stored, attention over the pages, the next tokens picked, all on the
GPU; the step is captured in a CUDA graph on first use and replayed, with
the decode launches of a compressed model in it.

Decoder layers as in neuralzip_b200.gpu.tp (self_attn.{q,k,v,o}_proj, with
or without q_norm and k_norm) with rotary positions whose frequencies do
not depend on the length; anything else is refused.
"""

from __future__ import annotations

import contextlib
import sys

import torch
from torch.nn import functional as F

from neuralzip_b200.gpu import paged
from neuralzip_b200.gpu.tp import decoder_layers

# Model types whose attention is known to be nothing but what _Layer reads from
# it. Others can have all the same modules and differ all the same: layers
# without rotary positions, queries scaled by position, states beside the cache.
_MODEL_TYPES = ("llama", "qwen2")
_STATIC_ROPE = ("default", "linear", "llama3", "yarn")
_PROJECTIONS = ("q_proj", "k_proj", "v_proj", "o_proj")
_NORMS = ("q_norm", "k_norm")
_EOS_IDS = 8
_LOOK_EVERY = 16  # steps between looks (from the host) at whether all requests have ended


class PagedCache:
    """Keys and values of `requests` requests at a time, in `pages` pages of
    `page_size` tokens shared by all of them, for each of `layers` layers;
    with the block table, the lengths and the free pages, on the GPU."""

    def __init__(self, layers, kv_heads, head_dim, *, requests, pages, page_size, max_length, dtype, device):
        if not 0 < requests <= paged.MAX_REQUESTS:
            raise ValueError(f"requests must be 1 to {paged.MAX_REQUESTS}, not {requests}.")
        if pages < 1 or max_length < 1:
            raise ValueError("pages and max_length must be at least 1.")
        paged._page_shift(page_size)
        self.page_size = page_size
        self.max_length = max_length
        shape = (pages, page_size, kv_heads, head_dim)
        self.keys = [torch.empty(shape, dtype=dtype, device=device) for _ in range(layers)]
        self.values = [torch.empty(shape, dtype=dtype, device=device) for _ in range(layers)]
        width = -(-max_length // page_size)
        self.block_table = torch.full((requests, width), -1, dtype=torch.int32, device=device)
        self.lengths = torch.zeros(requests, dtype=torch.int32, device=device)
        self.free_pages = torch.arange(pages, dtype=torch.int32, device=device)
        self.used = torch.zeros(1, dtype=torch.int32, device=device)

    @property
    def requests(self):
        return self.lengths.shape[0]

    @property
    def pages(self):
        return self.free_pages.shape[0]

    def pages_for(self, tokens):
        return -(-tokens // self.page_size)

    def reserve(self, new_tokens, *, rows, row_stride=0):
        """Room for new tokens, lengths updated in place (paged.reserve_pages)."""
        return paged.reserve_pages(self.lengths, new_tokens, self.block_table, self.free_pages, self.used,
                                   page_size=self.page_size, rows=rows, row_stride=row_stride,
                                   lengths_out=self.lengths, used_out=self.used)

    def release(self, done):
        """Ends the requests that the bool tensor `done` marks (paged.release_pages)."""
        paged.release_pages(self.lengths, done, self.block_table, self.free_pages, self.used,
                            page_size=self.page_size, lengths_out=self.lengths, used_out=self.used)


def _rotates_neighbours(attention):
    """Whether the attention's rotary pairs are neighbours (2i, 2i + 1), not
    halves (i, i + half): asked of its module's own rotate_half."""
    rotate_half = getattr(sys.modules.get(type(attention).__module__), "rotate_half", None)
    if rotate_half is None:
        raise ValueError(f"{type(attention).__name__} rotates positions in an unknown way.")
    turned = rotate_half(torch.arange(1.0, 5.0).view(1, 1, 1, 4)).flatten().tolist()
    if turned == [-3.0, -4.0, 1.0, 2.0]:
        return False
    if turned == [-2.0, 1.0, -4.0, 3.0]:
        return True
    raise ValueError(f"{type(attention).__name__} rotates positions in an unknown way.")


def _token_ids(name, tokens):
    """Token ids as a 1-D tensor; anything but whole numbers is refused, not rounded."""
    ids = torch.as_tensor(tokens)
    if ids.numel() and (ids.is_floating_point() or ids.is_complex() or ids.dtype is torch.bool):
        raise TypeError(f"{name} must be whole numbers, not {ids.dtype}.")
    return ids.reshape(-1).long()


class _Layer:
    """What the paged attention needs to know of one attention module."""

    def __init__(self, attention, config):
        children = dict(attention.named_children())
        strange = set(children) - {*_PROJECTIONS, *_NORMS}
        missing = set(_PROJECTIONS) - set(children)
        if strange or missing or list(attention.parameters(recurse=False)):
            raise ValueError(f"{type(attention).__name__} is not an attention of {', '.join(_PROJECTIONS)}"
                             f" (with or without {', '.join(_NORMS)}).")
        if not getattr(attention, "use_rope", True) or not getattr(attention, "is_causal", True):
            raise ValueError("Layers without rotary positions or causal attention are not supported.")
        self.attention = attention
        self.dim = int(attention.head_dim)
        self.heads = attention.q_proj.out_features // self.dim
        self.kv_heads = attention.k_proj.out_features // self.dim
        self.scale = float(attention.scaling)
        window = getattr(attention, "sliding_window", None)
        if getattr(config, "sliding_window", None) and not hasattr(attention, "sliding_window"):
            raise ValueError("The config has a sliding window, the attention does not say which layers it is for.")
        self.window = None if window is None else int(window)
        self.norms, self.eps = [None, None], None
        for i, name in enumerate(_NORMS):
            norm = children.get(name)
            if norm is None:
                continue
            weight, eps = getattr(norm, "weight", None), getattr(norm, "variance_epsilon", None)
            if eps is None or weight is None or tuple(weight.shape) != (self.dim,) or len(list(norm.parameters())) != 1:
                raise ValueError(f"{name} is not a root-mean-square norm of each head.")
            if self.eps not in (None, float(eps)):  # the rotary pass takes one for both
                raise ValueError(f"{' and '.join(_NORMS)} must have the same epsilon, not {self.eps} and {float(eps)}.")
            self.norms[i], self.eps = weight.detach(), float(eps)
        self.eps = 1e-6 if self.eps is None else self.eps


class PagedGenerator:
    """Greedy generation of up to `requests` prompts at a time with `model`
    (a causal language model on a CUDA device).

    The cache has room for `tokens` tokens in all (in whole pages; default:
    what `requests` requests of `max_length` need), any of which any request
    can use, up to `max_length` (prompt and new tokens) a request. `cuda_graph=False` runs each step's
    launches one by one (needed where a step cannot be captured: some
    collectives, experts picked on the host).

    Model types but llama and qwen2 are refused without `other_types=True`:
    what is checked then is that the attention has the modules, windows and
    rotary positions described above; that it does nothing besides (no layer
    without positions, no scaling by position, no state of its own, no
    clipping) is for the caller to know.

    The model's own modules are left as they are: its attention is replaced
    only while the generator runs it. One call at a time."""

    def __init__(self, model, *, requests, max_length, tokens=None, page_size=16, cuda_graph=True,
                 other_types=False):
        config = model.config
        base = getattr(model, "model", None)
        rotary = getattr(base, "rotary_emb", None)
        if rotary is None or not hasattr(rotary, "inv_freq"):
            raise ValueError("The model has no rotary embedding (expected model.model.rotary_emb).")
        if getattr(rotary, "rope_type", "default") not in _STATIC_ROPE:
            raise ValueError(f"Rotary positions of type {rotary.rope_type!r} change with the length and are not supported.")
        if getattr(config, "attn_logit_softcapping", None):
            raise ValueError("Attention with capped scores is not supported.")
        kind = getattr(config, "model_type", None)
        if kind not in _MODEL_TYPES and not other_types:
            raise ValueError(f"Models of type {kind!r} are supported only with other_types=True (see there).")
        self.model = model
        self._rotary = rotary
        self._layers = [_Layer(layer.self_attn, config) for layer in decoder_layers(model)]
        first = self._layers[0]
        if any((l.heads, l.kv_heads, l.dim) != (first.heads, first.kv_heads, first.dim) for l in self._layers):
            raise ValueError("All layers must have the same heads.")
        if first.dim % 8 or first.dim > paged.MAX_HEAD_WIDTH:
            raise ValueError(f"The head width must be a multiple of 8 up to {paged.MAX_HEAD_WIDTH}, not {first.dim}.")
        self._interleaved = _rotates_neighbours(first.attention)
        weight = model.get_input_embeddings().weight
        self.device, self.dtype = weight.device, weight.dtype
        if self.device.type != "cuda":
            raise ValueError(f"The model must be on a CUDA device, not on {self.device}.")
        paged._page_shift(page_size)
        if tokens is None:  # every request ends inside a page of its own
            tokens = requests * -(-max_length // page_size) * page_size
        self.cache = PagedCache(len(self._layers), first.kv_heads, first.dim, requests=requests,
                                pages=-(-tokens // page_size), page_size=page_size, max_length=max_length,
                                dtype=self.dtype, device=self.device)
        self._table = paged.rotary_table(rotary.inv_freq.to(self.device), max_length,
                                         float(getattr(rotary, "attention_scaling", 1.0)))
        # The step's inputs and outputs, at fixed addresses so that a captured step can be replayed.
        self._ids = torch.zeros((requests, 1), dtype=torch.long, device=self.device)
        self._new = torch.zeros(requests, dtype=torch.int32, device=self.device)
        self._eos = torch.full((_EOS_IDS,), -1, dtype=torch.long, device=self.device)
        self._count = torch.zeros(1, dtype=torch.long, device=self.device)
        self._tokens = torch.zeros((requests, max_length), dtype=torch.long, device=self.device)
        self._refused = torch.zeros(1, dtype=torch.int32, device=self.device)
        # A 4-D mask is passed through as it is; the replaced attention looks at none.
        self._mask = torch.zeros((1, 1, 1, 1), dtype=self.dtype, device=self.device)
        self._cuda_graph = bool(cuda_graph)
        self._graph = None
        self._left = 0  # steps that the requests taken up still have room for

    # ---- the model with paged attention ----------------------------------------------------

    @contextlib.contextmanager
    def _replaced(self, attend):
        """The model with its attention over the cache: `attend(layer index,
        layer, query, key, value)` on the rows of a call, flattened."""
        def forward_of(index, layer):
            attention = layer.attention

            def forward(hidden_states, *_args, **_kwargs):
                rows = hidden_states.shape[0] * hidden_states.shape[1]
                query = attention.q_proj(hidden_states).view(rows, layer.heads, layer.dim)
                key = attention.k_proj(hidden_states).view(rows, layer.kv_heads, layer.dim)
                value = attention.v_proj(hidden_states).view(rows, layer.kv_heads, layer.dim)
                out = attend(index, layer, query, key, value)
                return attention.o_proj(out.reshape(*hidden_states.shape[:2], -1)), None

            return forward

        modules = [layer.attention for layer in self._layers] + [self._rotary]
        if any("forward" in module.__dict__ for module in modules):
            raise RuntimeError("The model's attention is replaced already.")
        try:
            for index, layer in enumerate(self._layers):
                layer.attention.forward = forward_of(index, layer)
            self._rotary.forward = lambda *_args, **_kwargs: (None, None)  # the attention rotates by its own table
            yield
        finally:
            for module in modules:
                module.__dict__.pop("forward", None)

    def _store(self, reserved, index, layer, query, key, value, key_out=None):
        cache = self.cache
        return paged.rotary_store(query, key, value, reserved.positions, reserved.slots, self._table, cache.keys[index],
                                  cache.values[index], interleaved=self._interleaved, query_norm=layer.norms[0],
                                  key_norm=layer.norms[1], eps=layer.eps, query_out=query, key_out=key_out)

    def _prefill(self, ids, lengths):
        """Runs the prompts, packed one behind the other in `ids`; returns each one's first new token."""
        new = torch.zeros(self.cache.requests, dtype=torch.int32)
        new[:len(lengths)] = torch.tensor(lengths, dtype=torch.int32)
        rows = sum(lengths)
        reserved = self.cache.reserve(new.to(self.device), rows=rows)
        self._refused.copy_(reserved.refused)

        def attend(index, layer, query, key, value):
            turned = torch.empty_like(key)
            query = self._store(reserved, index, layer, query, key, value, turned)
            out = torch.empty_like(query)
            first = 0
            for length in lengths:  # each prompt attends to itself
                at = slice(first, first + length)
                q, k, v = (x[at].transpose(0, 1)[None] for x in (query, turned, value))
                mask = None
                if layer.window is not None and length > layer.window:
                    place = torch.arange(length, device=self.device)
                    mask = (place <= place[:, None]) & (place > place[:, None] - layer.window)
                out[at] = F.scaled_dot_product_attention(q, k, v, attn_mask=mask, is_causal=mask is None,
                                                         scale=layer.scale, enable_gqa=True)[0].transpose(0, 1)
                first += length
            return out

        last = torch.tensor(lengths, device=self.device).cumsum(0) - 1
        with self._replaced(attend):
            logits = self.model(input_ids=ids[None], position_ids=reserved.positions[None].long(), attention_mask=self._mask,
                                use_cache=False, logits_to_keep=last).logits
        return logits[0].argmax(-1)

    def _take(self, tokens):
        """Notes the new tokens: a request that has ended takes no more."""
        self._tokens.index_copy_(1, self._count, tokens[:, None])
        self._count.add_(1)
        self._ids.copy_(tokens[:, None])
        ended = (tokens[:, None] == self._eos).any(1)
        self._new.masked_fill_(ended, 0)

    def _step(self):
        """One token for each request that goes on."""
        cache = self.cache
        reserved = cache.reserve(self._new, rows=cache.requests, row_stride=1)
        self._refused.add_(reserved.refused)

        def attend(index, layer, query, key, value):
            query = self._store(reserved, index, layer, query, key, value)
            return paged.paged_attention(query, cache.keys[index], cache.values[index], cache.block_table,
                                         cache.lengths, scale=layer.scale, window=layer.window)

        with self._replaced(attend):
            logits = self.model(input_ids=self._ids, position_ids=reserved.positions[:, None].long(),
                                attention_mask=self._mask, use_cache=False, logits_to_keep=1).logits
        self._take(logits[:, -1].argmax(-1))

    def _capture(self):
        """Captures the step, after a warm-up whose effects are undone (it
        takes pages that the replays then take again)."""
        state = (self.cache.lengths, self.cache.used, self._ids, self._new, self._count, self._refused)
        before = [t.clone() for t in state]
        current = torch.cuda.current_stream(self.device)
        side = torch.cuda.Stream(device=self.device)
        side.wait_stream(current)
        with torch.cuda.stream(side):
            self._step()
        current.wait_stream(side)
        for tensor, value in zip(state, before):
            tensor.copy_(value)
        torch.cuda.synchronize(self.device)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            self._step()
        self._graph = graph

    # ---- generation ---------------------------------------------------------------------------

    def start(self, prompts, *, max_new_tokens, eos_token_id=None):
        """Takes up the prompts and their first new tokens; `advance` then
        gives one more a call."""
        with torch.cuda.device(self.device), torch.no_grad():
            self._start(prompts, max_new_tokens, eos_token_id)

    def _start(self, prompts, max_new_tokens, eos_token_id):
        cache = self.cache
        prompts = [_token_ids("Prompts", p) for p in prompts]
        if not 0 < len(prompts) <= cache.requests:
            raise ValueError(f"There must be 1 to {cache.requests} prompts, not {len(prompts)}.")
        if not all(len(p) for p in prompts):
            raise ValueError("A prompt must have at least one token.")
        ids, vocabulary = torch.cat([p.to(self.device) for p in prompts]), self.model.get_input_embeddings().weight.shape[0]
        if not 0 <= int(ids.min()) <= int(ids.max()) < vocabulary:
            raise ValueError(f"Token ids must be 0 to {vocabulary - 1}.")
        if max_new_tokens < 1:
            raise ValueError("max_new_tokens must be at least 1.")
        longest = max(len(p) for p in prompts) + max_new_tokens - 1  # the last token is not cached
        if longest > cache.max_length:
            raise ValueError(f"The longest request needs {longest} cached tokens; max_length is {cache.max_length}.")
        need = sum(cache.pages_for(len(p) + max_new_tokens - 1) for p in prompts)
        if need > cache.pages:
            raise ValueError(f"The requests need {need} pages of {cache.page_size} tokens; the cache has {cache.pages}.")
        eos = [] if eos_token_id is None else _token_ids("eos_token_id", eos_token_id).tolist()
        if len(eos) > _EOS_IDS:
            raise ValueError(f"At most {_EOS_IDS} end tokens.")
        self._left = 0
        cache.release(torch.ones(cache.requests, dtype=torch.bool, device=self.device))
        self._eos.copy_(torch.tensor(eos + [-1] * (_EOS_IDS - len(eos))))
        self._new.zero_()
        self._new[:len(prompts)] = 1
        self._count.zero_()
        tokens = torch.zeros(cache.requests, dtype=torch.long, device=self.device)
        tokens[:len(prompts)] = self._prefill(ids, [len(p) for p in prompts])
        self._take(tokens)
        if self._cuda_graph and self._graph is None and max_new_tokens > 1:
            self._capture()
        self._left = max_new_tokens - 1

    def advance(self):
        """One more token for each request that has not ended, up to the
        `max_new_tokens` that it was taken up with."""
        if self._left < 1:
            raise RuntimeError("There is nothing to advance: start() takes up prompts, with max_new_tokens of room.")
        self._left -= 1
        with torch.no_grad(), torch.cuda.device(self.device):
            if self._graph is not None:
                self._graph.replay()
            else:
                self._step()

    def generate(self, prompts, *, max_new_tokens, eos_token_id=None):
        """The new tokens of each prompt (a sequence of token ids or a 1-D
        tensor), as a list of CPU tensors: `max_new_tokens` of them, or up to
        and with the first of `eos_token_id`."""
        prompts = list(prompts)
        with torch.cuda.device(self.device):
            self.start(prompts, max_new_tokens=max_new_tokens, eos_token_id=eos_token_id)
            for step in range(1, max_new_tokens):
                if eos_token_id is not None and step % _LOOK_EVERY == 0 and not bool(self._new.any()):
                    break
                self.advance()
            count = int(self._count)
            tokens = self._tokens[:len(prompts), :count].cpu()
            refused = int(self._refused)
            self._left = 0
            self.cache.release(torch.ones(self.cache.requests, dtype=torch.bool, device=self.device))
        if refused:
            raise RuntimeError("The cache ran out of pages.")
        eos = self._eos.cpu()
        out = []
        for row in tokens:
            ends = (row[:, None] == eos).any(1).nonzero()
            out.append(row[:int(ends[0]) + 1] if len(ends) else row)
        return out

    def close(self):
        """Frees the captured step (before a process group it uses is destroyed, say)."""
        self._graph = None
