"""Cases of the paged-generation operators: page reservation and release, rotary positions with the cache write, and
attention of one new token over the paged cache.

`run` computes each in elementary torch operations, or, where `own` is true, through neuralzip_b200.gpu.paged."""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
DEVICE = "cuda"


def listed():
    return [
        # Batch-1 generation with the 14/2-head, 64-wide attention of the Qwen2.5-0.5B benchmark: prompt 32 and 128 new
        # tokens. The smallest call: latency counts.
        attention("attend_b1_short", batch=1, heads=14, kv_heads=2, dim=64, shortest=160, longest=160, page=16),
        # Batch-8 generation of the Llama-3-8B benchmark (prompt 128, 256 new tokens), the requests at ragged lengths.
        attention("attend_b8_ragged", batch=8, heads=32, kv_heads=8, dim=128, shortest=129, longest=384, page=16,
                  dtype="fp16", lse=True),
        # One long document at the Llama-3-70B heads: few rows, the work has to be split over the length.
        attention("attend_b1_long", batch=1, heads=64, kv_heads=8, dim=128, shortest=65537, longest=65537, page=64),
        # A small fp32 model without shared heads, an odd head width and a sliding window; one request is empty.
        attention("attend_fp32_window", batch=5, heads=12, kv_heads=12, dim=80, shortest=0, longest=4093, page=32,
                  dtype="fp32", window=1000, lse=True),
        # Serving: many requests of very different lengths in a cache of gigabytes.
        attention("attend_b32_large", batch=32, heads=32, kv_heads=8, dim=128, shortest=2047, longest=32768, page=32),
        # One token for each of 8 requests: the call before every attention of a generation step.
        rotary("rotary_step", tokens=8, heads=32, kv_heads=8, dim=128, rot=128, norm=False),
        # Prompts of about 8k tokens at the Llama-3-70B heads, with query and key norms, padded rows behind them.
        rotary("rotary_prompts", tokens=8191, heads=64, kv_heads=8, dim=128, rot=128, norm=True, pad=57),
        # A partial, interleaved rotation of an 80-wide head in fp32.
        rotary("rotary_partial", tokens=777, heads=20, kv_heads=5, dim=80, rot=32, norm=False, interleaved=True,
               dtype="fp32"),
        # The step's bookkeeping: one more token for each of 64 requests, some of which start a page.
        reserve("reserve_step", batch=64, shortest=1, longest=1, cached=4096, page=16, stride=1),
        # Admission of prompts: block tables, positions and slots of 64k tokens.
        reserve("reserve_prompts", batch=129, shortest=1, longest=1024, cached=0, page=16, stride=0),
        # The end of some requests of a small and of a large batch.
        release("release_b8", batch=8, cached=384, page=16),
        release("release_b512", batch=512, cached=8190, page=16),
    ]


def attention(name, *, batch, heads, kv_heads, dim, shortest, longest, page, dtype="bf16", window=0, lse=False):
    return {"name": name, "op": "attention", "batch": batch, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "shortest": shortest, "longest": longest, "page": page, "dtype": dtype, "window": window, "lse": lse}


def rotary(name, *, tokens, heads, kv_heads, dim, rot, norm, pad=0, interleaved=False, dtype="bf16"):
    return {"name": name, "op": "rotary", "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim, "rot": rot,
            "norm": norm, "pad": pad, "interleaved": interleaved, "dtype": dtype, "page": 16}


def reserve(name, *, batch, shortest, longest, cached, page, stride):
    return {"name": name, "op": "reserve", "batch": batch, "shortest": shortest, "longest": longest, "cached": cached,
            "page": page, "stride": stride}


def release(name, *, batch, cached, page):
    return {"name": name, "op": "release", "batch": batch, "cached": cached, "page": page}


def _between(rng, low, high):
    """An integer in [low, high], spread over its logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49))))))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "rotary", "rotary", "reserve", "release"])
    page = rng.choice([8, 16, 32, 64, 128])
    if op == "attention":
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        kv_heads = rng.choice([1, 2, 4, 5, 8])
        heads = kv_heads * rng.choice([1, 2, 3, 4, 7, 8, 12, 16])
        dim = rng.choice([32, 64, 64, 80, 96, 128, 128, 128, 192, 256])
        longest = _between(rng, 1, 65536)
        most = int(2 ** 31 / (2 * kv_heads * dim * BYTES[dtype] * longest))
        batch = _between(rng, 1, max(1, min(256, most)))
        case = attention("", batch=batch, heads=heads, kv_heads=kv_heads, dim=dim,
                         shortest=rng.randint(0, longest), longest=longest, page=page, dtype=dtype,
                         window=rng.choice([0, 0, 0, _between(rng, 1, longest)]), lse=rng.random() < 0.5)
    elif op == "rotary":
        dim = rng.choice([32, 64, 80, 96, 128, 128, 192, 256])
        kv_heads = rng.choice([1, 2, 3, 4, 8])
        case = rotary("", tokens=_between(rng, 1, 8192), heads=kv_heads * rng.choice([1, 3, 4, 7, 8]),
                      kv_heads=kv_heads, dim=dim, rot=rng.choice([dim, dim, dim // 2, 16]),
                      norm=rng.random() < 0.5, pad=rng.choice([0, rng.randint(1, 64)]),
                      interleaved=rng.random() < 0.3, dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]))
    elif op == "reserve":
        batch = _between(rng, 1, 1024)
        if rng.random() < 0.5:
            case = reserve("", batch=batch, shortest=0, longest=1, cached=_between(rng, 1, 8192), page=page, stride=1)
        else:
            longest = _between(rng, 1, max(1, 131072 // batch))
            case = reserve("", batch=batch, shortest=rng.randint(0, longest), longest=longest,
                           cached=rng.choice([0, _between(rng, 1, 2048)]), page=page,
                           stride=rng.choice([0, 0, longest + rng.randint(0, 5)]))
    else:
        case = release("", batch=_between(rng, 1, 1024), cached=_between(rng, 1, 8192), page=page)
    del case["name"]
    return case


def _spread(low, high, count):
    """`count` whole numbers from `low` to `high`, `high` among them."""
    if count == 1:
        return [high]
    return [low + (high - low) * i // (count - 1) for i in range(count)]


def _ceil(a, b):
    return -(-a // b)


def _generator(seed):
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _shuffled(values, gen):
    values = torch.tensor(values, dtype=torch.int32, device=DEVICE)
    return values[torch.randperm(len(values), generator=gen, device=DEVICE)]


def _order(n, gen):
    return torch.randperm(n, generator=gen, device=DEVICE).to(torch.int32)


def prepare(case, seed):
    gen = _generator(seed)
    return {"attention": _prepare_attention, "rotary": _prepare_rotary, "reserve": _prepare_reserve,
            "release": _prepare_release}[case["op"]](case, gen)


def _prepare_attention(case, gen):
    dtype, page, batch = DTYPES[case["dtype"]], case["page"], case["batch"]
    lengths = _shuffled(_spread(case["shortest"], case["longest"], batch), gen)
    width = max(1, _ceil(case["longest"], page))
    held = (lengths.long() + page - 1) // page
    pages = sum(_ceil(n, page) for n in _spread(case["shortest"], case["longest"], batch)) + 3
    order = _order(pages, gen)
    # Every request's pages lie anywhere in the pool; entries behind its last page are -1.
    first = held.cumsum(0) - held
    column = torch.arange(width, device=DEVICE)
    table = torch.where(column < held[:, None], order[(first[:, None] + column).clamp(max=pages - 1)].long(), -1)
    shape = (pages, page, case["kv_heads"], case["dim"])
    return {"case": case, "lengths": lengths, "table": table.to(torch.int32),
            "query": (2 * torch.randn((batch, case["heads"], case["dim"]), generator=gen, device=DEVICE)).to(dtype),
            "keys": torch.randn(shape, generator=gen, device=DEVICE, dtype=dtype),
            "values": torch.randn(shape, generator=gen, device=DEVICE, dtype=dtype)}


def _prepare_rotary(case, gen):
    dtype, page, tokens, dim = DTYPES[case["dtype"]], case["page"], case["tokens"], case["dim"]
    rows, furthest = tokens + case["pad"], 4096
    pages = _ceil(tokens, page) + 2
    heads, kv_heads = case["heads"], case["kv_heads"]
    # The projections' outputs side by side, as one product writes them: each of the three is a strided view.
    qkv = torch.randn((rows, heads + 2 * kv_heads, dim), generator=gen, device=DEVICE, dtype=dtype)
    slots = torch.full((rows,), -1, dtype=torch.int32, device=DEVICE)
    slots[:tokens] = _order(pages * page, gen)[:tokens]
    positions = torch.zeros(rows, dtype=torch.int32, device=DEVICE)
    positions[:tokens] = torch.randint(furthest, (tokens,), generator=gen, device=DEVICE, dtype=torch.int32)
    angles = torch.arange(furthest, device=DEVICE, dtype=torch.float64)[:, None] * 10000.0 ** (
        -torch.arange(case["rot"] // 2, device=DEVICE, dtype=torch.float64) * 2 / case["rot"])
    weights = [1 + 0.1 * torch.randn(dim, generator=gen, device=DEVICE) for _ in range(2)]
    shape = (pages, page, kv_heads, dim)
    return {"case": case, "query": qkv[:, :heads], "key": qkv[:, heads:heads + kv_heads],
            "value": qkv[:, heads + kv_heads:], "slots": slots, "positions": positions,
            "rotary": torch.cat([angles.cos(), angles.sin()], 1).float(),
            "query_norm": weights[0].to(dtype) if case["norm"] else None,
            "key_norm": weights[1].to(dtype) if case["norm"] else None,
            "keys": torch.randn(shape, generator=gen, device=DEVICE, dtype=dtype),
            "values": torch.randn(shape, generator=gen, device=DEVICE, dtype=dtype)}


def _held_table(lengths, order, page, width):
    """Block table of requests that hold the first pages of `order`, in request order."""
    held = (lengths.long() + page - 1) // page
    first = held.cumsum(0) - held
    column = torch.arange(width, device=DEVICE)
    at = (first[:, None] + column).clamp(max=order.numel() - 1)
    return torch.where(column < held[:, None], order[at].long(), -1).to(torch.int32)


def _reserve_sizes(case):
    new = _spread(case["shortest"], case["longest"], case["batch"])
    cached = _spread(0, case["cached"], case["batch"])
    width = _ceil(case["cached"] + case["longest"], case["page"]) + 1
    held = sum(_ceil(n, case["page"]) for n in cached)
    rows = case["batch"] * case["stride"] if case["stride"] else sum(new)
    pages = held + sum(_ceil(n, case["page"]) + 1 for n in new)
    return new, cached, width, held, max(1, rows), pages


def _prepare_reserve(case, gen):
    new, cached, width, held, rows, pages = _reserve_sizes(case)
    lengths = _shuffled(cached, gen)
    order = _order(pages, gen)
    return {"case": case, "lengths": lengths, "new": _shuffled(new, gen), "free": order, "rows": rows,
            "table": _held_table(lengths, order, case["page"], width),
            "used": torch.full((1,), held, dtype=torch.int32, device=DEVICE)}


def _prepare_release(case, gen):
    cached = _spread(1, case["cached"], case["batch"])
    held = sum(_ceil(n, case["page"]) for n in cached)
    lengths, order = _shuffled(cached, gen), _order(held + 5, gen)
    return {"case": case, "lengths": lengths, "free": order,
            "done": torch.rand(case["batch"], generator=gen, device=DEVICE) < 0.5,
            "table": _held_table(lengths, order, case["page"], _ceil(case["cached"], case["page"])),
            "used": torch.full((1,), held, dtype=torch.int32, device=DEVICE)}


def run(state):
    return {"attention": _run_attention, "rotary": _run_rotary, "reserve": _run_reserve,
            "release": _run_release}[state["case"]["op"]](state)


def _run_attention(s):
    c = s["case"]
    if own:
        from neuralzip_b200.gpu import paged

        out = paged.paged_attention(s["query"], s["keys"], s["values"], s["table"], s["lengths"],
                                    window=c["window"] or None, return_lse=c["lse"])
        return list(out) if c["lse"] else [out]
    batch, kv_heads, dim = c["batch"], c["kv_heads"], c["dim"]
    at = s["table"].clamp(min=0).long()
    keys = s["keys"][at].reshape(batch, -1, kv_heads, dim).float()
    values = s["values"][at].reshape(batch, -1, kv_heads, dim).float()
    query = s["query"].float().view(batch, kv_heads, -1, dim)
    scores = torch.einsum("bhgd,blhd->bhgl", query, keys) * dim ** -0.5
    place = torch.arange(keys.shape[1], device=keys.device)
    seen = place < s["lengths"][:, None]
    if c["window"]:
        seen = seen & (place >= s["lengths"][:, None] - c["window"])
    scores = torch.where(seen[:, None, None], scores, -math.inf)
    most = scores.amax(-1, keepdim=True)
    most = torch.where(most == -math.inf, 0.0, most)
    weights = torch.exp(scores - most)
    total = weights.sum(-1, keepdim=True)
    out = torch.einsum("bhgl,blhd->bhgd", weights, values) / torch.where(total == 0, 1.0, total)
    out = out.reshape(batch, -1, dim).to(s["query"].dtype)
    return [out, (most + torch.log(total)).reshape(batch, -1)] if c["lse"] else [out]


def _rotated(x, cos, sin, rot, interleaved):
    turned = x[..., :rot]
    if interleaved:
        a, b = turned[..., 0::2], turned[..., 1::2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = turned[..., :rot // 2], turned[..., rot // 2:]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([turned, x[..., rot:]], -1)


def _normed(x, weight, eps):
    if weight is None:
        return x
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * weight.float()


def _run_rotary(s):
    c = s["case"]
    if own:
        from neuralzip_b200.gpu import paged

        out = paged.rotary_store(s["query"], s["key"], s["value"], s["positions"], s["slots"], s["rotary"], s["keys"],
                                 s["values"], interleaved=c["interleaved"], query_norm=s["query_norm"],
                                 key_norm=s["key_norm"], eps=1e-6)
        return [out, s["keys"], s["values"]]
    rot, dtype = c["rot"], s["query"].dtype
    turn = s["rotary"][s["positions"].long()][:, None]
    cos, sin = turn[..., :rot // 2], turn[..., rot // 2:]
    query = _rotated(_normed(s["query"].float(), s["query_norm"], 1e-6), cos, sin, rot, c["interleaved"]).to(dtype)
    key = _rotated(_normed(s["key"].float(), s["key_norm"], 1e-6), cos, sin, rot, c["interleaved"]).to(dtype)
    slots, value = s["slots"].long(), s["value"]
    if c["pad"]:
        kept = slots >= 0
        slots, key, value = slots[kept], key[kept], value[kept]
    s["keys"].view(-1, c["kv_heads"], c["dim"])[slots] = key
    s["values"].view(-1, c["kv_heads"], c["dim"])[slots] = value
    return [query, s["keys"], s["values"]]


def _run_reserve(s):
    c = s["case"]
    page, stride, rows = c["page"], c["stride"], s["rows"]
    if own:
        from neuralzip_b200.gpu import paged

        r = paged.reserve_pages(s["lengths"], s["new"], s["table"], s["free"], s["used"], page_size=page, rows=rows,
                                row_stride=stride)
        return [r.positions, r.slots, r.row_offsets, r.lengths, r.used, r.refused, s["table"]]
    lengths, new, table = s["lengths"].long(), s["new"].long(), s["table"]
    width, free = table.shape[1], s["free"].numel()
    batch = torch.arange(len(new), device=new.device)
    ends = new.cumsum(0)
    starts = batch * stride if stride else ends - new
    fits = (lengths + new <= width * page) & ((new <= stride) if stride else (ends <= rows))
    held = (lengths + page - 1) // page
    need = torch.where(fits, (lengths + new + page - 1) // page - held, 0)
    upto = need.cumsum(0)
    served = fits & ((need == 0) | (s["used"] + upto <= free))
    need = torch.where(served, need, 0)
    column = torch.arange(width, device=new.device)
    taken = (column >= held[:, None]) & (column < (held + need)[:, None])
    source = s["used"].long() + upto[:, None] - need[:, None] + column - held[:, None]
    table.copy_(torch.where(taken, s["free"][source.clamp(0, free - 1)], table))
    row = torch.arange(rows, device=new.device)
    owner = row // stride if stride else torch.searchsorted(ends, row, right=True)
    live = owner < len(new)
    owner = owner.clamp(max=len(new) - 1)
    step = row - starts[owner]
    live = live & served[owner] & (step < new[owner])
    position = torch.where(live, lengths[owner] + step, 0)
    slot = table[owner, position // page].long() * page + position % page
    offsets = torch.cat([starts, starts[-1:] + (stride if stride else new[-1:])])
    return [position.int(), torch.where(live, slot, -1).int(), offsets.int(),
            torch.where(served, lengths + new, lengths).int(),
            (s["used"] + need.sum()).int(), (~served).sum().int().reshape(1), table]


def _run_release(s):
    c = s["case"]
    page = c["page"]
    if own:
        from neuralzip_b200.gpu import paged

        lengths, used = paged.release_pages(s["lengths"], s["done"], s["table"], s["free"], s["used"], page_size=page)
        return [lengths, used, s["free"]]
    lengths, table = s["lengths"].long(), s["table"]
    count = torch.where(s["done"], (lengths + page - 1) // page, 0)
    ends = count.cumsum(0)
    # The pages go back under the top of the stack, in request order, and each request's in table order.
    base = s["used"].long() - ends[-1]
    place = torch.arange(s["free"].numel(), device=table.device) - base
    back = (place >= 0) & (place < ends[-1])
    owner = torch.searchsorted(ends, place, right=True).clamp(max=len(ends) - 1)
    column = (place - ends[owner] + count[owner]).clamp(0, table.shape[1] - 1)
    s["free"].copy_(torch.where(back, table[owner, column], s["free"]))
    return [torch.where(s["done"], 0, s["lengths"]), base.int(), s["free"]]


def work(case):
    return {"attention": _work_attention, "rotary": _work_rotary, "reserve": _work_reserve,
            "release": _work_release}[case["op"]](case)


def _work_attention(c):
    lengths = _spread(c["shortest"], c["longest"], c["batch"])
    seen = sum(min(n, c["window"]) if c["window"] else n for n in lengths)
    size = BYTES[c["dtype"]]
    rows = c["batch"] * c["heads"]
    return {"bytes": 2 * seen * c["kv_heads"] * c["dim"] * size + 2 * rows * c["dim"] * size
            + 4 * rows * c["lse"] + 4 * c["batch"] + 4 * sum(_ceil(n, c["page"]) for n in lengths),
            "flops": 4 * seen * c["heads"] * c["dim"]}


def _work_rotary(c):
    size, rows = BYTES[c["dtype"]], c["tokens"] + c["pad"]
    values = rows * c["heads"] * c["dim"] + 2 * c["tokens"] * c["kv_heads"] * c["dim"]
    return {"bytes": 2 * values * size + 8 * rows + 4 * c["rot"] * min(rows, 4096),
            "flops": 3 * rows * (c["heads"] + c["kv_heads"]) * c["rot"]}


def _work_reserve(c):
    new, cached, _width, _held, rows, _pages = _reserve_sizes(c)
    taken = sum(new) // c["page"]
    return {"bytes": 16 * c["batch"] + 8 * rows + 8 * taken + 12, "flops": 0}


def _work_release(c):
    half = sum(_ceil(n, c["page"]) for n in _spread(1, c["cached"], c["batch"])) // 2
    return {"bytes": 9 * c["batch"] + 8 * half + 8, "flops": 0}


def exact(case, seed):
    if case["op"] in ("reserve", "release"):
        return None
    state = prepare(case, seed)
    return _exact_attention(state) if case["op"] == "attention" else _exact_rotary(state)


def _exact_attention(s):
    """Request by request: softmax(q . k / sqrt(dim)) v and the logarithm of the softmax's denominator."""
    c = s["case"]
    group = c["heads"] // c["kv_heads"]
    out = torch.zeros((c["batch"], c["heads"], c["dim"]), dtype=torch.float64, device=DEVICE)
    lse = torch.full((c["batch"], c["heads"]), -math.inf, dtype=torch.float64, device=DEVICE)
    for b, length in enumerate(s["lengths"].tolist()):
        start = max(0, length - c["window"]) if c["window"] else 0
        if length == start:
            continue
        at = torch.arange(start, length, device=DEVICE)
        page, line = s["table"][b].long()[at // c["page"]], at % c["page"]
        for h in range(c["kv_heads"]):
            heads = slice(h * group, (h + 1) * group)
            scores = s["query"][b, heads].double() @ s["keys"][page, line, h].double().T / math.sqrt(c["dim"])
            out[b, heads] = torch.softmax(scores, -1) @ s["values"][page, line, h].double()
            lse[b, heads] = torch.logsumexp(scores, -1)
    return [out, lse] if c["lse"] else [out]


def _exact_rotary(s):
    """Each pair as a complex number, turned by multiplication with cos + i sin."""
    c = s["case"]
    rot, half = c["rot"], c["rot"] // 2
    turn = s["rotary"].double()[s["positions"].long()]
    turn = torch.complex(turn[:, :half], turn[:, half:])[:, None]

    def turned(x, weight):
        x = x.double()
        if weight is not None:
            x = x / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / c["dim"] + 1e-6) * weight.double()
        pairs = x[..., :rot].reshape(*x.shape[:2], half, 2) if c["interleaved"] else \
            x[..., :rot].reshape(*x.shape[:2], 2, half).transpose(2, 3)
        pairs = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
        pairs = pairs if c["interleaved"] else pairs.transpose(2, 3)
        return torch.cat([pairs.reshape(*x.shape[:2], rot), x[..., rot:]], -1)

    tokens = c["tokens"]
    keys, values = s["keys"].double(), s["values"].double()
    slots = s["slots"][:tokens].long()
    keys.view(-1, c["kv_heads"], c["dim"])[slots] = turned(s["key"], s["key_norm"])[:tokens]
    values.view(-1, c["kv_heads"], c["dim"])[slots] = s["value"][:tokens].double()
    return [turned(s["query"], s["query_norm"]), keys, values]
