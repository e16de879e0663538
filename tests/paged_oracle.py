"""Plain 64-bit CPU forms of the paged-cache operators, from their definitions."""

import math

import torch


def reserve(lengths, new, table, free, used, page, rows, stride):
    """reserve_pages request by request, in Python integers."""
    lengths, new, free, used = [[int(x) for x in t] for t in (lengths, new, free, used)]
    used = used[0]
    table = [list(map(int, row)) for row in table.tolist()]
    width = len(table[0]) if table else 0
    positions, slots, offsets = [0] * rows, [-1] * rows, []
    lengths_out, asked, taken, refused, packed = list(lengths), 0, 0, 0, 0
    available = len(free) - used if 0 <= used <= len(free) else 0
    for b, (n, m) in enumerate(zip(lengths, new)):
        row = b * stride if stride else packed
        offsets.append(row)
        packed += max(m, 0)
        ok = n >= 0 and m >= 0 and n + m <= width * page
        if m > 0:
            ok = ok and row + m <= rows and (not stride or m <= stride)
        held = -(-n // page) if ok else 0
        need = -(-(n + m) // page) - held if ok else 0
        first, asked = asked, asked + need
        if not ok or (need and asked > available):
            refused += 1
            continue
        if need:
            taken = asked
        for j in range(need):
            table[b][held + j] = free[used + first + j]
        lengths_out[b] = n + m
        for i in range(m):
            p = n + i
            positions[row + i] = p
            page_id = table[b][p // page]
            slots[row + i] = page_id * page + p % page if 0 <= page_id < len(free) else -1
    offsets.append(len(lengths) * stride if stride else packed)
    return positions, slots, offsets, lengths_out, [used + taken], [refused], table


def release(lengths, done, table, free, used, page):
    lengths, free, used = [int(x) for x in lengths], [int(x) for x in free], int(used[0])
    width = table.shape[1]
    pages = []
    for b, n in enumerate(lengths):
        if done[b]:
            pages += [int(x) for x in table[b, :min(width, -(-max(n, 0) // page))]]
            lengths[b] = 0
    base = used - len(pages)
    for i, page_id in enumerate(pages):
        if 0 <= base + i < len(free):
            free[base + i] = page_id
    return lengths, [max(base, 0)], free


def rotated(x, positions, rotary, interleaved=False, norm=None, eps=1e-6):
    """(rows, heads, width) in 64 bits: optional norm, then the rotation."""
    x = x.detach().cpu().double()
    if norm is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * norm.cpu().double()
    rotary = rotary.cpu().double()
    rot = rotary.shape[1]
    out = x.clone()
    for t, p in enumerate(positions.tolist()):
        known = 0 <= p < rotary.shape[0]
        for i in range(rot // 2):
            c, s = (rotary[p, i], rotary[p, rot // 2 + i]) if known else (math.nan, math.nan)
            a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
            out[t, :, a] = x[t, :, a] * c - x[t, :, b] * s
            out[t, :, b] = x[t, :, b] * c + x[t, :, a] * s
    return out


def rotated_many(x, positions, rotary, interleaved=False, norm=None, eps=1e-6):
    """`rotated` for many rows: all pairs at once, on x's device."""
    x, rotary = x.detach().double(), rotary.double()
    if norm is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * norm.double()
    rot, p = rotary.shape[1], positions.long()
    known = (p >= 0) & (p < rotary.shape[0])
    turn = torch.where(known[:, None], rotary[torch.where(known, p, 0)], math.nan)[:, None]
    c, s = turn[..., :rot // 2], turn[..., rot // 2:]
    first, second = (slice(0, rot, 2), slice(1, rot, 2)) if interleaved else (slice(0, rot // 2), slice(rot // 2, rot))
    out = x.clone()
    out[..., first] = x[..., first] * c - x[..., second] * s
    out[..., second] = x[..., second] * c + x[..., first] * s
    return out


def stored_many(pages, rows, slots):
    """`stored` for many rows."""
    out = pages.detach().double().reshape(-1, *pages.shape[2:]).clone()
    real = (slots >= 0) & (slots < out.shape[0])
    out[slots[real].long()] = rows.double()[real]
    return out.reshape(pages.shape)


def stored(pages, rows, slots):
    """The cache (64 bits) after `rows` were written to their slots."""
    pages = pages.detach().cpu().double().clone()
    flat = pages.reshape(-1, *pages.shape[2:])
    for row, slot in zip(rows, slots.tolist()):
        if 0 <= slot < flat.shape[0]:
            flat[slot] = row
    return flat.reshape(pages.shape)


def attend(query, keys, values, table, lengths, scale=None, window=None):
    """(out, lse, size, reach) in 64 bits: size is sum_j p_j |v_j|, reach the largest scale * sum_d |q_d k_jd| (what
    the errors of the sums and of the scores scale with)."""
    query, keys, values = (t.detach().cpu().double() for t in (query, keys, values))
    table, lengths = table.cpu(), lengths.cpu()
    batch, heads, dim = query.shape
    pages, page, kv_heads, _ = keys.shape
    scale = dim ** -0.5 if scale is None else scale
    out = torch.zeros(batch, heads, dim, dtype=torch.float64)
    size = torch.zeros(batch, heads, dim, dtype=torch.float64)
    lse = torch.full((batch, heads), -math.inf, dtype=torch.float64)
    reach = torch.zeros(batch, heads, dtype=torch.float64)
    for b in range(batch):
        n = min(max(int(lengths[b]), 0), table.shape[1] * page)
        at = torch.arange(max(0, n - window) if window else 0, n)
        ids = table[b].long()[at // page]
        real = (ids >= 0) & (ids < pages)
        ids, line = ids[real], (at % page)[real]
        if not len(ids):
            continue
        k, v = keys[ids, line], values[ids, line]
        for h in range(heads):
            kv = h // (heads // kv_heads)
            scores = (k[:, kv] @ query[b, h]) * scale
            p = torch.softmax(scores, 0)
            out[b, h] = p @ v[:, kv]
            size[b, h] = p @ v[:, kv].abs()
            lse[b, h] = torch.logsumexp(scores, 0)
            reach[b, h] = (k[:, kv].abs() @ query[b, h].abs()).max() * scale
    return out, lse, size, reach
