"""The paged-cache operators on the GPU against their definitions in 64 bits (tests/paged_oracle.py)."""

import ctypes
import math
import threading

import pytest
import torch
from torch.autograd import forward_ad

import paged_oracle as oracle
from neuralzip_b200 import _native
from neuralzip_b200.gpu import paged

pytestmark = pytest.mark.gpu
DEVICE = "cuda"
HALF_ULP = {t: torch.finfo(t).eps / 2 for t in (torch.bfloat16, torch.float16, torch.float32)}
# Half the smallest subnormal: how far a rounding near zero may be off.
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}


def _gen(seed):
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _randn(shape, gen, dtype):
    return torch.randn(shape, generator=gen, device=DEVICE).to(dtype)


def _int(values):
    return torch.tensor(list(values), dtype=torch.int32, device=DEVICE)


# ---- page bookkeeping -----------------------------------------------------------------

def _held(lengths, width, order, page):
    table, used = torch.full((len(lengths), width), -7, dtype=torch.int32), 0
    for b, n in enumerate(lengths):
        count = min(width, -(-max(n, 0) // page))
        table[b, :count] = order[used:used + count]
        used += count
    return table, used


RESERVE = {
    "one token": ([0], [1], 16, 4, 8, 0, None),
    "nothing new": ([5, 16, 0], [0, 0, 0], 16, 4, 8, 0, None),
    "page borders": ([15, 16, 17, 31, 32, 0], [1, 1, 1, 1, 1, 1], 16, 4, 20, 1, None),
    "page borders inside": ([15, 0, 3, 8], [18, 16, 40, 9], 8, 8, 40, 0, None),
    "pages of one token": ([3, 0, 2], [2, 5, 1], 1, 9, 20, 0, None),
    "padded rows": ([0, 7, 3], [5, 0, 2], 4, 6, 20, 9, None),
    "too few pages": ([4, 4, 4, 3], [9, 1, 9, 1], 4, 8, 9, 0, None),
    "row of the table full": ([4, 30, 2], [3, 3, 3], 4, 8, 30, 0, None),
    "negative counts": ([4, -3, 2, 1], [3, 3, -1, 2], 4, 8, 30, 0, None),
    "rows too few": ([0, 0, 0], [5, 6, 2], 4, 8, 30, 0, 9),
    "rows of a stride too few": ([0, 0, 0], [3, 4, 1], 4, 8, 30, 3, 7),
    "rows behind": ([1, 2], [3, 3], 4, 8, 30, 0, 21),
    "no rows": ([1, 2], [0, 0], 4, 8, 30, 0, 0),
    "used above the pages": ([1, 2], [3, 1], 4, 8, 3, 0, None),
}


@pytest.mark.parametrize("case", RESERVE)
@pytest.mark.parametrize("in_place", [False, True])
def test_reserve(case, in_place):
    lengths, new, page, width, pages, stride, rows = RESERVE[case]
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(1)).to(torch.int32)
    table, used = _held(lengths, width, torch.cat([order, order]), page)
    if rows is None:
        rows = stride * len(new) if stride else sum(max(x, 0) for x in new)
    if case == "used above the pages":
        used = pages + 2
    want = oracle.reserve(lengths, new, table, order, [used], page, rows, stride)
    args = [_int(lengths), _int(new), table.to(DEVICE), order.to(DEVICE), _int([used])]
    out = {"lengths_out": args[0], "used_out": args[4]} if in_place else {}
    r = paged.reserve_pages(*args, page_size=page, rows=rows, row_stride=stride, **out)
    got = (r.positions, r.slots, r.row_offsets, r.lengths, r.used, r.refused, args[2])
    for name, a, b in zip(("positions", "slots", "offsets", "lengths", "used", "refused", "table"), got, want):
        assert a.tolist() == b, name
    assert (r.lengths is args[0]) == in_place and (in_place or args[0].tolist() == lengths)


@pytest.mark.parametrize("new,rows", [([3, 2 ** 31 - 1], 5), ([3, 2 ** 31 - 1, 2], 5), ([3, 2 ** 30 - 1], 5),
                                      ([2 ** 30, 3], 5), ([2, 2 ** 30, 2 ** 31 - 1, 1], 9), ([1] * 40 + [2 ** 31 - 1], 41),
                                      ([4] * 300 + [2 ** 31 - 1] * 3 + [1] * 800, 1203)])
@pytest.mark.parametrize("in_place", [False, True])
def test_reserve_counts_beyond_all_rows(new, rows, in_place):
    """Requests of more rows than there can be are refused and leave those before them alone; offsets end at 2^30."""
    page, width, pages = 4, 8, 700
    lengths = [b % 7 for b in range(len(new))]
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(3)).to(torch.int32)
    held = [-(-n // page) for n in lengths]
    table, used = _held(lengths, width, torch.arange(sum(held), dtype=torch.int32) % pages, page)
    used = min(used, 20)
    want = oracle.reserve(lengths, new, table, order, [used], page, rows, 0)
    want[2][:] = [min(x, 2 ** 30) for x in want[2]]
    args = [_int(lengths), _int(new), table.to(DEVICE), order.to(DEVICE), _int([used])]
    out = {"lengths_out": args[0], "used_out": args[4]} if in_place else {}
    r = paged.reserve_pages(*args, page_size=page, rows=rows, **out)
    got = (r.positions, r.slots, r.row_offsets, r.lengths, r.used, r.refused, args[2])
    for name, a, b in zip(("positions", "slots", "offsets", "lengths", "used", "refused", "table"), got, want):
        assert a.tolist() == b, name


def test_reserve_all_rows_there_can_be():
    """One request of 2^30 new tokens, which is the most that a call has rows for."""
    rows, page = 1 << 30, 1 << 20
    table = torch.full((1, 1024), -1, dtype=torch.int32, device=DEVICE)
    r = paged.reserve_pages(_int([0]), _int([rows]), table, _int(range(1024)), _int([0]), page_size=page, rows=rows)
    assert [r.lengths.tolist(), r.used.tolist(), r.refused.tolist(), r.row_offsets.tolist()] == [[rows], [1024], [0], [0, rows]]
    assert table[0].tolist() == list(range(1024))
    place = torch.arange(rows, dtype=torch.int32, device=DEVICE)
    assert torch.equal(r.positions, place) and torch.equal(r.slots, place)


@pytest.mark.parametrize("batch,longest,page,stride", [(64, 1, 16, 1), (129, 700, 16, 0), (1023, 9, 8, 11),
                                                       (4096, 3, 4, 0), (257, 257, 64, 0), (1, 70001, 32, 0)])
def test_reserve_and_release_large(batch, longest, page, stride):
    g = torch.Generator().manual_seed(batch)
    lengths = torch.randint(0, 300, (batch,), generator=g)
    new = torch.randint(0, longest + 1, (batch,), generator=g)
    new[0] = longest
    width = (299 + longest) // page + 1
    held = (lengths + page - 1) // page
    need = int(((lengths + new + page - 1) // page - held).sum())
    pages = int(held.sum()) + max(need - 3, 0)  # a few requests may be refused
    order = torch.randperm(pages, generator=g).to(torch.int32)
    table, used = _held(lengths.tolist(), width, order, page)
    rows = (batch * stride if stride else int(new.sum())) + 5
    want = oracle.reserve(lengths, new, table, order, [used], page, rows, stride)
    wide = torch.full((batch, width + 3), -7, dtype=torch.int32, device=DEVICE)  # a strided block table
    view = wide[:, :width]
    view.copy_(table)
    r = paged.reserve_pages(lengths.to(DEVICE, torch.int32), new.to(DEVICE, torch.int32), view, order.to(DEVICE),
                            _int([used]), page_size=page, rows=rows, row_stride=stride)
    for name, a, b in zip(("positions", "slots", "offsets", "lengths", "used", "refused", "table"),
                          (r.positions, r.slots, r.row_offsets, r.lengths, r.used, r.refused, view), want):
        assert torch.equal(a.cpu(), torch.tensor(b, dtype=torch.int32).view(a.shape)), name
    assert (wide[:, width:] == -7).all()
    done = torch.rand(batch, generator=g) < 0.6
    free = order.to(DEVICE)
    want = oracle.release(r.lengths.cpu(), done, view.cpu(), order, r.used.cpu(), page)
    got = paged.release_pages(r.lengths, done.to(DEVICE), view, free, r.used, page_size=page)
    for a, b in zip((*got, free), want):
        assert torch.equal(a.cpu(), torch.tensor(b, dtype=torch.int32))
    left, base = got[0].tolist(), int(got[1])
    held = [x for b, n in enumerate(left) for x in view[b, :-(-n // page)].tolist()]
    assert sorted(free[base:].tolist() + held) == list(range(pages))  # every page is free or held, once


# In place: clusters of 1, 2, 4 and 8 CTAs, with 256 threads each or 1024, and beyond 8192 rows four of them a thread.
@pytest.mark.parametrize("batch,longest,page,stride", [(64, 30, 16, 0), (64, 90, 4, 0), (256, 21, 2, 0), (256, 40, 2, 45),
                                                       (129, 1024, 16, 0), (1025, 5, 1, 0), (1023, 9, 1, 11),
                                                       (4096, 3, 4, 0), (4096, 9, 1, 10), (1, 70001, 2, 0)])
def test_reserve_and_release_in_place(batch, longest, page, stride):
    """As generation calls them: each call reads the lengths and the stack's top that it updates."""
    g = torch.Generator().manual_seed(batch + longest)
    lengths = torch.randint(0, 50, (batch,), generator=g)
    width = (49 + longest) // page + 1
    held = (lengths + page - 1) // page
    pages = int(held.sum()) + 2 * batch * -(-longest // page)
    order = torch.randperm(pages, generator=g).to(torch.int32)
    table, used = _held(lengths.tolist(), width, order, page)
    state = [lengths.to(DEVICE, torch.int32), table.to(DEVICE), order.to(DEVICE), _int([used])]
    for turn in range(6):  # grow, end some, grow, ...
        before = [t.cpu() for t in state]
        if turn % 2 == 0:
            new = torch.randint(0, longest + 1, (batch,), generator=g)
            new[0] = longest - turn
            rows = (batch * stride if stride else int(new.sum())) + turn
            want = oracle.reserve(before[0], new, before[1], before[2], before[3].tolist(), page, rows, stride)
            r = paged.reserve_pages(state[0], new.to(DEVICE, torch.int32), *state[1:], page_size=page, rows=rows,
                                    row_stride=stride, lengths_out=state[0], used_out=state[3])
            got = (r.positions, r.slots, r.row_offsets, state[0], state[3], r.refused, state[1])
            assert r.lengths is state[0] and r.used is state[3] and torch.equal(state[2].cpu(), before[2])
        else:
            done = torch.rand(batch, generator=g) < (0.9 if batch > 1 else 1.1)
            want = oracle.release(before[0], done, before[1], before[2], before[3], page)
            got = paged.release_pages(state[0], done.to(DEVICE), *state[1:], page_size=page, lengths_out=state[0],
                                      used_out=state[3])
            assert got[0] is state[0] and got[1] is state[3] and torch.equal(state[1].cpu(), before[1])
            got = (*got, state[2])
        for i, (a, b) in enumerate(zip(got, want, strict=True)):
            assert torch.equal(a.cpu(), torch.tensor(b, dtype=torch.int32).view(a.shape)), (turn, i)
        left, top = state[0].tolist(), int(state[3])
        owned = [x for b, n in enumerate(left) for x in state[1][b, :-(-n // page)].tolist()]
        assert sorted(state[2][top:].tolist() + owned) == list(range(pages))  # every page is free or held, once


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("batch,longest", [(200, 4000), (1, 1000000), (2000, 500)])
def test_reserve_and_release_four_rows_a_thread(batch, longest, in_place):
    """More rows and pages than the GPU has threads for."""
    g = torch.Generator().manual_seed(batch)
    new, lengths = torch.randint(longest // 2, longest + 1, (batch,), generator=g), torch.zeros(batch, dtype=torch.int64)
    pages, rows = int(new.sum()) + 7, int(new.sum()) + 3
    order = torch.randperm(pages, generator=g).to(torch.int32)
    args = [lengths.to(DEVICE, torch.int32), torch.full((batch, longest), -7, dtype=torch.int32, device=DEVICE),
            order.to(DEVICE), _int([0])]
    out = {"lengths_out": args[0], "used_out": args[3]} if in_place else {}
    r = paged.reserve_pages(args[0], new.to(DEVICE, torch.int32), *args[1:], page_size=1, rows=rows, **out)
    ends = new.cumsum(0)
    owner = torch.repeat_interleave(torch.arange(batch), new)
    place = torch.arange(len(owner)) - (ends - new)[owner]
    assert torch.equal(r.positions.cpu(), torch.cat([place, torch.zeros(3, dtype=torch.int64)]).int())
    assert torch.equal(r.slots.cpu(), torch.cat([order[:rows - 3], torch.full((3,), -1, dtype=torch.int32)]))
    table = torch.full((batch, longest), -7, dtype=torch.int32)
    table[owner, place] = order[:rows - 3]
    assert torch.equal(args[1].cpu(), table) and torch.equal(r.lengths.cpu(), new.int())
    assert r.used.tolist() == [rows - 3] and r.refused.tolist() == [0]
    done = torch.rand(batch, generator=g) < 0.95 if batch > 1 else torch.ones(1, dtype=torch.bool)
    out = {"lengths_out": r.lengths, "used_out": r.used} if in_place else {}
    left, used = paged.release_pages(r.lengths, done.to(DEVICE), args[1], args[2], r.used, page_size=1, **out)
    back = order[:rows - 3][done[owner]]
    free = order.clone()
    free[rows - 3 - len(back):rows - 3] = back
    assert torch.equal(args[2].cpu(), free) and torch.equal(left.cpu(), torch.where(done, 0, new).int())
    assert used.tolist() == [rows - 3 - len(back)]


@pytest.mark.parametrize("lengths,done,used,in_place", [
    ([0, 5, 17], [True, True, False], 3, False), ([4, 5, 17], [False] * 3, 4, True), ([4, -5, 99], [True] * 3, 20, True),
    ([4, 8, 16], [True] * 3, 2, False)])  # the last: more pages than the stack gave out
def test_release(lengths, done, used, in_place):
    order = torch.randperm(24, generator=torch.Generator().manual_seed(2)).to(torch.int32)
    table, _ = _held(lengths, 5, order, 4)
    want = oracle.release(lengths, done, table, order, [used], 4)
    args = [_int(lengths), torch.tensor(done, device=DEVICE), table.to(DEVICE), order.to(DEVICE), _int([used])]
    out = {"lengths_out": args[0], "used_out": args[4]} if in_place else {}
    got = paged.release_pages(*args, page_size=4, **out)
    assert [got[0].tolist(), got[1].tolist(), args[3].tolist()] == list(want)
    assert torch.equal(args[2].cpu(), table)


@pytest.mark.parametrize("used", [40, 64, 90, 5])
@pytest.mark.parametrize("in_place", [False, True])
def test_release_of_more_pages_than_32_bits_count(used, in_place):
    """Requests that share one row of 2^20 pages, 2^32 in all: the stack's top gets what lies directly under it."""
    batch, width, pages = 4096, 1 << 20, 64
    tail, done = [3, 0, 5, 7, 2, 11], [True, True, True, False, True, True]
    lengths = _int([width] * (batch - 6) + tail)
    mask = torch.ones(batch, dtype=torch.bool, device=DEVICE)
    mask[-6:] = torch.tensor(done, device=DEVICE)
    row, free, top = torch.arange(width, dtype=torch.int32, device=DEVICE), _int(range(100, 164)), _int([used])
    out = {"lengths_out": lengths, "used_out": top} if in_place else {}
    got = paged.release_pages(lengths, mask, row.expand(batch, width), free, top, page_size=1, **out)
    ids = list(range(width - 100, width)) + [x for n, d in zip(tail, done) if d for x in range(n)]
    want = [ids[i - used] if i < used else 100 + i for i in range(pages)]
    assert free.tolist() == want and got[1].tolist() == [0]
    assert got[0].tolist() == [0] * (batch - 6) + [0 if d else n for n, d in zip(tail, done)]


def test_reserve_from_several_threads():
    """Host threads with different numbers of requests, whose calls meet in the library (ctypes lets go of the
    interpreter's lock), do not take each other's shared memory."""
    lib, statuses = _native.load(), {}
    calls = {}
    for batch in (3100, 4096, 3500, 3008):
        t = {"lengths": torch.zeros(batch), "new_tokens": torch.ones(batch), "block_table": torch.zeros(batch),
             "free_pages": torch.arange(batch), "used": torch.zeros(1), "positions": torch.zeros(batch),
             "slots": torch.zeros(batch), "row_offsets": torch.zeros(batch + 1), "lengths_out": torch.zeros(batch),
             "used_out": torch.zeros(1), "refused": torch.zeros(1)}
        t = {name: x.to(DEVICE, torch.int32) for name, x in t.items()}
        args = _native.Reserve(**{name: x.data_ptr() for name, x in t.items()}, table_stride=1, requests=batch, width=1,
                               pages=batch, rows=batch, row_stride=1, page_shift=0)
        calls[batch] = t, args, torch.cuda.Stream()

    def work(batch):
        _, args, stream = calls[batch]
        call, address, stream = lib.nz_pages_reserve, ctypes.byref(args), ctypes.c_void_p(stream.cuda_stream)
        with torch.cuda.device(0):
            statuses[batch] = {call(address, stream) for _ in range(20000)}

    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(batch,)) for batch in calls]
    for thread in threads:
        thread.start()
    for thread in threads:
        thread.join()
    torch.cuda.synchronize()
    assert statuses == {batch: {_native.OK} for batch in calls}
    for batch, (t, _, _) in calls.items():
        assert torch.equal(t["slots"], t["free_pages"]) and int(t["used_out"]) == batch


def test_lengths_out_must_not_overlap_in_part():
    both = torch.zeros(5, dtype=torch.int32, device=DEVICE)
    table, free, used = torch.zeros(4, 2, dtype=torch.int32, device=DEVICE), _int(range(8)), _int([0])
    with pytest.raises(ValueError, match="overlaps"):
        paged.reserve_pages(both[:4], _int([1] * 4), table, free, used, page_size=4, rows=4, lengths_out=both[1:])
    with pytest.raises(ValueError, match="overlaps"):
        paged.release_pages(both[:4], torch.ones(4, dtype=torch.bool, device=DEVICE), table, free, used, page_size=4,
                            lengths_out=both[1:])


# ---- rotary positions and the cache write -------------------------------------------------

def _rotary_inputs(seed, rows, heads, kv_heads, dim, rot, dtype, page=4, norm=False, far=64):
    gen = _gen(seed)
    pages = rows // page + 3
    fused = _randn((rows, heads + 2 * kv_heads, dim), gen, dtype)
    slots = torch.randperm(pages * page, generator=gen, device=DEVICE)[:rows].to(torch.int32)
    positions = torch.randint(far, (rows,), generator=gen, device=DEVICE, dtype=torch.int32)
    inv = 10000.0 ** (-torch.arange(rot // 2, dtype=torch.float64, device=DEVICE) * 2 / max(rot, 1))
    cache = [_randn((pages, page, kv_heads, dim), gen, dtype) for _ in range(2)]
    norms = [(1 + 0.2 * _randn((dim,), gen, torch.float32)).to(dtype) for _ in range(2)] if norm else [None, None]
    return {"query": fused[:, :heads], "key": fused[:, heads:heads + kv_heads], "value": fused[:, heads + kv_heads:],
            "positions": positions, "slots": slots, "rotary": paged.rotary_table(inv, far), "key_pages": cache[0],
            "value_pages": cache[1], "query_norm": norms[0], "key_norm": norms[1]}


def _near(got, want, moved, dtype):
    """A value rounded once to dtype from 32-bit arithmetic: half a step of
    the value, plus 32 roundings of 2^-24 (the norm's sum of up to 256
    squares in groups of at most 16 a lane and 5 exchanges, its root, quotient
    and two products; the rotation's two products and sum) of the terms,
    whose size `moved` bounds."""
    got = got.cpu().double()
    bound = (want.abs() + moved * 2.0 ** -19) * HALF_ULP[dtype] + moved * 2.0 ** -19 + TINY[dtype]
    assert ((got - want).abs() <= bound).all(), float(((got - want).abs() / bound).max())


def _check_rotary(inputs, interleaved=False, key_out=False, eps=1e-6, **more):
    dtype = inputs["query"].dtype
    before = [inputs[n].clone() for n in ("key_pages", "value_pages")]
    source = {n: inputs[n].clone() for n in ("query", "key", "value")}
    if key_out:
        more["key_out"] = torch.empty_like(inputs["key"])
    out = paged.rotary_store(**inputs, interleaved=interleaved, eps=eps, **more)
    pos, rotary = inputs["positions"], inputs["rotary"]

    def want(x, norm):
        return oracle.rotated(x, pos, rotary, interleaved, norm, eps)

    def moved(x, norm):  # |a| + |b| of a pair, above what a rotation adds up
        x = oracle.rotated(x, pos, torch.tensor([[1.0, 0.0]]).repeat(1, 0), False, norm, eps)
        return 2 * x.abs().amax(-1, keepdim=True).expand_as(x)

    query, key = want(source["query"], inputs["query_norm"]), want(source["key"], inputs["key_norm"])
    _near(out, query, moved(source["query"], inputs["query_norm"]), dtype)
    if key_out:
        _near(more["key_out"], key, moved(source["key"], inputs["key_norm"]), dtype)
    big = moved(source["key"], inputs["key_norm"])
    slots = inputs["slots"]
    _near(inputs["key_pages"], oracle.stored(before[0], key, slots),
          oracle.stored(torch.zeros_like(before[0]), big, slots), dtype)
    stored = oracle.stored(before[1], source["value"].cpu().double(), slots)
    assert torch.equal(inputs["value_pages"].cpu().double(), stored)
    return out


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("heads,kv_heads,dim,rot", [(8, 2, 128, 128), (14, 2, 64, 64), (5, 1, 80, 32), (3, 3, 256, 256),
                                                    (4, 2, 96, 96), (7, 7, 16, 8), (2, 1, 8, 8), (6, 2, 40, 20),
                                                    (2, 2, 18, 10), (3, 1, 2, 2), (2, 1, 64, 0), (2, 2, 250, 126)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("norm", [False, True])
def test_rotary_store(dtype, heads, kv_heads, dim, rot, interleaved, norm):
    inputs = _rotary_inputs(dim + rot, 13, heads, kv_heads, dim, rot, dtype, norm=norm)
    _check_rotary(inputs, interleaved, key_out=norm)


@pytest.mark.parametrize("rows", [1, 2, 33, 1025])
def test_rotary_store_rows(rows):
    _check_rotary(_rotary_inputs(rows, rows, 8, 2, 64, 64, torch.bfloat16, page=16, norm=True))


def test_rotary_store_padding_and_bad_slots():
    """Slots outside the cache leave it alone; positions outside the table give NaN in what they would rotate."""
    inputs = _rotary_inputs(3, 9, 4, 2, 32, 16, torch.bfloat16)
    size = inputs["key_pages"].shape[0] * 4
    inputs["slots"][2], inputs["slots"][5], inputs["slots"][6] = -1, size, 2 ** 31 - 1
    inputs["positions"][2] = 0
    _check_rotary(inputs)
    inputs["positions"][0], inputs["positions"][1] = -1, 64
    out = paged.rotary_store(**inputs)
    assert out[:2, :, :16].isnan().all() and not out[:2, :, 16:].isnan().any() and not out[2:].isnan().any()


def test_rotary_store_in_place_strided_and_odd_addresses():
    inputs = _rotary_inputs(4, 11, 4, 2, 64, 64, torch.float16)
    want = paged.rotary_store(**{**inputs, "key_pages": inputs["key_pages"].clone()})
    # A cache whose heads come before its tokens, and one that starts at an odd element.
    heads_first = inputs["key_pages"].permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)
    odd = torch.zeros(inputs["value_pages"].numel() + 1, dtype=torch.float16, device=DEVICE)[1:].view(
        inputs["value_pages"].shape)
    odd.copy_(inputs["value_pages"])
    inputs = {**inputs, "key_pages": heads_first, "value_pages": odd}
    _check_rotary(dict(inputs))
    fused = inputs["query"]
    got = paged.rotary_store(**inputs, query_out=fused)
    assert got is fused and torch.equal(got, want)


def _check_many_rows(inputs, interleaved=False, eps=1e-6, in_place=False, key_out=False):
    """_check_rotary for many rows, some of them padding or with positions outside the table."""
    dtype, rows, heads = inputs["query"].dtype, *inputs["query"].shape[:2]
    size = inputs["key_pages"].shape[0] * inputs["key_pages"].shape[1]
    for at, slot in ((0, -1), (rows // 3, size), (rows // 2, -2 ** 31), (rows - 2, 2 ** 31 - 1), (rows - 1, -1)):
        inputs["slots"][at] = slot
    for at, position in ((1, -1), (rows // 2, inputs["rotary"].shape[0]), (rows - 3, 2 ** 31 - 1)):
        inputs["positions"][at] = position
    before = {n: inputs[n].clone() for n in ("query", "key", "value", "key_pages", "value_pages")}
    more = {"query_out": inputs["query"]} if in_place else {}
    if key_out:
        more["key_out"] = torch.empty_like(inputs["key"])
    out = paged.rotary_store(**inputs, interleaved=interleaved, eps=eps, **more)
    assert out.shape == (rows, heads, inputs["query"].shape[2]) and (not in_place or out is inputs["query"])

    def check(got, want, moved):
        assert torch.equal(got.isnan(), want.isnan())
        got, want, moved = got.double().nan_to_num(0.0), want.nan_to_num(0.0), moved.nan_to_num(0.0)
        bound = (want.abs() + moved * 2.0 ** -19) * HALF_ULP[dtype] + moved * 2.0 ** -19 + TINY[dtype]  # as _near
        assert ((got - want).abs() <= bound).all(), float(((got - want).abs() / bound).max())

    def both(name, norm):  # the rotated rows, and the size that their errors scale with
        want = oracle.rotated_many(before[name], inputs["positions"], inputs["rotary"], interleaved, norm, eps)
        still = oracle.rotated_many(before[name], inputs["positions"] * 0, torch.tensor([[1.0, 0.0]], device=DEVICE), False,
                                    norm, eps)
        return want, 2 * still.abs().amax(-1, keepdim=True).expand_as(want)

    check(out, *both("query", inputs["query_norm"]))
    key, moved = both("key", inputs["key_norm"])
    if key_out:
        check(more["key_out"], key, moved)
    slots = inputs["slots"]
    check(inputs["key_pages"], oracle.stored_many(before["key_pages"], key, slots),
          oracle.stored_many(torch.zeros_like(before["key_pages"]), moved, slots))
    assert torch.equal(inputs["value_pages"].double(), oracle.stored_many(before["value_pages"], before["value"], slots))
    for name in ("key", "value") + (() if in_place else ("query",)):
        assert torch.equal(inputs[name], before[name])


def _many_rows(heads, kv_heads, dim, dtype, rows=7):
    """A few more rows than many_elements() in nz_rotary.cu asks for."""
    least = 6 << 20 if dtype is torch.float32 else 4 << 20
    return least // ((heads + 2 * kv_heads) * dim) + rows


# The streaming kernel, but for 20 + 5 heads x 80, 3 + 1 x 16, 8 + 8 without rotation and, in 16 bits, 14 + 2 x 64, which
# leave too many of its lanes idle: steps that a kind's heads fill and that they do not, groups of 4 to 32 lanes, some of
# them without work.
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("heads,kv_heads,dim,rot", [(32, 8, 128, 128), (32, 8, 80, 80), (12, 12, 96, 96), (14, 2, 64, 64),
                                                    (15, 3, 64, 64), (7, 7, 256, 256), (5, 5, 192, 128), (9, 3, 128, 64),
                                                    (64, 1, 32, 16), (8, 8, 128, 0), (20, 5, 80, 32), (3, 1, 16, 16)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("norm", [False, True])
def test_rotary_store_many_rows(dtype, heads, kv_heads, dim, rot, interleaved, norm):
    inputs = _rotary_inputs(dim + heads, _many_rows(heads, kv_heads, dim, dtype), heads, kv_heads, dim, rot, dtype, page=16,
                            norm=norm, far=500)
    _check_many_rows(inputs, interleaved, 1e-5, in_place=norm, key_out=norm != interleaved)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dim", [128, 80])
def test_rotary_store_many_rows_strided(dtype, dim):
    """Pages whose heads come before their tokens, rows with room between them, keys and values of other strides."""
    rows = _many_rows(24, 4, dim, dtype, 0)
    for extra in (0, 1):  # at the limit and one above it
        inputs = _rotary_inputs(rows, rows + extra, 24, 4, dim, dim, dtype, page=8, norm=True, far=99)
        inputs["key_pages"] = inputs["key_pages"].permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)
        wide = torch.zeros(*inputs["value_pages"].shape[:3], dim + 16, dtype=dtype, device=DEVICE)
        wide[..., 8:8 + dim] = inputs["value_pages"]
        inputs["value_pages"] = wide[..., 8:8 + dim]
        inputs["key"] = inputs["key"].transpose(0, 1).contiguous().transpose(0, 1)
        inputs["value"] = inputs["value"].contiguous()
        _check_many_rows(inputs, key_out=True)
        assert (wide[..., :8] == 0).all() and (wide[..., 8 + dim:] == 0).all()


def test_rotary_store_many_rows_at_odd_addresses():
    """Vectors of 16 bytes do not fit: the kernel of few rows takes them."""
    dtype = torch.bfloat16
    inputs = _rotary_inputs(5, _many_rows(16, 4, 64, dtype), 16, 4, 64, 64, dtype, page=16)
    odd = torch.empty(inputs["query"].numel() + 1, dtype=dtype, device=DEVICE)[1:].view(inputs["query"].shape)
    odd.copy_(inputs["query"])
    _check_many_rows({**inputs, "query": odd}, in_place=True)


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_store_many_rows_captured(interleaved):
    """The streaming kernel in a graph, behind and before kernels that write its inputs and read its outputs."""
    dtype = torch.bfloat16
    inputs = _rotary_inputs(6, _many_rows(32, 8, 128, dtype), 32, 8, 128, 128, dtype, page=16, norm=True, far=99)
    feed = torch.empty_like(inputs["query"])
    paged.rotary_store(**inputs, interleaved=interleaved)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        inputs["query"].copy_(feed)
        paged.rotary_store(**inputs, interleaved=interleaved, query_out=inputs["query"])
        seen = inputs["query"] + 0
        inputs["query"].zero_()
    for seed in range(3):
        feed.copy_(_randn(feed.shape, _gen(seed), dtype))
        want = paged.rotary_store(**{**inputs, "query": feed}, interleaved=interleaved)
        graph.replay()
        assert torch.equal(seen, want) and not inputs["query"].any()


def test_rotary_table_keeps_far_phases():
    inv = torch.tensor([1.0, 0.37], device=DEVICE)
    table = paged.rotary_table(inv, 70001, 1.5)[70000].cpu()
    angle = 70000 * inv.cpu().double()
    want = 1.5 * torch.cat([angle.cos(), angle.sin()])
    # Rounded once to 32 bits; the 64-bit angle is off by 2^-53 of itself.
    assert (table.double() - want).abs().max() <= 1.5 * 2.0 ** -24 + 1e-10


# ---- attention ------------------------------------------------------------------------------

def _attention_inputs(seed, lengths, heads, kv_heads, dim, dtype, page=16, width=None, stale=math.nan, sharp=2.0):
    """Pages lie anywhere in the pool; every slot no request holds (the rest
    of last pages, free pages) holds `stale`."""
    gen = _gen(seed)
    width = width or max(1, max(-(-max(n, 0) // page) for n in lengths))
    held = [min(width, -(-max(n, 0) // page)) for n in lengths]
    pages = sum(held) + 2
    order = torch.randperm(pages, generator=gen, device=DEVICE).to(torch.int32)
    table = torch.full((len(lengths), width), -1, dtype=torch.int32, device=DEVICE)
    keys = torch.full((pages, page, kv_heads, dim), stale, device=DEVICE).to(dtype)
    values = keys.clone()
    first = 0
    for b, (n, count) in enumerate(zip(lengths, held)):
        table[b, :count] = order[first:first + count]
        first += count
        at = torch.arange(min(max(n, 0), width * page), device=DEVICE)
        ids = table[b].long()[at // page]
        keys[ids, at % page] = _randn((len(at), kv_heads, dim), gen, dtype)
        values[ids, at % page] = _randn((len(at), kv_heads, dim), gen, dtype)
    query = (sharp * torch.randn((len(lengths), heads, dim), generator=gen, device=DEVICE)).to(dtype)
    return [query, keys, values, table, _int(lengths)]


def _check_attention(inputs, scale=None, window=None, **more):
    """out is off by the rounding to its type plus, relative to sum p |v|:
    the error of the exponentials, twice that of a score (a dot product in
    32 bits: one rounding of 2^-23 of sum |q k| for each 8 of the width, and
    16 for the joins and the scaling), what p loses where it is held in two
    16-bit parts (2^-15 covers it), and a rounding of 2^-23 for each 16
    positions and 64 for the joins. lse is off by the score's error and the
    sum's."""
    query, keys, values, table, lengths = inputs
    out, lse = paged.paged_attention(*inputs, scale=scale, window=window, return_lse=True, **more)
    assert torch.equal(out, paged.paged_attention(*inputs, scale=scale, window=window)) or "out" in more
    keys, values = (t.nan_to_num(0.0, 0.0, 0.0) if t.isnan().any() or t.isinf().any() else t for t in (keys, values))
    want, want_lse, size, reach = oracle.attend(query, keys, values, table, lengths, scale, window)
    dtype, dim = query.dtype, query.shape[2]
    step = 2.0 ** -23
    score = reach * (dim / 8 + 16) * step + want_lse.abs().nan_to_num(0.0, 0.0, 0.0) * step
    sums = (keys.shape[1] * table.shape[1] / 16 + 64) * step
    parts = 2.0 ** -20 if dtype is torch.float32 else 2.0 ** -15
    error = size * (2 * score[..., None] + parts + sums)
    bound = (want.abs() + error) * HALF_ULP[dtype] + error + TINY[dtype]
    off = (out.cpu().double() - want).abs()
    assert (off <= bound).all(), float((off / bound).max())
    empty = want_lse == -math.inf
    got = lse.cpu().double()
    assert torch.equal(got == -math.inf, empty)
    assert ((got - want_lse).abs()[~empty] <= (score + sums + step)[~empty]).all()
    return out, lse


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("heads,kv_heads,dim", [(14, 2, 64), (8, 2, 128), (4, 4, 128), (12, 1, 80), (32, 2, 96),
                                                (9, 3, 256), (16, 1, 256), (20, 1, 128), (6, 2, 192), (2, 1, 8),
                                                (5, 5, 16), (33, 3, 40), (40, 1, 64)])
def test_attention_heads(dtype, heads, kv_heads, dim):
    _check_attention(_attention_inputs(dim, [0, 1, 15, 16, 17, 63, 64, 65, 200], heads, kv_heads, dim, dtype))


@pytest.mark.parametrize("page", [1, 2, 4, 8, 16, 32, 64, 256])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_attention_pages(page, dtype):
    _check_attention(_attention_inputs(page, [1, 257, 0, 31, 130], 8, 2, 64, dtype, page))


@pytest.mark.parametrize("lengths", [[5000], [4097, 3, 0, 1], [1, 9000, 2, 700, 64], [0, 0], list(range(0, 300, 7)),
                                     [17001], list(range(0, 2100, 70))])
@pytest.mark.parametrize("heads,kv_heads,dim,dtype", [(8, 2, 128, torch.bfloat16), (12, 12, 64, torch.float16),
                                                      (4, 1, 80, torch.float32), (24, 2, 128, torch.bfloat16),
                                                      (6, 6, 80, torch.float32), (10, 1, 256, torch.float16),
                                                      (7, 7, 192, torch.bfloat16)])
def test_attention_lengths(lengths, heads, kv_heads, dim, dtype):
    _check_attention(_attention_inputs(len(lengths), lengths, heads, kv_heads, dim, dtype))


def test_attention_many_requests():
    """4096 requests, most of them short, some empty; and a table wide enough that the work is split."""
    g = torch.Generator().manual_seed(3)
    lengths = torch.randint(0, 40, (4096,), generator=g).tolist()
    _check_attention(_attention_inputs(1, lengths, 2, 1, 32, torch.bfloat16, 8))
    lengths[77], lengths[4000] = 3001, 2500
    _check_attention(_attention_inputs(2, lengths, 2, 1, 32, torch.float16, 8))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("lengths,width", [([700, 20, 1500], 94), ([40000, 3, 9000], 2500)])
def test_attention_captured(dtype, lengths, width):
    """A cluster's launch and a split one with its join, captured, replayed on changed lengths and contents."""
    inputs = _attention_inputs(12, lengths, 8, 2, 64, dtype, width=width, stale=0.0)
    paged.paged_attention(*inputs)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = paged.paged_attention(*inputs, return_lse=True)
    for change in range(3):
        inputs[4][:] = _int([[n, 0, n // 2][(i + change) % 3] for i, n in enumerate(lengths)])
        inputs[0].mul_(-1.5)
        graph.replay()
        want, want_lse = paged.paged_attention(*inputs, return_lse=True)
        assert torch.equal(out, want) and torch.equal(lse, want_lse)


@pytest.mark.parametrize("window", [1, 2, 15, 16, 17, 100, 512, 5000])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_attention_window(window, dtype):
    inputs = _attention_inputs(window, [0, 1, 15, 16, 17, 99, 2000], 8, 2, 64, dtype)
    # Nothing before the window may be read either.
    query, keys, values, table, lengths = inputs
    for b, n in enumerate(lengths.tolist()):
        at = torch.arange(max(0, n - window), device=DEVICE)
        ids = table[b].long()[at // 16]
        for cache in (keys, values):
            cache[ids, at % 16] = math.nan
    _check_attention(inputs, window=window)


@pytest.mark.parametrize("stale", [math.inf, -math.inf, math.nan, 1e4])
def test_attention_ignores_masked_places(stale):
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        _check_attention(_attention_inputs(5, [1, 20, 33, 0], 4, 2, 64, dtype, 32, stale=stale))


def test_attention_bad_pages_and_lengths():
    """Ids outside the cache count as masked, lengths are held to the table's row, negative ones are empty."""
    inputs = _attention_inputs(6, [40, 40, 40, 40, 16], 4, 2, 64, torch.bfloat16, 8, width=5)
    query, keys, values, table, lengths = inputs
    table[0, 1], table[1, 4], table[2, :] = -1, keys.shape[0], -5
    table[3, 0] = 2 ** 31 - 1
    _check_attention(inputs)
    lengths[:] = _int([39, -1, -2 ** 31, 41, 2 ** 31 - 1])
    table[4, 2:] = table[0, 2:]
    _check_attention(inputs)


def test_attention_peaked_scores():
    """One key far above the rest, in each place of a tile and across splits; and scores far below zero."""
    for place in (0, 7, 8, 15, 16, 1000, 2999):
        inputs = _attention_inputs(place, [3000], 4, 2, 64, torch.bfloat16, sharp=0.1)
        query, keys, values, table, _ = inputs
        keys[table[0, place // 16], place % 16] = query.view(2, 2, 64)[:, 0] * 100
        _check_attention(inputs, scale=1.0)
    inputs = _attention_inputs(1, [700], 4, 2, 64, torch.float32, sharp=0.0)
    inputs[0] += 1
    inputs[1] -= 300
    _check_attention(inputs, scale=0.01)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("length,gap", [(60001, 18.0), (3001, 17.0), (300, 16.5), (60001, 30.0)])
def test_attention_small_weights_add_up(dtype, length, gap):
    """One key far above all others, whose weights are each below 2^-24 of its own, but whose sum is not."""
    inputs = _attention_inputs(4, [length], 2, 1, 64, dtype)
    query, keys, values, table, _ = inputs
    query.zero_()
    query[..., 0] = 1
    keys[..., 0] = 0
    at = length // 3
    keys[table[0, at // 16], at % 16, 0, 0] = gap
    values.abs_().add_(1)
    values[table[0, at // 16], at % 16] = 0
    out, _ = _check_attention(inputs, scale=1.0)
    # About length * e^-gap * 1.8; for 60001 and 30 that is 1e-8, which fp16 rounds to zero (its half step there is 2^-25).
    if length * math.exp(-gap) > 2 * TINY[dtype]:
        assert (out > 0).all()


def test_attention_strides():
    inputs = _attention_inputs(8, [100, 37], 8, 4, 64, torch.bfloat16)
    want = paged.paged_attention(*inputs)
    query, keys, values, table, lengths = inputs
    wide = torch.zeros(2, 8, 192, dtype=query.dtype, device=DEVICE)
    wide[..., 64:128] = query
    heads_first = keys.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)
    both = torch.stack([keys, values], 1)
    tables = torch.full((2, 40), -1, dtype=torch.int32, device=DEVICE)
    tables[:, :table.shape[1]] = table
    odd = torch.empty(2 * 8 * 64 + 1, dtype=query.dtype, device=DEVICE)[1:].view(2, 8, 64)  # not 16-byte aligned
    odd.copy_(query)
    for q, k, v, t in ((wide[..., 64:128], keys, values, table), (query, heads_first, values, table),
                       (query, both[:, 0], both[:, 1], table), (query, keys, values, tables),
                       (odd, keys, values, tables[:, :table.shape[1]])):
        assert torch.equal(paged.paged_attention(q, k, v, t, lengths), want)
    out = torch.zeros(8, 2, 65, dtype=query.dtype, device=DEVICE)[..., 1:].transpose(0, 1)
    assert paged.paged_attention(*inputs, out=out) is out and torch.equal(out, want)


def test_attention_offsets_beyond_32_bits():
    """Pages whose elements lie behind 2^32 from the cache's start."""
    kv_heads, dim, page = 8, 128, 16
    pages = (1 << 32) // (page * kv_heads * dim) + 8
    keys = torch.empty((pages, page, kv_heads, dim), dtype=torch.bfloat16, device=DEVICE)
    values = torch.empty_like(keys)
    small = _attention_inputs(9, [100], 16, kv_heads, dim, torch.bfloat16)
    count = small[3].shape[1]
    far = torch.arange(pages - count, pages, device=DEVICE)
    ids = small[3][0].long()
    keys[far], values[far] = small[1][ids], small[2][ids]
    want = paged.paged_attention(*small)
    got = paged.paged_attention(small[0], keys, values, far.to(torch.int32)[None], small[4])
    assert torch.equal(got, want)
    rotary = _rotary_inputs(2, 4, 16, kv_heads, dim, dim, torch.bfloat16, page=page)
    slots = torch.tensor([pages * page - 1 - i for i in range(4)], dtype=torch.int32, device=DEVICE)
    paged.rotary_store(**{**rotary, "slots": slots, "key_pages": keys, "value_pages": values})
    assert torch.equal(values[-1, -4:].flip(0), rotary["value"])


def test_operators_on_another_stream_and_captured():
    """A step (reserve, rotary and write, attention) captured once and
    replayed equals the same steps enqueued one by one; two graphs of it
    share the cache but no workspace."""
    def state():
        gen = _gen(11)
        lengths, page, width, heads, kv_heads, dim = [3, 0, 500, 31, 1000], 16, 70, 8, 2, 64
        order = torch.randperm(300, generator=gen, device=DEVICE).to(torch.int32)
        table, used = _held(lengths, width, order.cpu(), page)
        keys, values = (_randn((300, page, kv_heads, dim), gen, torch.bfloat16) for _ in range(2))
        qkv = _randn((5, heads + 2 * kv_heads, dim), gen, torch.bfloat16)
        inv = 100.0 ** -(torch.arange(dim // 2, device=DEVICE) / (dim / 2))
        return dict(lengths=_int(lengths), used=_int([used]), free=order, table=table.to(DEVICE), keys=keys,
                    values=values, qkv=qkv, rotary=paged.rotary_table(inv, 2000), new=_int([1] * 5))

    def step(s):
        r = paged.reserve_pages(s["lengths"], s["new"], s["table"], s["free"], s["used"], page_size=16, rows=5,
                                row_stride=1, lengths_out=s["lengths"], used_out=s["used"])
        qkv = s["qkv"]
        q = paged.rotary_store(qkv[:, :8], qkv[:, 8:10], qkv[:, 10:], r.positions, r.slots, s["rotary"], s["keys"],
                               s["values"])
        out = paged.paged_attention(q, s["keys"], s["values"], s["table"], s["lengths"])
        qkv[:, :8].copy_(out)  # the next step's inputs depend on this one's result
        return out

    eager, captured = state(), state()
    wants = [step(eager).clone() for _ in range(20)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(side):
        warm = state()
        step(warm)
        for _ in range(2):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                out = step(captured)
            graphs.append((graph, out))
        for i, want in enumerate(wants):
            graph, out = graphs[i % 2]
            graph.replay()
            assert torch.equal(out, want), i
    torch.cuda.current_stream().wait_stream(side)
    for name in ("lengths", "used", "table", "keys", "values"):
        assert torch.equal(eager[name], captured[name]), name


def test_two_streams_at_once():
    """Calls on two streams share nothing, split ones with their workspaces included."""
    cases = [_attention_inputs(seed, lengths, 8, 2, 64, torch.bfloat16, width=2500)
             for seed, lengths in ((1, [40000, 3, 9000]), (2, [17, 39999, 20000]))]
    want = [paged.paged_attention(*c) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(paged.paged_attention(*cases[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[i]) for i in range(2) for x in got[i])


def test_captured_behind_copies_and_another_stream():
    """In a graph each call waits for all that comes before it: copies, fills, other kernels, other streams."""
    for lengths, width in (([300, 20], 32), ([40000, 3, 9000], 2500)):
        inputs = _attention_inputs(5, lengths, 8, 2, 64, torch.bfloat16, width=width)
        query, rest = inputs[0], inputs[1:]
        feed, other = torch.randn_like(query), torch.randn_like(query)
        held, early, late = torch.empty_like(query), torch.empty_like(query), torch.empty_like(query)
        paged.paged_attention(held.zero_(), *rest, out=early), paged.paged_attention(held, *rest, out=late)
        main, side, graph = torch.cuda.Stream(), torch.cuda.Stream(), torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=main):
            held.copy_(feed)
            paged.paged_attention(held, *rest, out=early)
            held.zero_()
            side.wait_stream(main)
            with torch.cuda.stream(side):
                held.add_(other)
                torch.cuda._sleep(200000)
                held.add_(feed)
            main.wait_stream(side)
            paged.paged_attention(held, *rest, out=late)
            held.fill_(7)
        for _ in range(3):
            for tensor in (feed, other):
                tensor.normal_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(early, paged.paged_attention(feed, *rest))
            assert torch.equal(late, paged.paged_attention(other + feed, *rest))
            assert bool((held == 7).all())


def test_known_layouts_refuse_a_table_that_needs_a_gradient():
    inputs = _rotary_inputs(4, 11, 4, 2, 64, 64, torch.bfloat16)
    for _ in range(2):
        paged.rotary_store(**inputs)
    rotary = inputs["rotary"].clone().requires_grad_()
    with pytest.raises(RuntimeError, match="no_grad"):
        paged.rotary_store(**{**inputs, "rotary": rotary})
    with torch.no_grad():
        paged.rotary_store(**{**inputs, "rotary": rotary})


def test_known_layouts_refuse_dual_tensors():
    """A tangent is not dropped: whoever differentiates forwards, by levels or by torch.func, is told."""
    inputs, rotary = _attention_inputs(3, [100, 37, 0], 8, 4, 64, torch.bfloat16), _rotary_inputs(4, 11, 4, 2, 64, 64, torch.bfloat16)
    for _ in range(2):
        paged.paged_attention(*inputs)
        paged.rotary_store(**rotary)
    for grad in (torch.no_grad, torch.enable_grad):
        with forward_ad.dual_level(), grad():
            for i in range(3):
                call = list(inputs)
                call[i] = forward_ad.make_dual(call[i], torch.ones_like(call[i]))
                with pytest.raises(RuntimeError, match="forward-mode"):
                    paged.paged_attention(*call)
            for name in ("query", "key", "value", "rotary", "key_pages", "value_pages"):
                with pytest.raises(RuntimeError, match="forward-mode"):
                    paged.rotary_store(**{**rotary, name: forward_ad.make_dual(rotary[name], torch.ones_like(rotary[name]))})
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda q: paged.paged_attention(q, *inputs[1:]), (inputs[0],), (torch.ones_like(inputs[0]),))


@pytest.mark.parametrize("known", [False, True])
def test_writes_are_seen_by_autograd(known, monkeypatch):
    """A backward pass that saved a tensor which a call wrote since is refused, not computed from what it holds now."""
    attention = _attention_inputs(3, [100, 37, 0], 8, 4, 64, torch.bfloat16)
    rotary = _rotary_inputs(4, 11, 4, 2, 64, 64, torch.float16, norm=True)
    rotary["key_out"] = torch.empty_like(rotary["key"])
    rotary["query_out"] = torch.empty_like(rotary["query"])
    out = torch.empty_like(attention[0])
    order = torch.randperm(24, generator=torch.Generator().manual_seed(2)).to(torch.int32)
    table, used = _held([4, 5, 17], 9, order, 4)
    table, free, lengths, top = table.to(DEVICE), order.to(DEVICE), _int([4, 5, 17]), _int([used])

    def calls():
        paged.rotary_store(**rotary)
        paged.paged_attention(*attention, out=out)
        paged.reserve_pages(lengths, _int([0, 1, 0]), table, free, top, page_size=4, rows=3, lengths_out=lengths, used_out=top)
        paged.release_pages(lengths, torch.tensor([False, False, True], device=DEVICE), table, free, top, page_size=4,
                            lengths_out=lengths, used_out=top)

    if known:
        calls()
    else:
        monkeypatch.setattr(paged, "_calls", None)
        monkeypatch.setattr(paged, "_remember", lambda *_: None)
    written = [rotary[n] for n in ("key_pages", "value_pages", "query_out", "key_out")] + [out, table, free, lengths, top]
    before = [t._version for t in written]
    read = [rotary["query"], rotary["key"], *attention]
    same = [t._version for t in read]
    calls()
    assert [t._version for t in read] == same
    assert all(t._version > v for t, v in zip(written, before))
    x = torch.ones_like(out, requires_grad=True)
    loss = (x * out).sum()
    calls()
    with pytest.raises(RuntimeError, match="inplace operation"):
        loss.backward()
    with torch.inference_mode():  # whose tensors count nothing
        again = [t.clone() for t in attention]
        assert torch.equal(paged.paged_attention(*again, out=torch.empty_like(again[0])), out)


def test_calls_of_known_layouts_equal_checked_calls(monkeypatch):
    """The second call of a layout goes through the extension module; it does what the checked call does."""
    inputs = _attention_inputs(3, [100, 37, 0], 8, 4, 64, torch.bfloat16)
    rotary = _rotary_inputs(4, 11, 4, 2, 64, 64, torch.float16, norm=True)
    order = torch.randperm(24, generator=torch.Generator().manual_seed(2)).to(torch.int32)
    table, used = _held([4, 5, 17], 9, order, 4)

    def results():
        state = [_int([4, 5, 17]), table.to(DEVICE), order.to(DEVICE), _int([used])]
        reserved = paged.reserve_pages(state[0], _int([3, 1, 9]), *state[1:], page_size=4, rows=16)
        released = paged.release_pages(reserved.lengths, torch.tensor([True, False, True], device=DEVICE), *state[1:3],
                                       reserved.used, page_size=4)
        pages = {n: rotary[n].clone() for n in ("key_pages", "value_pages")}
        turned = paged.rotary_store(**{**rotary, **pages}, eps=1e-5)
        out, lse = paged.paged_attention(*inputs, scale=0.3, window=50, return_lse=True)
        alone = paged.paged_attention(*inputs)
        return [*reserved, state[1], *released, state[2], turned, *pages.values(), out, lse, alone]

    results()
    calls = paged._calls
    assert calls is not None  # the module that travels with the library
    known = results()
    monkeypatch.setattr(paged, "_calls", None)
    monkeypatch.setattr(paged, "_remember", lambda *_: None)
    for a, b in zip(known, results(), strict=True):
        assert a.dtype is b.dtype and a.shape == b.shape and a.stride() == b.stride()
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    # A layout it knows is still refused for what the layout does not show.
    monkeypatch.setattr(paged, "_calls", calls)
    with pytest.raises(RuntimeError, match="no_grad"):
        paged.paged_attention(inputs[0].clone().requires_grad_(), *inputs[1:])
    with pytest.raises(TypeError, match="scale"):
        paged.paged_attention(*inputs, scale="1")
    with pytest.raises(TypeError, match="eps"):
        paged.rotary_store(**rotary, eps=None)
    odd = torch.zeros(inputs[1].numel() + 1, dtype=torch.bfloat16, device=DEVICE)[1:].view(inputs[1].shape)
    with pytest.raises(ValueError, match="16-byte"):
        paged.paged_attention(inputs[0], odd, *inputs[2:])
    with pytest.raises(TypeError, match="whole number"):
        paged.paged_attention(*inputs, window=50.0)
