"""The paged-cache operators' refusals and host logic, which need no GPU."""

import ctypes
import shutil
import subprocess
from pathlib import Path

import pytest
import torch
from torch.autograd import forward_ad

import paged_oracle as oracle
from neuralzip_b200 import _native
from neuralzip_b200.gpu import paged

ROOT = Path(__file__).resolve().parents[1]
I32 = torch.int32


def _reserve_args(**change):
    args = dict(lengths=torch.zeros(3, dtype=I32), new_tokens=torch.ones(3, dtype=I32),
                block_table=torch.zeros(3, 4, dtype=I32), free_pages=torch.arange(12, dtype=I32),
                used=torch.zeros(1, dtype=I32), page_size=16, rows=3)
    args.update(change)
    return args


@pytest.mark.parametrize("change,error,match", [
    ({}, ValueError, "CUDA device"),
    ({"lengths": [0, 0, 0]}, TypeError, "lengths must be a tensor"),
    ({"lengths": torch.zeros(3)}, TypeError, "lengths must be torch.int32"),
    ({"lengths": torch.zeros(0, dtype=I32)}, ValueError, "1 to 4096 requests"),
    ({"lengths": torch.zeros(4097, dtype=I32)}, ValueError, "1 to 4096 requests"),
    ({"lengths": torch.zeros(3, 1, dtype=I32)}, ValueError, "1 dimensions"),
    ({"lengths": torch.zeros(6, dtype=I32)[::2]}, ValueError, "contiguous"),
    ({"new_tokens": torch.ones(2, dtype=I32)}, ValueError, "new_tokens must have 3"),
    ({"block_table": torch.zeros(2, 4, dtype=I32)}, ValueError, "3 rows"),
    ({"block_table": torch.zeros(4, 3, dtype=I32).T}, ValueError, "columns must be contiguous"),
    ({"block_table": torch.zeros(1, 4, dtype=I32).expand(3, 4)}, ValueError, "rows must not overlap"),
    ({"free_pages": torch.arange(12)}, TypeError, "free_pages must be torch.int32"),
    ({"used": torch.zeros(2, dtype=I32)}, ValueError, "used must have 1"),
    ({"page_size": 24}, ValueError, "power of two"),
    ({"page_size": 0}, ValueError, "power of two"),
    ({"page_size": 16.0}, TypeError, "whole number"),
    ({"page_size": True}, TypeError, "whole number"),
    ({"rows": -1}, ValueError, "rows"),
    ({"row_stride": -1}, ValueError, "rows"),
    ({"lengths_out": torch.zeros(2, dtype=I32)}, ValueError, "lengths_out"),
    ({"used_out": torch.zeros(1)}, TypeError, "used_out"),
    ({"used": torch.zeros(1, dtype=I32, device="meta")}, ValueError, "one device"),
])
def test_reserve_refusals(change, error, match):
    with pytest.raises(error, match=match):
        paged.reserve_pages(**_reserve_args(**change))


@pytest.mark.parametrize("change,error,match", [
    ({}, ValueError, "CUDA device"),
    ({"done": torch.zeros(3, dtype=I32)}, TypeError, "done must be torch.bool"),
    ({"done": torch.zeros(4, dtype=torch.bool)}, ValueError, "done must have 3"),
    ({"page_size": 3}, ValueError, "power of two"),
    ({"lengths_out": torch.zeros(3)}, TypeError, "lengths_out"),
])
def test_release_refusals(change, error, match):
    args = _reserve_args(done=torch.zeros(3, dtype=torch.bool))
    for name in ("new_tokens", "rows"):
        del args[name]
    args.update(change)
    with pytest.raises(error, match=match):
        paged.release_pages(**args)


def _rotary_args(**change):
    def t(*shape, dtype=torch.bfloat16):
        return torch.zeros(shape, dtype=dtype)

    args = dict(query=t(5, 4, 64), key=t(5, 2, 64), value=t(5, 2, 64), positions=torch.zeros(5, dtype=I32),
                slots=torch.zeros(5, dtype=I32), rotary=torch.zeros(9, 64), key_pages=t(3, 16, 2, 64),
                value_pages=t(3, 16, 2, 64))
    args.update(change)
    return args


B = torch.bfloat16


@pytest.mark.parametrize("change,error,match", [
    ({}, ValueError, "CUDA device"),
    ({"query": None}, TypeError, "query must be a tensor"),
    ({"query": torch.zeros(5, 4, 64, dtype=torch.float64)}, TypeError, "bfloat16, float16 or float32"),
    ({"query": torch.zeros(5, 4, dtype=B)}, ValueError, "3 dimensions"),
    ({"query": torch.zeros(5, 4, 32, dtype=B)}, ValueError, "head width"),
    ({"query": torch.zeros(5, 64, 4, dtype=B).transpose(1, 2)}, ValueError, "last dimension of query"),
    ({"key": torch.zeros(5, 3, 64, dtype=B)}, ValueError, "key must have the shape"),
    ({"value": torch.zeros(5, 2, 64)}, TypeError, "value must be torch.bfloat16"),
    ({"positions": torch.zeros(5, dtype=torch.int64)}, TypeError, "positions must be torch.int32"),
    ({"slots": torch.zeros(4, dtype=I32)}, ValueError, "slots must have 5"),
    ({"rotary": torch.zeros(9, 64, dtype=B)}, TypeError, "rotary must be torch.float32"),
    ({"rotary": torch.zeros(9, 66)}, ValueError, "rotated width"),
    ({"rotary": torch.zeros(9, 3)}, ValueError, "rotated width"),
    ({"rotary": torch.zeros(64, 9).T}, ValueError, "last dimension of rotary"),
    ({"key_pages": torch.zeros(3, 12, 2, 64, dtype=B)}, ValueError, "power of two"),
    ({"key_pages": torch.zeros(3, 16, 2, 64)}, TypeError, "key_pages must be torch.bfloat16"),
    ({"value_pages": torch.zeros(2, 16, 2, 64, dtype=B)}, ValueError, "value_pages must have the shape"),
    ({"value_pages": torch.zeros(1, 16, 2, 64, dtype=B).expand(3, 16, 2, 64)}, ValueError, "overlap"),
    ({"query_out": torch.zeros(5, 1, 64, dtype=B).expand(5, 4, 64)}, ValueError, "overlap"),
    ({"query_out": torch.zeros(5, 4, 64)}, TypeError, "query_out"),
    ({"key_out": torch.zeros(5, 4, 64, dtype=B)}, ValueError, "key_out must have the shape"),
    ({"query_norm": torch.ones(64)}, TypeError, "query_norm must be torch.bfloat16"),
    ({"key_norm": torch.ones(32, dtype=B)}, ValueError, "key_norm must have 64"),
    ({"query": torch.zeros(5, 4, 64, dtype=B, requires_grad=True)}, RuntimeError, "no_grad"),
    ({"query_norm": torch.ones(64, dtype=B, requires_grad=True)}, RuntimeError, "no_grad"),
])
def test_rotary_refusals(change, error, match):
    with pytest.raises(error, match=match):
        paged.rotary_store(**_rotary_args(**change))


def test_rotary_refuses_wide_and_odd_heads():
    for dim in (258, 63):
        change = {n: torch.zeros(5, h, dim, dtype=B) for n, h in (("query", 4), ("key", 2), ("value", 2))}
        change.update({n: torch.zeros(3, 16, 2, dim, dtype=B) for n in ("key_pages", "value_pages")})
        with pytest.raises(ValueError, match="even and at most 256"):
            paged.rotary_store(**_rotary_args(**change))


def _attention_args(dim=64, dtype=B, **change):
    args = dict(query=torch.zeros(3, 4, dim, dtype=dtype), key_pages=torch.zeros(5, 16, 2, dim, dtype=dtype),
                value_pages=torch.zeros(5, 16, 2, dim, dtype=dtype), block_table=torch.zeros(3, 2, dtype=I32),
                lengths=torch.ones(3, dtype=I32))
    args.update(change)
    return args


@pytest.mark.parametrize("change,error,match", [
    ({}, ValueError, "CUDA device"),
    ({"query": torch.zeros(3, 5, 64, dtype=B)}, ValueError, "no multiple"),
    ({"query": torch.zeros(3, 0, 64, dtype=B)}, ValueError, "no multiple"),
    ({"query": torch.zeros(2, 4, 64, dtype=B)}, ValueError, "lengths must have 2"),
    ({"query": torch.zeros(3, 4, 64)}, TypeError, "key_pages must be torch.float32"),
    ({"dim": 60}, ValueError, "multiple of 8"),
    ({"dim": 264}, ValueError, "multiple of 8"),
    ({"lengths": torch.ones(3, dtype=torch.int64)}, TypeError, "lengths must be torch.int32"),
    ({"block_table": torch.zeros(3, 2)}, TypeError, "block_table must be torch.int32"),
    ({"block_table": torch.zeros(4, 2, dtype=I32)}, ValueError, "3 rows"),
    ({"value_pages": torch.zeros(5, 8, 2, 64, dtype=B)}, ValueError, "value_pages must have the shape"),
    ({"key_pages": torch.zeros(5, 16, 2, 68, dtype=B)[..., :64]}, ValueError, "16-byte"),
    ({"value_pages": torch.zeros(5 * 16 * 2 * 64 + 1, dtype=B)[1:].view(5, 16, 2, 64)}, ValueError, "16-byte"),
    ({"window": 0}, ValueError, "window"),
    ({"out": torch.zeros(3, 4, 64)}, TypeError, "out must be"),
    ({"out": torch.zeros(3, 1, 64, dtype=B).expand(3, 4, 64)}, ValueError, "overlap"),
    ({"query": torch.zeros(3, 4, 64, dtype=B, requires_grad=True)}, RuntimeError, "no_grad"),
])
def test_attention_refusals(change, error, match):
    with pytest.raises(error, match=match):
        paged.paged_attention(**_attention_args(**change))


@pytest.mark.parametrize("out", ["query_out", "key_out"])
def test_rotary_refuses_outputs_that_need_a_gradient(out):
    shape = (5, 4 if out == "query_out" else 2, 64)
    with pytest.raises(RuntimeError, match="no_grad"):
        paged.rotary_store(**_rotary_args(**{out: torch.zeros(shape, dtype=B, requires_grad=True)}))


def test_rotary_refuses_a_table_that_needs_a_gradient():
    with pytest.raises(RuntimeError, match="no_grad"):
        paged.rotary_store(**_rotary_args(rotary=torch.zeros(9, 64, requires_grad=True)))


def test_attention_refuses_an_output_that_needs_a_gradient():
    with pytest.raises(RuntimeError, match="no_grad"):
        paged.paged_attention(**_attention_args(out=torch.zeros(3, 4, 64, dtype=B, requires_grad=True)))


@pytest.mark.parametrize("name", ["query", "key", "value", "rotary", "key_pages", "value_pages", "query_norm", "key_norm"])
def test_rotary_refuses_dual_tensors(name):
    args = _rotary_args(query_norm=torch.ones(64, dtype=B), key_norm=torch.ones(64, dtype=B))
    with forward_ad.dual_level(), torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
        paged.rotary_store(**{**args, name: forward_ad.make_dual(args[name], torch.ones_like(args[name]))})


@pytest.mark.parametrize("name", ["query", "key_pages", "value_pages", "out"])
def test_attention_refuses_dual_tensors(name):
    args = _attention_args(out=torch.zeros(3, 4, 64, dtype=B))
    with forward_ad.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
        paged.paged_attention(**{**args, name: forward_ad.make_dual(args[name], torch.ones_like(args[name]))})
    with forward_ad.dual_level(), pytest.raises(ValueError, match="CUDA device"):  # others are as they were
        paged.paged_attention(**args)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rot", [0, 2, 6, 8])
def test_oracle_of_many_rows_is_the_oracle(interleaved, rot):
    g = torch.Generator().manual_seed(rot)
    x, rotary, norm = (torch.randn(shape, generator=g) for shape in ((5, 3, 8), (7, rot), (8,)))
    positions, slots = torch.tensor([0, 6, 7, -1, 3]), torch.tensor([4, -1, 0, 8, 2])
    for weights in (None, norm):
        rows = oracle.rotated(x, positions, rotary, interleaved, weights)
        many = oracle.rotated_many(x, positions, rotary, interleaved, weights)
        assert torch.allclose(rows, many, rtol=1e-14, atol=1e-14, equal_nan=True)
        pages = torch.randn(2, 4, 3, 8, generator=g)
        assert torch.equal(oracle.stored(pages, rows, slots).nan_to_num(9.0),
                           oracle.stored_many(pages, rows, slots).nan_to_num(9.0))


def test_numbers_out_of_range():
    with pytest.raises(ValueError, match="float32"):
        paged._number("scale", 1e39)
    with pytest.raises(TypeError, match="a number"):
        paged._number("scale", "1")


def test_native_refusals():
    """The C entry points check their own sizes and pointers before any CUDA call."""
    lib = _native.load()
    for struct, name, bad in (
            (_native.Reserve, "nz_pages_reserve", [{}, {"requests": 4097}, {"requests": 1}, {"page_shift": 21},
                                                  {"requests": 1, "rows": 2 ** 31}, {"requests": 1, "pages": 2 ** 30}]),
            (_native.Release, "nz_pages_release", [{}, {"requests": 4097}, {"requests": 1}, {"requests": 1, "width": 2 ** 31}]),
            (_native.Rotary, "nz_rotary_store", [{}, {"dim": 258}, {"dim": 64, "rot": 66}, {"dim": 63},
                                                 {"dim": 64, "tokens": 1, "heads": 1}, {"dim": 64, "heads": 65537},
                                                 {"dim": 64, "tokens": 2 ** 31, "heads": 2}]),
            (_native.Attention, "nz_paged_attention", [{}, {"dim": 264}, {"dim": 64}, {"dim": 64, "heads": 3, "kv_heads": 2},
                                                       {"dim": 64, "heads": 2, "kv_heads": 2, "requests": 4097},
                                                       {"dim": 64, "heads": 2, "kv_heads": 2, "requests": 1},
                                                       {"dim": 64, "heads": 2, "kv_heads": 2, "requests": 1, "query": 16,
                                                        "out": 16, "lengths": 16, "pages": 1, "key_pages": 24,
                                                        "value_pages": 32}])):
        assert getattr(lib, name)(None, None) == _native.EVALUE
        for fields in bad:
            args = struct(**fields)
            assert getattr(lib, name)(ctypes.byref(args), None) == _native.EVALUE, (name, fields)


def test_struct_layouts_match_header(tmp_path):
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    probe = tmp_path / "probe.c"
    pairs = (("nz_reserve", _native.Reserve), ("nz_release", _native.Release), ("nz_rotary", _native.Rotary),
             ("nz_attention", _native.Attention))
    lines = [f'printf("%zu ", sizeof({name}));' for name, _ in pairs]
    want = [ctypes.sizeof(struct) for _, struct in pairs]
    for name, struct in pairs:
        for field, _kind in struct._fields_:
            lines.append(f'printf("%zu ", offsetof({name}, {field}));')
            want.append(getattr(struct, field).offset)
    probe.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "nz_b200.h"\nint main(void){' + "\n".join(lines)
                     + "return 0;}\n")
    subprocess.run([cc, f"-I{ROOT / 'include'}", str(probe), "-o", str(tmp_path / "probe")], check=True)
    got = subprocess.run([str(tmp_path / "probe")], capture_output=True, text=True, check=True).stdout.split()
    assert [int(x) for x in got] == want
