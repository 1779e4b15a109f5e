"""Refusals of the paged-cache entry points, without GPU work, and the CPU statements the
GPU tests compare with."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import paged_oracle as PO
from polyhedral_b200 import _lib, paged

PTR = ctypes.c_void_p(256)


@pytest.fixture(scope="module")
def lib():
    from polyhedral_b200 import build
    build.build()
    return _lib.load()


def _fields(header_name):
    from tests.test_capi import _struct_fields
    return _struct_fields(header_name)


@pytest.mark.parametrize("cname,pyname", [("pa_paged_step_args", "PaPagedStepArgs"),
                                          ("pa_paged_append_args", "PaPagedAppendArgs")])
def test_struct_layout_matches_header(cname, pyname):
    assert _fields(cname) == [f[0] for f in getattr(_lib, pyname)._fields_]


def _step_args():
    a = _lib.PaPagedStepArgs()
    for name, kind in a._fields_:
        if kind is _lib.c_vp:
            setattr(a, name, 256)
    a.free_head_out = 512
    a.requests, a.page_size, a.table_width, a.tokens, a.free_count, a.table_stride = 4, 16, 8, 4, 9, 8
    return a


@pytest.mark.parametrize("field,value,word", [
    ("requests", 0, b"requests=0"), ("requests", 16385, b"requests=16385"),
    ("page_size", 0, b"page_size=0"), ("table_width", 0, b"table_width=0"),
    ("tokens", -1, b"tokens=-1"), ("free_count", -1, b"free_count=-1"),
    ("table_stride", 7, b"table_stride=7"), ("old_lens", None, b"null"),
    ("slot_map", None, b"null"), ("free_head_out", 256, b"free_head_out")])
def test_step_refusals(lib, field, value, word):
    a = _step_args()
    setattr(a, field, value)
    assert lib.pa_paged_step(ctypes.byref(a), None) == _lib.PA_ERR_ARG
    assert word in lib.pa_last_error()


def _append_args():
    a = _lib.PaPagedAppendArgs()
    for name, kind in a._fields_:
        setattr(a, name, 256 if kind is _lib.c_vp else 64)
    a.D, a.kv_heads = 64, 2
    return a


@pytest.mark.parametrize("field,value,word", [
    ("D", 12, b"D=12"), ("D", 0, b"D=0"), ("kv_heads", 0, b"kv_heads=0"), ("pages", 0, b"pages=0"),
    ("page_size", 0, b"page_size=0"), ("k", None, b"null"), ("k", 264, b"16-byte aligned"),
    ("k_token_stride", 12, b"multiples of 8"), ("vc_head_stride", 1, b"multiples of 8"),
    ("pages", 1 << 30, b"32 bits"), ("tokens", -1, b"tokens=-1")])
def test_append_refusals(lib, field, value, word):
    a = _append_args()
    setattr(a, field, value)
    assert lib.pa_paged_append(ctypes.byref(a), None) == _lib.PA_ERR_ARG
    assert word in lib.pa_last_error()


def test_python_layer_refuses_without_gpu_work():
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="GPU only"):
        paged.make_step(torch.zeros(2, 4, dtype=torch.int32), i, i, i, i[:1], page_size=16, tokens=2)
    with pytest.raises(ValueError, match="requests, width"):
        paged.make_step(i, i, i, i, i[:1], page_size=16, tokens=2)
    k = torch.zeros(2, 1, 64, dtype=torch.bfloat16)
    c = torch.zeros(2, 16, 1, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="GPU only"):
        paged.append_kv(k, k, c, c, i)
    with pytest.raises(ValueError, match="kv_heads, D"):
        paged.append_kv(k, k[:1], c, c, i)
    with pytest.raises(ValueError, match="share shape"):
        paged.append_kv(k, k, c, c[:1], i)


def test_statement_of_the_tables():
    """By hand: pages of 4; request 0 has 3 tokens and gets 2, request 1 none and 5."""
    table = np.array([[7, -1, -1], [-1, -1, -1]])
    t, qs, lens, slots, pos, head, missing = PO.step_tables(table, [3, 0], [2, 5], [2, 9, 4, 6], 1, 4, 8)
    assert t.tolist() == [[7, 9, -1], [4, 6, -1]]
    assert (qs, lens, head, missing) == ([0, 2, 7], [5, 5], 4, 0)
    assert slots == [31, 36, 16, 17, 18, 19, 24, -1] and pos == [3, 4, 0, 1, 2, 3, 4, -1]
    t, _, _, slots, _, head, missing = PO.step_tables(table, [3, 0], [2, 5], [2, 9], 1, 4, 8)
    assert t.tolist() == [[7, 9, -1], [-1, -1, -1]] and (head, missing) == (2, 2)
    assert slots == [31, 36, -1, -1, -1, -1, -1, -1]
