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
    for i, (name, kind) in enumerate(a._fields_):
        if kind is _lib.c_vp:
            setattr(a, name, 4096 * i)
    a.requests, a.page_size, a.table_width, a.tokens, a.free_count, a.table_stride = 4, 16, 8, 4, 9, 8
    return a


@pytest.mark.parametrize("field,value,word", [
    ("requests", 0, b"requests=0"), ("requests", 16385, b"requests=16385"),
    ("page_size", 0, b"page_size=0"), ("table_width", 0, b"table_width=0"),
    ("tokens", -1, b"tokens=-1"), ("free_count", -1, b"free_count=-1"),
    ("table_stride", 7, b"table_stride=7"), ("old_lens", None, b"null"),
    ("slot_map", None, b"null"), ("free_head_out", "free_head", b"free_head_out"),
    ("seq_lens", "old_lens", b"overlaps"), ("old_lens", "q_start", b"overlaps"),
    ("positions", "new_lens", b"overlaps"), ("free_pages", "block_table", b"overlaps")])
def test_step_refusals(lib, field, value, word):
    a = _step_args()
    # a name: the same memory as that argument's, from its second entry on
    same = getattr(a, value) if isinstance(value, str) else value
    if isinstance(value, str) and field != "free_head_out":
        same += 4
    setattr(a, field, same)
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


def _attn_args():
    a = _lib.PaPagedAttnArgs()
    for name, kind in a._fields_:
        if kind is _lib.c_vp:
            setattr(a, name, 256)
        elif kind is _lib.c_i64:
            setattr(a, name, 64)
    a.requests, a.tokens, a.heads, a.kv_heads, a.D, a.dtype = 3, 8, 4, 2, 64, 0
    a.pages, a.page_size, a.table_width = 10, 16, 4
    return a


def test_attn_struct_layout_and_packing():
    assert _fields("pa_paged_attn_args") == [f[0] for f in _lib.PaPagedAttnArgs._fields_]
    # packed bytes are the struct's
    a = _attn_args()
    a.pred = _lib.PaPred(5, 7, 8, 9)
    a.scale = 0.25
    vals = []
    for name, kind in a._fields_:
        v = getattr(a, name)
        vals += [getattr(v, f[0]) for f in v._fields_] if isinstance(v, ctypes.Structure) else [v]
    packed = _lib.packer(_lib.PaPagedAttnArgs)(*vals)
    assert bytes(a)[:len(packed)] == packed and len(bytes(a)) - len(packed) < 8


@pytest.mark.parametrize("field,value,word", [
    ("requests", 0, b"requests=0"), ("requests", 65537, b"requests=65537"), ("tokens", -1, b"tokens=-1"),
    ("tokens", 2**30, b"2^31"), ("heads", 5, b"multiple of kv_heads"), ("kv_heads", 0, b"kv_heads=0"),
    ("heads", 258, b"129 query heads"), ("D", 96, b"D=96"), ("dtype", 2, b"dtype 2"),
    ("page_size", 24, b"page_size=24"), ("page_size", 8, b"page_size=8"),
    ("page_size", 2048, b"page_size=2048"), ("max_new", -1, b"max_new=-1"), ("max_len", -2, b"max_len=-2"),
    ("seq_lens", None, b"null seq_lens"), ("pages", 0, b"pages=0"), ("pages", 2**28, b"32 bits"),
    ("table_width", 0, b"table_width=0"), ("table_width", 2**21, b"2^24 tokens"), ("q", None, b"null"),
    ("k_cache", 264, b"16-byte aligned"), ("o", 8, b"16-byte aligned"),
    ("k_page_stride", 12, b"multiples of 8"), ("q_head_stride", -64, b"multiples of 8")])
def test_attn_refusals(lib, field, value, word):
    a = _attn_args()
    setattr(a, field, value)
    rc = lib.pa_paged_attn(ctypes.byref(a), PTR, 1 << 30, PTR, 1 << 40, None)
    assert rc == _lib.PA_ERR_ARG
    assert word in lib.pa_last_error()


def test_attn_mask_refusals(lib):
    a = _attn_args()
    for pred, word in (((9, 0, 0, 0), b"unknown mask kind"), ((2, 0, 0, 0), b"DILATED"),
                       ((1, -1, 0, 0), b"WINDOW"), ((3, 5, 0, 0), b"LOCAL_STRIDED")):
        a.pred = _lib.PaPred(*pred)
        assert lib.pa_paged_plan(ctypes.byref(a), PTR, 1 << 30, None) == _lib.PA_ERR_ARG
        assert word in lib.pa_last_error()
        assert lib.pa_paged_attn(ctypes.byref(a), PTR, 1 << 30, PTR, 1 << 40, None) == _lib.PA_ERR_ARG


def test_attention_python_refusals():
    i = torch.zeros(2, dtype=torch.int32)
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16)
    c = torch.zeros(2, 16, 2, 64, dtype=torch.bfloat16)
    t = torch.zeros(2, 4, dtype=torch.int32)
    s = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="GPU only"):
        paged.paged_attention(q, c, c, t, i, s, 0, 0, 0, 0)
    with pytest.raises(RuntimeError, match="GPU only"):
        paged.make_plan(i, s, 0, 0, 0, 0, tokens=2, heads=4, kv_heads=2, head_dim=64, page_size=16)
    with pytest.raises(ValueError, match="tokens, heads, D"):
        paged.paged_attention(q[0], c, c, t, i, s, 0, 0, 0, 0)
    with pytest.raises(ValueError, match="pages, page_size"):
        paged.paged_attention(q, c[0], c, t, i, s, 0, 0, 0, 0)
    with pytest.raises(ValueError, match="share shape"):
        paged.paged_attention(q, c, c[:1], t, i, s, 0, 0, 0, 0)
    with pytest.raises(ValueError, match="last dimension"):
        paged.paged_attention(q, c.transpose(2, 3), c.transpose(2, 3), t, i, s, 0, 0, 0, 0)
    with pytest.raises(ValueError, match="requests"):
        paged.make_plan(s.view(3, 1), s, 0, 0, 0, 0, tokens=2, heads=4, kv_heads=2, head_dim=64,
                        page_size=16)


def test_statement_of_the_attention():
    """Against softmax over a gathered dense sequence, with a bad page left out."""
    g = torch.Generator().manual_seed(0)
    q = torch.randn(3, 2, 8, generator=g)
    kc, vc = torch.randn(4, 4, 1, 8, generator=g), torch.randn(4, 4, 1, 8, generator=g)
    table = torch.tensor([[2, 0, 7]])
    o, lse = PO.paged_attention(q, kc, vc, table, [10], [0, 3], 0, 0, 0, 0)
    k = torch.cat([kc[2], kc[0]])[:, 0].double()
    v = torch.cat([vc[2], vc[0]])[:, 0].double()
    for t in range(3):
        keys = min(8, 7 + t + 1)                # page 7 does not exist: keys 8, 9 are not there
        z = q[t].double() @ k[:keys].t() / 8**0.5
        assert torch.allclose(o[t], torch.softmax(z, 1) @ v[:keys])
        assert torch.allclose(lse[:, t], torch.logsumexp(z, 1))
