"""Serving over a paged K/V cache: the tables of a step, the cache's new rows, and the
attention of every request's new tokens under the framework's masks.

A cache is a pair of tensors [pages, page_size, kv_heads, D]; a request's token at
position p lies in row ``p % page_size`` of page ``block_table[request, p // page_size]``,
and its *slot* is ``page * page_size + row``.  One step of a serving loop:

    step = paged.make_step(block_table, old_lens, new_lens, free_pages, free_head,
                           page_size=P, tokens=T)
    plan = paged.make_plan(step.seq_lens, step.q_start, *mask.spec, tokens=T, ...)
    for layer in layers:
        paged.append_kv(k, v, k_cache, v_cache, step.slot_map)
        o = paged.paged_attention(q, k_cache, v_cache, block_table, step.seq_lens,
                                  step.q_start, *mask.spec, plan=plan)
    free_head = step.free_head

Everything is stream-ordered and nothing is read back by the host, so a step of fixed
shapes can be captured in a CUDA graph.  The reference has no counterpart.
"""
import ctypes

import torch

from . import _lib

_DTYPES = {torch.bfloat16: _lib.PA_BF16, torch.float16: _lib.PA_F16}


def _int32(name, t, shape, device):
    if not isinstance(t, torch.Tensor) or t.dtype != torch.int32:
        raise TypeError(f"{name} must be an int32 tensor")
    if t.shape != shape:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return t.data_ptr()


class PagedStep:
    """What one step needs besides its activations, on the GPU (``make_step``):
    ``q_start`` [requests + 1] (first new token of every request, and their number),
    ``seq_lens`` [requests] (tokens after the step), ``slot_map`` and ``positions``
    [tokens] (-1 behind the last new token; a slot is -1 too where no page could be
    had), ``free_head`` [1] (pages of the free list taken so far: the next step's
    ``free_head``) and ``missing`` [1] (pages that could not be had)."""

    __slots__ = ("q_start", "seq_lens", "slot_map", "positions", "free_head", "missing")

    def __init__(self, requests, tokens, device):
        buf = torch.empty(2 * requests + 2 * tokens + 3, dtype=torch.int32, device=device)
        (self.q_start, self.seq_lens, self.slot_map, self.positions, self.free_head,
         self.missing) = buf.split([requests + 1, requests, tokens, tokens, 1, 1])


def make_step(block_table, old_lens, new_lens, free_pages, free_head, *, page_size, tokens,
              out=None):
    """Tables of one step from the requests' lengths, in one launch.

    ``block_table`` [requests, width] int32 is updated in place: a request whose
    ``old_lens + new_lens`` tokens need more pages gets them from ``free_pages``, from entry
    ``free_head`` [1] on, requests in order; no other entry is touched.  ``tokens`` is the
    capacity of the slot map (at least the sum of ``new_lens``).  ``out`` (a
    ``PagedStep`` of the same sizes) is filled instead of a new one; its ``free_head``
    must not be the one given.  All arguments are int32 tensors on one CUDA device."""
    if not isinstance(block_table, torch.Tensor) or block_table.dim() != 2:
        raise ValueError("block_table must be a [requests, width] tensor")
    if not block_table.is_cuda:
        raise RuntimeError("make_step runs on the GPU only")
    if block_table.dtype != torch.int32:
        raise TypeError("block_table must be an int32 tensor")
    B, width = block_table.shape
    if width > 1 and block_table.stride(1) != 1:
        raise ValueError("block_table: last dimension must be contiguous")
    dev, tokens = block_table.device, int(tokens)
    if tokens < 0:
        raise ValueError(f"tokens={tokens} is negative")
    a = _lib.PaPagedStepArgs()
    a.old_lens = _int32("old_lens", old_lens, (B,), dev)
    a.new_lens = _int32("new_lens", new_lens, (B,), dev)
    a.free_pages = _int32("free_pages", free_pages, (free_pages.numel(),), dev)
    a.free_head = _int32("free_head", free_head, (1,), dev)
    st = out
    if st is None:
        st = PagedStep(B, tokens, dev)
    elif st.seq_lens.shape[0] != B or st.slot_map.shape[0] != tokens:
        raise ValueError("out was made for other sizes")
    elif st.seq_lens.device != dev:
        raise ValueError(f"out is on {st.seq_lens.device}, expected {dev}")
    a.requests, a.page_size, a.table_width, a.tokens = B, int(page_size), width, tokens
    a.free_count, a.table_stride = free_pages.numel(), block_table.stride(0)
    a.block_table = block_table.data_ptr()
    a.q_start, a.seq_lens = st.q_start.data_ptr(), st.seq_lens.data_ptr()
    a.slot_map, a.positions = st.slot_map.data_ptr(), st.positions.data_ptr()
    a.free_head_out, a.missing = st.free_head.data_ptr(), st.missing.data_ptr()
    _lib.call("pa_paged_step", ctypes.byref(a), _lib.stream_handle(dev), device=dev)
    return st


def _check_cache(name, t, like=None):
    if t.dim() != 4:
        raise ValueError(f"{name} must be [pages, page_size, kv_heads, D]")
    if t.stride(3) != 1:
        raise ValueError(f"{name}: last dimension must be contiguous")
    if like is not None and (t.shape != like.shape or t.dtype != like.dtype
                             or t.device != like.device):
        raise ValueError("k_cache and v_cache must share shape, dtype and device")


def append_kv(k, v, k_cache, v_cache, slot_map):
    """Write the new rows k, v [tokens, kv_heads, D] into the caches [pages, page_size,
    kv_heads, D] at ``slot_map`` [tokens] (int32; slots outside the cache, such as -1,
    are skipped).  bf16 or fp16; all on one CUDA device.  Two tokens of one call must not
    share a slot."""
    if k.dim() != 3 or v.shape != k.shape:
        raise ValueError("k and v must share shape [tokens, kv_heads, D]")
    _check_cache("k_cache", k_cache)
    _check_cache("v_cache", v_cache, k_cache)
    if not (k.is_cuda and k_cache.is_cuda):
        raise RuntimeError("append_kv runs on the GPU only")
    if k.dtype not in _DTYPES or v.dtype != k.dtype or k_cache.dtype != k.dtype:
        raise TypeError(f"k, v and the caches must share dtype bf16 or fp16, got "
                        f"{k.dtype}/{v.dtype}/{k_cache.dtype}")
    T, H, D = k.shape
    if k_cache.shape[2] != H or k_cache.shape[3] != D:
        raise ValueError(f"rows of [{H}, {D}] do not fit a cache of {tuple(k_cache.shape)}")
    dev = k_cache.device
    if k.device != dev or v.device != dev:
        raise ValueError("k, v and the caches must be on one device")
    if T and (k.stride(2) != 1 or v.stride(2) != 1):
        raise ValueError("k and v: last dimension must be contiguous")
    a = _lib.PaPagedAppendArgs()
    a.slot_map = _int32("slot_map", slot_map, (T,), dev)
    a.k, a.v, a.k_cache, a.v_cache = (k.data_ptr(), v.data_ptr(), k_cache.data_ptr(),
                                      v_cache.data_ptr())
    a.tokens, a.kv_heads, a.D = T, H, D
    a.pages, a.page_size = k_cache.shape[0], k_cache.shape[1]
    a.k_token_stride, a.k_head_stride, _ = k.stride()
    a.v_token_stride, a.v_head_stride, _ = v.stride()
    a.kc_page_stride, a.kc_row_stride, a.kc_head_stride, _ = k_cache.stride()
    a.vc_page_stride, a.vc_row_stride, a.vc_head_stride, _ = v_cache.stride()
    _lib.call("pa_paged_append", ctypes.byref(a), _lib.stream_handle(dev), device=dev)
