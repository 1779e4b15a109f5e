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


class PagedPlan:
    """Shares of work of one step's attention (``make_plan``): the same for every layer,
    read by the forwards and never written, so they may run on several streams.  It
    keeps the ``seq_lens`` and ``q_start`` it was built from."""

    def __init__(self, args, seq_lens, q_start):
        self.args, self.seq_lens, self.q_start = args, seq_lens, q_start
        lib = _lib.load()
        nbytes = lib.pa_paged_plan_size(ctypes.byref(args))
        self.scratch_bytes = lib.pa_paged_scratch_size(ctypes.byref(args))
        self.buffer = torch.empty(max(nbytes, 1), dtype=torch.uint8, device=seq_lens.device)
        self.nbytes = nbytes
        # what a forward on this plan has to bring
        self.key = (args.tokens, args.heads, args.kv_heads, args.D, args.page_size,
                    args.pred.kind, args.pred.p0, args.pred.p1, args.pred.p2)
        _lib.call("pa_paged_plan", ctypes.byref(args), self.buffer.data_ptr(), nbytes,
                  _lib.stream_handle(seq_lens.device), device=seq_lens.device)

    def status(self):
        """Device status of the forwards on this plan so far (synchronises): 0, or the code
        of the bounded wait that ran out."""
        st = _lib.c_i32(0)
        with _lib.on_device(self.buffer.device):
            _lib.load().pa_paged_status(self.buffer.data_ptr(), ctypes.byref(st),
                                        _lib.stream_handle(self.buffer.device))
        return int(st.value)


def make_plan(seq_lens, q_start, kind, p0, p1, p2, *, tokens, heads, kv_heads, head_dim,
              page_size, max_new=0, max_len=0):
    """Share out the attention of one step among the GPU's multiprocessors, from the
    requests' lengths (``seq_lens`` [requests], ``q_start`` [requests + 1], int32 on the
    GPU, as ``make_step`` gives them) and the mask.  ``tokens`` is the number of rows of q.
    ``max_new`` / ``max_len`` are upper bounds on a request's new tokens / tokens, where the
    caller knows them (0: unknown): they choose the kernel, and whether work is split along
    the keys.  Build it once per step and pass it to every layer's ``paged_attention``."""
    if not isinstance(seq_lens, torch.Tensor) or seq_lens.dim() != 1:
        raise ValueError("seq_lens must be a [requests] tensor")
    if not seq_lens.is_cuda:
        raise RuntimeError("make_plan runs on the GPU only")
    B, dev = seq_lens.shape[0], seq_lens.device
    a = _lib.PaPagedAttnArgs()
    a.seq_lens = _int32("seq_lens", seq_lens, (B,), dev)
    a.q_start = _int32("q_start", q_start, (B + 1,), dev)
    a.requests, a.tokens, a.heads, a.kv_heads = B, int(tokens), int(heads), int(kv_heads)
    a.D, a.page_size = int(head_dim), int(page_size)
    a.table_width = max(2**24 // max(a.page_size, 1), 1)     # lengths are what seq_lens says
    a.max_new, a.max_len = int(max_new), int(max_len)
    a.pred = _lib.PaPred(int(kind), int(p0), int(p1), int(p2))
    return PagedPlan(a, seq_lens, q_start)


def paged_attention(q, k_cache, v_cache, block_table, seq_lens, q_start, kind, p0, p1, p2,
                    scale=None, *, plan=None, return_lse=False, out=None, lse_out=None,
                    max_new=0, max_len=0, check=False):
    """Attention of every request's new tokens over its paged cache, which holds their
    keys and values already (``append_kv``).

    q: [tokens, heads, D] (bf16 or fp16, D in {64, 128}), the new tokens of request b in rows
    ``q_start[b]`` to ``q_start[b + 1]``, at its last positions; the caches [pages,
    page_size, kv_heads, D] (page_size a power of two in [16, 1024]; heads a multiple of
    kv_heads); ``block_table`` [requests, width], ``seq_lens`` [requests], ``q_start``
    [requests + 1] int32.  ``kind, p0, p1, p2`` is the mask on positions (``masks_gpu``): any
    of the framework's.  Returns o like q, or (o, lse) with lse [heads, tokens] fp32 (natural
    log); a token that sees no key gets o = 0, lse = -inf; rows of no request are not
    written.  Cache rows that the mask hides from a token, and those behind a request's last
    token, take no part whatever they hold; table entries outside the cache hold no keys.

    ``plan`` is ``make_plan``'s for these lengths and this mask; without one it is built
    first (``max_new`` / ``max_len`` as there).  ``out`` / ``lse_out`` are written in place of
    new tensors.  ``check`` synchronises and raises if the kernel reported a failure."""
    if q.dim() != 3:
        raise ValueError("q must be [tokens, heads, D]")
    _check_cache("k_cache", k_cache)
    _check_cache("v_cache", v_cache, k_cache)
    dev = k_cache.device
    if not (q.is_cuda and k_cache.is_cuda):
        raise RuntimeError("paged_attention runs on the GPU only")
    if q.dtype not in _DTYPES or k_cache.dtype != q.dtype:
        raise TypeError(f"q and the caches must share dtype bf16 or fp16, got "
                        f"{q.dtype}/{k_cache.dtype}")
    T, H, D = q.shape
    pages, page_size, Hkv, Dc = k_cache.shape
    if Dc != D or Hkv < 1 or H % Hkv:
        raise ValueError(f"q of {H} heads of {D} does not fit a cache of {Hkv} heads of {Dc}")
    if q.device != dev or block_table.device != dev:
        raise ValueError("q, block_table and the caches must be on one device")
    if T and q.stride(2) != 1:
        raise ValueError("q: last dimension must be contiguous")
    B = seq_lens.shape[0]
    if block_table.dtype != torch.int32:
        raise TypeError("block_table must be an int32 tensor")
    if block_table.dim() != 2 or block_table.shape[0] != B:
        raise ValueError(f"block_table must be [{B}, width]")
    width = block_table.shape[1]
    if width > 1 and block_table.stride(1) != 1:
        raise ValueError("block_table: last dimension must be contiguous")
    lens_ptr = _int32("seq_lens", seq_lens, (B,), dev)
    start_ptr = _int32("q_start", q_start, (B + 1,), dev)
    if plan is None:
        plan = make_plan(seq_lens, q_start, kind, p0, p1, p2, tokens=T, heads=H, kv_heads=Hkv,
                         head_dim=D, page_size=page_size, max_new=max_new, max_len=max_len)
    elif plan.key != (T, H, Hkv, D, page_size, kind, p0, p1, p2) or plan.args.requests != B:
        raise ValueError("plan was built for other sizes or another mask")
    elif plan.buffer.device != dev:
        raise ValueError(f"plan is on {plan.buffer.device}, expected {dev}")
    o = out
    if o is None:
        o = torch.empty((T, H, D), dtype=q.dtype, device=dev)
    elif o.shape != q.shape or o.dtype != q.dtype or o.device != dev or (T and o.stride(2) != 1):
        raise ValueError("out must be like q, its last dimension contiguous")
    lse = lse_out
    if return_lse and lse is None:
        lse = torch.empty((H, T), dtype=torch.float32, device=dev)
    elif lse is not None and (lse.shape != (H, T) or lse.dtype != torch.float32
                              or lse.device != dev or (T > 1 and lse.stride(1) != 1)):
        raise ValueError("lse_out must be fp32 [heads, tokens], its last dimension contiguous")
    a = _lib.PaPagedAttnArgs.from_buffer_copy(plan.args)
    a.q, a.k_cache, a.v_cache, a.o = (q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
                                      o.data_ptr())
    a.block_table, a.seq_lens, a.q_start = block_table.data_ptr(), lens_ptr, start_ptr
    a.dtype, a.pages, a.table_width = _DTYPES[q.dtype], pages, width
    a.table_stride = block_table.stride(0)
    a.q_token_stride, a.q_head_stride, _ = q.stride()
    a.k_page_stride, a.k_row_stride, a.k_head_stride, _ = k_cache.stride()
    a.v_page_stride, a.v_row_stride, a.v_head_stride, _ = v_cache.stride()
    a.o_token_stride, a.o_head_stride, _ = o.stride()
    if lse is not None:
        a.lse, a.lse_head_stride = lse.data_ptr(), lse.stride(0)
    a.scale = float(scale) if scale else 0.0
    scratch = None
    if plan.scratch_bytes:
        scratch = torch.empty(plan.scratch_bytes, dtype=torch.uint8, device=dev)
    _lib.call("pa_paged_attn", ctypes.byref(a), plan.buffer.data_ptr(), plan.nbytes,
              scratch.data_ptr() if scratch is not None else None, plan.scratch_bytes,
              _lib.stream_handle(dev), device=dev)
    if check:
        st = plan.status()
        if st:
            raise _lib.PolyattnError("pa_paged_attn", _lib.PA_ERR_DEVICE,
                                     f"device status {st} (a bounded wait ran out)")
    return (o, lse) if return_lse else o
