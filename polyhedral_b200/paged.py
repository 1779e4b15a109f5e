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

There are no gradients: these serve.  Everything is stream-ordered and nothing is read
back by the host, so a step of fixed shapes can be captured in a CUDA graph.  The reference
has no counterpart.
"""
import functools

import torch

from . import _lib

_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)

_DTYPES = {torch.bfloat16: _lib.PA_BF16, torch.float16: _lib.PA_F16}

_pack_step = _lib.packer(_lib.PaPagedStepArgs)
_pack_append = _lib.packer(_lib.PaPagedAppendArgs)
_pack_attn = _lib.packer(_lib.PaPagedAttnArgs)


def _launch(name, device, *args):
    """Call a C-ABI entry point on CUDA device number `device` and torch's current stream of
    it, as ``_lib.call`` does, in less host time."""
    lib = _lib.load()
    stream = _raw_stream(device) if _raw_stream else _lib.stream_handle(device)
    if _current_device() == device:
        rc = getattr(lib, name)(*args, stream)
    else:
        with torch.cuda.device(device):
            rc = getattr(lib, name)(*args, stream)
    if rc:
        raise _lib.PolyattnError(name, rc, lib.pa_last_error().decode(errors="replace"))


def _bad_int32(name, t, shape, device):
    if not isinstance(t, torch.Tensor) or t.dtype != torch.int32:
        raise TypeError(f"{name} must be an int32 tensor")
    if t.shape != shape:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {shape}")
    if t.get_device() != device:
        raise ValueError(f"{name} is on {t.device}, expected cuda:{device}")
    raise ValueError(f"{name} must be contiguous")


def _int32(name, t, n, device):
    """Address of an int32 tensor [n] on CUDA device number `device`."""
    if (not isinstance(t, torch.Tensor) or t.dtype is not torch.int32 or t.dim() != 1
            or t.numel() != n or t.get_device() != device or not t.is_contiguous()):
        _bad_int32(name, t, (n,), device)
    return t.data_ptr()


def _table(t, who, device=None):
    """(requests, width, row stride) of a block table."""
    if not isinstance(t, torch.Tensor) or t.dim() != 2:
        raise ValueError("block_table must be a [requests, width] tensor")
    if not t.is_cuda:
        raise RuntimeError(f"{who} runs on the GPU only")
    if t.dtype is not torch.int32:
        raise TypeError("block_table must be an int32 tensor")
    B, width = t.shape
    row, col = t.stride()
    if col != 1 and width > 1:
        raise ValueError("block_table: last dimension must be contiguous")
    if device is not None and t.get_device() != device:
        raise ValueError(f"block_table is on {t.device}, expected cuda:{device}")
    return B, width, row


class PagedStep:
    """What one step needs besides its activations, on the GPU (``make_step``):
    ``q_start`` [requests + 1] (first new token of every request, and their number),
    ``seq_lens`` [requests] (tokens after the step), ``slot_map`` and ``positions``
    [tokens] (-1 behind the last new token; a slot is -1 too where no page could be
    had), ``free_head`` [1] (pages of the free list taken so far: the next step's
    ``free_head``) and ``missing`` [1] (pages that could not be had)."""

    __slots__ = ("q_start", "seq_lens", "slot_map", "positions", "free_head", "missing",
                 "requests", "tokens", "device")

    def __init__(self, requests, tokens, device):
        buf = torch.empty(2 * requests + 2 * tokens + 3, dtype=torch.int32, device=device)
        (self.q_start, self.seq_lens, self.slot_map, self.positions, self.free_head,
         self.missing) = buf.split_with_sizes((requests + 1, requests, tokens, tokens, 1, 1))
        self.requests, self.tokens, self.device = requests, tokens, buf.get_device()


def make_step(block_table, old_lens, new_lens, free_pages, free_head, *, page_size, tokens,
              out=None):
    """Tables of one step from the requests' lengths, in one launch.

    ``block_table`` [requests, width] int32 is updated in place: a request whose
    ``old_lens + new_lens`` tokens need more pages gets them from ``free_pages``, from entry
    ``free_head`` [1] on, requests in order; no other entry is touched.  ``tokens`` is the
    capacity of the slot map (at least the sum of ``new_lens``).  ``out`` (a
    ``PagedStep`` of the same sizes) is filled instead of a new one; none of its tensors may
    be an argument too (the next step's ``old_lens`` is this one's ``seq_lens``: use two
    in turn).  All arguments are int32 tensors on one CUDA device; at most
    16384 requests, of at most 2**31 - 1 tokens each (those behind have no slot and no
    position)."""
    B, width, row = _table(block_table, "make_step")
    dev = block_table.get_device()
    if tokens < 0:
        raise ValueError(f"tokens={tokens} is negative")
    old = _int32("old_lens", old_lens, B, dev)
    new = _int32("new_lens", new_lens, B, dev)
    n_free = free_pages.numel()
    free = _int32("free_pages", free_pages, n_free, dev)
    head = _int32("free_head", free_head, 1, dev)
    st = out
    if st is None:
        st = PagedStep(B, tokens, block_table.device)
    elif st.requests != B or st.tokens != tokens:
        raise ValueError("out was made for other sizes")
    elif st.device != dev:
        raise ValueError(f"out is on cuda:{st.device}, expected cuda:{dev}")
    args = _pack_step(B, page_size, width, tokens, n_free, row, old, new, free, head,
                      block_table.data_ptr(), st.q_start.data_ptr(), st.seq_lens.data_ptr(),
                      st.slot_map.data_ptr(), st.positions.data_ptr(), st.free_head.data_ptr(),
                      st.missing.data_ptr())
    _launch("pa_paged_step", dev, args)
    return st


def _caches(k_cache, v_cache):
    """Shapes and strides of a pair of caches: (shape, k strides, v strides)."""
    if k_cache.dim() != 4 or v_cache.dim() != 4:
        raise ValueError("k_cache and v_cache must be [pages, page_size, kv_heads, D]")
    shape, ks, vs = k_cache.shape, k_cache.stride(), v_cache.stride()
    if (v_cache.shape != shape or v_cache.dtype is not k_cache.dtype
            or v_cache.get_device() != k_cache.get_device()):
        raise ValueError("k_cache and v_cache must share shape, dtype and device")
    if ks[3] != 1 or vs[3] != 1:
        raise ValueError("k_cache and v_cache: last dimension must be contiguous")
    return shape, ks, vs


def append_kv(k, v, k_cache, v_cache, slot_map):
    """Write the new rows k, v [tokens, kv_heads, D] into the caches [pages, page_size,
    kv_heads, D] at ``slot_map`` [tokens] (int32; slots outside the cache, such as -1,
    are skipped).  bf16 or fp16; all on one CUDA device.  Two tokens of one call must not
    share a slot."""
    if k.dim() != 3 or v.shape != k.shape:
        raise ValueError("k and v must share shape [tokens, kv_heads, D]")
    (pages, page_size, H, D), ks, vs = _caches(k_cache, v_cache)
    if not (k.is_cuda and k_cache.is_cuda):
        raise RuntimeError("append_kv runs on the GPU only")
    if k.dtype not in _DTYPES or v.dtype is not k.dtype or k_cache.dtype is not k.dtype:
        raise TypeError(f"k, v and the caches must share dtype bf16 or fp16, got "
                        f"{k.dtype}/{v.dtype}/{k_cache.dtype}")
    T = k.shape[0]
    if k.shape != (T, H, D):
        raise ValueError(f"rows of {tuple(k.shape[1:])} do not fit a cache of "
                         f"{tuple(k_cache.shape)}")
    dev = k_cache.get_device()
    if k.get_device() != dev or v.get_device() != dev:
        raise ValueError("k, v and the caches must be on one device")
    kt, kh, k1 = k.stride()
    vt, vh, v1 = v.stride()
    if T and (k1 != 1 or v1 != 1):
        raise ValueError("k and v: last dimension must be contiguous")
    args = _pack_append(k.data_ptr(), v.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
                        _int32("slot_map", slot_map, T, dev), T, H, D, pages, page_size,
                        kt, kh, vt, vh, ks[0], ks[1], ks[2], vs[0], vs[1], vs[2])
    _launch("pa_paged_append", dev, args)


def _plan_args(head, tail, seq_lens, q_start):
    """Arguments of the plan's calls: there is no table yet, lengths are what seq_lens says."""
    B, T, H, Hkv, D, page, max_new, max_len = head
    return _pack_attn(0, 0, 0, 0, 0, 0, seq_lens, q_start, B, T, H, Hkv, D, 0, 0, page,
                      2**24 // page if page > 0 else 1, max_new, max_len, 0, 0, 0, 0, 0, 0, 0, 0, 0,
                      0, 0, 0, *tail, 0.0)


@functools.lru_cache(maxsize=256)
def _plan_sizes(head, device):
    """Bytes of a plan and of one call's scratch for these sizes on that device (they follow
    from the sizes and the number of multiprocessors)."""
    lib = _lib.load()
    args = _plan_args(head, (0, 0, 0, 0), 256, 256)
    with _lib.on_device(device):
        return max(lib.pa_paged_plan_size(args), 256), lib.pa_paged_scratch_size(args)


class PagedPlan:
    """Shares of work of one step's attention (``make_plan``): the same for every layer, and
    only read by the forwards (but for a status word, which a failure sets), so they may run on
    several streams.  It keeps the ``seq_lens`` and ``q_start`` it was built from; a forward
    that is given other lengths reports it (``status``)."""

    __slots__ = ("buffer", "nbytes", "scratch_bytes", "key", "head", "tail", "device",
                 "seq_lens", "q_start")

    def __init__(self, seq_lens, q_start, head, tail, key, device):
        self.seq_lens, self.q_start, self.key = seq_lens, q_start, key
        self.head, self.tail, self.device = head, tail, device
        self.nbytes, self.scratch_bytes = _plan_sizes(head, device)
        self.buffer = torch.empty(self.nbytes, dtype=torch.uint8, device=seq_lens.device)
        _launch("pa_paged_plan", device,
                _plan_args(head, tail, seq_lens.data_ptr(), q_start.data_ptr()),
                self.buffer.data_ptr(), self.nbytes)

    def status(self):
        """Device status of the forwards on this plan so far (synchronises): 0,
        ``_lib.DEV_OTHER_LENGTHS`` where one was given other lengths than the plan was built
        from, or the code of a bounded wait that ran out."""
        return _lib.device_status("pa_paged_status", self.buffer)


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
    B, dev = seq_lens.numel(), seq_lens.get_device()
    _int32("seq_lens", seq_lens, B, dev)
    _int32("q_start", q_start, B + 1, dev)
    return PagedPlan(seq_lens, q_start,
                     (B, tokens, heads, kv_heads, head_dim, page_size, max_new, max_len),
                     (kind, p0, p1, p2),
                     (B, tokens, heads, kv_heads, head_dim, page_size, kind, p0, p1, p2), dev)


def paged_attention(q, k_cache, v_cache, block_table, seq_lens, q_start, kind, p0, p1, p2,
                    scale=None, *, plan=None, return_lse=False, out=None, lse_out=None,
                    max_new=0, max_len=0, check=False):
    """Attention of every request's new tokens over its paged cache, which holds their
    keys and values already (``append_kv``).

    q: [tokens, heads, D] (bf16 or fp16, D in {64, 128}), the new tokens of request b in rows
    ``q_start[b]`` to ``q_start[b + 1]``, at its last positions; the caches [pages,
    page_size, kv_heads, D] (page_size a power of two in [16, 1024]; heads a multiple of
    kv_heads, at most 128 times); ``block_table`` [requests, width], ``seq_lens`` [requests],
    ``q_start`` [requests + 1] int32.  ``kind, p0, p1, p2`` is the mask on positions
    (``masks_gpu``): any of the framework's.  Returns o like q, or (o, lse) with lse [heads,
    tokens] fp32 (natural log); a token that sees no key gets o = 0, lse = -inf; rows of no
    request are not written.  Cache rows that the mask hides from a token, and those behind a
    request's last token, take no part whatever they hold; table entries outside the cache
    hold no keys.

    ``plan`` is ``make_plan``'s for these lengths and this mask; without one it is built
    first (``max_new`` / ``max_len`` as there).  The plan of another step gives wrong results
    and is reported: ``check`` or ``plan.status()`` shows it.  ``out`` / ``lse_out`` are written
    in place of new tensors and overlap no input; but ``out`` may be ``q``.  ``check``
    synchronises and raises if the kernel reported a failure."""
    if q.dim() != 3:
        raise ValueError("q must be [tokens, heads, D]")
    (pages, page_size, Hkv, Dc), ks, vs = _caches(k_cache, v_cache)
    dev = k_cache.get_device()
    dtype = q.dtype
    if not (q.is_cuda and k_cache.is_cuda):
        raise RuntimeError("paged_attention runs on the GPU only")
    if dtype not in _DTYPES or k_cache.dtype is not dtype:
        raise TypeError(f"q and the caches must share dtype bf16 or fp16, got "
                        f"{dtype}/{k_cache.dtype}")
    T, H, D = q.shape
    qt, qh, q1 = q.stride()
    if Dc != D or Hkv < 1 or H % Hkv:
        raise ValueError(f"q of {H} heads of {D} does not fit a cache of {Hkv} heads of {Dc}")
    if q.get_device() != dev:
        raise ValueError("q, block_table and the caches must be on one device")
    if T and q1 != 1:
        raise ValueError("q: last dimension must be contiguous")
    B, width, row = _table(block_table, "paged_attention", dev)
    lens_ptr = _int32("seq_lens", seq_lens, B, dev)
    start_ptr = _int32("q_start", q_start, B + 1, dev)
    if plan is None:
        plan = make_plan(seq_lens, q_start, kind, p0, p1, p2, tokens=T, heads=H, kv_heads=Hkv,
                         head_dim=D, page_size=page_size, max_new=max_new, max_len=max_len)
    elif plan.key != (B, T, H, Hkv, D, page_size, kind, p0, p1, p2):
        raise ValueError("plan was built for other sizes or another mask")
    elif plan.device != dev:
        raise ValueError(f"plan is on cuda:{plan.device}, expected cuda:{dev}")
    device = q.device
    if out is None:
        o = torch.empty(T, H, D, dtype=dtype, device=device)
        ot, oh = H * D, D
    else:
        o = out
        if o.shape != q.shape or o.dtype is not dtype or o.get_device() != dev:
            raise ValueError("out must be like q")
        ot, oh, o1 = o.stride()
        if T and o1 != 1:
            raise ValueError("out: last dimension must be contiguous")
    lse, lse_ptr, lse_row = lse_out, 0, 0
    if lse is not None:
        if lse.shape != (H, T) or lse.dtype is not torch.float32 or lse.get_device() != dev:
            raise ValueError("lse_out must be fp32 [heads, tokens]")
        lse_row, l1 = lse.stride()
        if T > 1 and l1 != 1:
            raise ValueError("lse_out: last dimension must be contiguous")
        lse_ptr = lse.data_ptr()
    elif return_lse:
        lse = torch.empty(H, T, dtype=torch.float32, device=device)
        lse_row, lse_ptr = T, lse.data_ptr()
    head, scratch, nbytes, scratch_ptr = plan.head, None, plan.scratch_bytes, 0
    if nbytes:
        scratch = torch.empty(nbytes, dtype=torch.uint8, device=device)
        scratch_ptr = scratch.data_ptr()
    args = _pack_attn(q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), o.data_ptr(), lse_ptr,
                      block_table.data_ptr(), lens_ptr, start_ptr, B, T, H, Hkv, D, _DTYPES[dtype],
                      pages, page_size, width, head[6], head[7], row, qt, qh, ks[0], ks[1], ks[2], vs[0],
                      vs[1], vs[2], ot, oh, lse_row, kind, p0, p1, p2, scale or 0.0)
    _launch("pa_paged_attn", dev, args, plan.buffer.data_ptr(), plan.nbytes, scratch_ptr, nbytes)
    if check:
        st = plan.status()
        if st:
            raise _lib.PolyattnError("pa_paged_attn", _lib.PA_ERR_DEVICE,
                                     f"device status {st} (" +
                                     ("the plan was built from other lengths"
                                      if st == _lib.DEV_OTHER_LENGTHS else
                                      "a bounded wait ran out") + ")")
    return (o, lse) if return_lse else o
