"""Serving over a paged K/V cache: the cases that are measured, their plain forms, and
the calls a user's program makes.

Four operators, the parts of one step of a serving loop:

  tables   block tables, slot map and positions of a step, built on the GPU from the
           requests' lengths
  append   the step's new K/V rows written into the paged cache by slot map
  attend   attention of every request's chunk of new tokens over its paged cache, with
           a causal mask, a sliding window, or a window and first tokens that stay
           visible (sinks)
  step     the three together, as a program runs them for one layer

``own`` False: ``run`` computes them with elementary torch operations; True: with the
framework's entry points.
"""
import math
import random

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# --------------------------------------------------------------------- cases
def _case(name, op, **kw):
    c = {"name": name, "op": op, "requests": 1, "new_lo": 1, "new_hi": 1, "old_lo": 0,
         "old_hi": 0, "page": 16, "heads": 32, "kv_heads": 8, "dim": 128, "dtype": "bf16",
         "mask": "causal", "window": 0, "sinks": 0}
    c.update(kw)
    return c


def listed():
    return [
        # one decode step of a small batch: the launch is all there is
        _case("tables: 8 requests decode", "tables", requests=8, old_lo=100, old_hi=2000),
        # a busy scheduler's step: many requests, chunks and single tokens mixed
        _case("tables: 1000 requests mixed", "tables", requests=1000, new_lo=1, new_hi=127,
              old_lo=0, old_hi=8000, page=32),
        # one decode step of a batch, one layer
        _case("append: 61 tokens", "append", requests=61, old_lo=17, old_hi=3000),
        # prefill chunks of several requests, one layer
        _case("append: 30011 tokens", "append", requests=11, new_lo=1, new_hi=5456, old_lo=0,
              old_hi=1000, page=64, dtype="fp16"),
        # a single user's next token, short context: latency
        _case("decode: 1 request", "attend", requests=1, old_lo=999, old_hi=999),
        # a server's decode batch, ragged contexts, small pages
        _case("decode: 64 requests", "attend", requests=64, old_lo=500, old_hi=8000),
        # few requests with very long contexts: work has to be split along the keys
        _case("decode: 4 long contexts", "attend", requests=4, old_lo=100001, old_hi=131071,
              page=64, heads=64, dtype="fp16"),
        # prefill chunks and single tokens in one batch, small heads
        _case("chunk: 24 requests mixed", "attend", requests=24, new_lo=1, new_hi=511, old_lo=0,
              old_hi=4001, page=32, heads=16, kv_heads=4, dim=64, dtype="fp16"),
        # a long prompt's next chunk: bound by the matrix products
        _case("chunk: 4096 over 16384", "attend", requests=1, new_lo=4096, new_hi=4096,
              old_lo=16384, old_hi=16384, page=128),
        # decode with a window of 1024 and 4 sinks: long contexts, few keys of each
        _case("sinks: 128 requests decode", "attend", requests=128, old_lo=900, old_hi=16383,
              mask="sinks", window=1024, sinks=4),
        # prefill chunks under the same mask, one key head per query head
        _case("sinks: 8 chunks of 2000", "attend", requests=8, new_lo=1900, new_hi=2100,
              old_lo=0, old_hi=8192, page=64, kv_heads=32, mask="sinks", window=1024, sinks=4),
        # tables, append and attention of a decode step, one layer
        _case("step: 32 requests decode", "step", requests=32, old_lo=200, old_hi=4000, page=32,
              mask="window", window=512),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["tables", "append", "attend", "attend", "attend", "attend", "step"])
    c = _case("", op)
    del c["name"]
    c["page"] = rng.choice([16, 32, 64, 128, 256])
    c["dim"] = rng.choice([64, 128])
    c["dtype"] = rng.choice(["bf16", "fp16"])
    c["kv_heads"] = rng.choice([1, 2, 3, 4, 5, 8, 16])
    c["heads"] = c["kv_heads"] * rng.choice([1, 2, 3, 4, 6, 7, 8])
    if op == "tables":
        c["requests"] = _log_int(rng, 1, 1000)
        c["new_hi"] = rng.choice([1, _log_int(rng, 1, 127)])
        c["old_hi"] = _log_int(rng, 1, 8000)
        return c
    if op == "append":
        tokens = _log_int(rng, 1, 30000)
        c["requests"] = _log_int(rng, 1, min(tokens, 100))
        c["new_hi"] = max(1, 2 * tokens // c["requests"] - 1)
        c["old_hi"] = _log_int(rng, 1, 1000)
        return c
    c["mask"] = rng.choice(["causal", "window", "sinks"])
    if c["mask"] != "causal":
        c["window"] = _log_int(rng, 16, 4096)
    if c["mask"] == "sinks":
        c["sinks"] = rng.choice([1, 4, 7, 16])
    if op == "step" or rng.random() < 0.5:          # decode, or a few tokens of each request
        c["requests"] = _log_int(rng, 1, 128)
        c["new_hi"] = c["new_lo"] = 1 if rng.random() < 0.7 else rng.randint(2, 4)
        most = 4_000_000 // (c["requests"] * c["kv_heads"])     # rows of keys held
        c["old_hi"] = _log_int(rng, 16, max(17, min(131071, most)))
        c["old_lo"] = c["old_hi"] // rng.choice([1, 2, 10])
        return c
    c["requests"] = _log_int(rng, 1, 24)             # chunks
    c["new_hi"] = _log_int(rng, 8, 4096)
    c["new_lo"] = rng.choice([1, c["new_hi"], max(1, c["new_hi"] // 2)])
    most = 2_000_000_000 // (c["requests"] * c["heads"] * c["new_hi"]) - c["new_hi"]
    c["old_hi"] = _log_int(rng, 1, max(2, min(32768, most)))
    c["old_lo"] = rng.choice([0, c["old_hi"]])
    # what the plain form holds of scores at once bounds the batch
    while c["requests"] * c["heads"] * c["new_hi"] * (c["new_hi"] + c["old_hi"]) > 2_600_000_000:
        c["new_hi"] = max(1, c["new_hi"] // 2)
        c["new_lo"] = min(c["new_lo"], c["new_hi"])
    return c


def _lengths(case):
    """(tokens already cached, new tokens) of every request: spread over the case's
    ranges, the same for every seed."""
    r = random.Random(7 * case["requests"] + case["new_hi"] + case["old_hi"])
    old = [r.randint(case["old_lo"], case["old_hi"]) for _ in range(case["requests"])]
    new = [r.randint(case["new_lo"], case["new_hi"]) for _ in range(case["requests"])]
    old[-1], new[-1] = case["old_hi"], case["new_hi"]
    return old, new


def _pages(n, page):
    return -(-n // page)


# --------------------------------------------------------------------- inputs
def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    old, new = _lengths(case)
    B, page, T = case["requests"], case["page"], sum(new)
    dt = _DTYPES[case["dtype"]]
    s = dict(case, tokens=T, max_new=max(new), max_len=max(o + n for o, n in zip(old, new)))
    s["scale"] = case["dim"] ** -0.5
    width = max(_pages(o + n, page) for o, n in zip(old, new)) + 2
    whole = sum(_pages(o + n, page) for o, n in zip(old, new))
    pages = whole + 5
    # the pages of all requests and the free ones, in the scattered order that a
    # running server's allocator leaves
    order = torch.randperm(pages, device=dev, generator=g).to(torch.int32)
    o_t, n_t = torch.tensor(old, device=dev), torch.tensor(new, device=dev)
    have = torch.div(o_t + page - 1, page, rounding_mode="floor")
    if case["op"] == "attend":                        # every page is in the table
        have = torch.div(o_t + n_t + page - 1, page, rounding_mode="floor")
    first = torch.cumsum(have, 0) - have
    col = torch.arange(width, device=dev)
    listed_ = col[None, :] < have[:, None]
    at = (first[:, None] + col[None, :]).clamp_(max=pages - 1)
    s["table"] = torch.where(listed_, order[at], torch.full_like(at, -1, dtype=torch.int32))
    used = int(have.sum())
    s["free"] = order
    s["head"] = torch.tensor([used], dtype=torch.int32, device=dev)
    s["old"], s["new"] = o_t.to(torch.int32), n_t.to(torch.int32)
    s["seq_lens"] = (o_t + n_t).to(torch.int32)
    s["q_start"] = torch.cat([n_t.new_zeros(1), torch.cumsum(n_t, 0)]).to(torch.int32)
    if case["op"] == "tables":
        return s
    shape = (pages, page, case["kv_heads"], case["dim"])
    s["k_cache"], s["v_cache"] = (torch.randn(shape, device=dev, generator=g, dtype=dt)
                                  for _ in range(2))
    if case["op"] != "attend":
        s["k"], s["v"] = (torch.randn((T,) + shape[2:], device=dev, generator=g, dtype=dt)
                          for _ in range(2))
    if case["op"] == "append":
        seq, pos = _places(s)
        page_of = order.long()[first[seq] + torch.div(pos, page, rounding_mode="floor")]
        fresh = pos >= (have * page)[seq]
        more = torch.div(o_t + n_t + page - 1, page, rounding_mode="floor") - have
        base = used + torch.cumsum(more, 0) - more
        extra = order.long()[(base[seq] + torch.div(pos, page, rounding_mode="floor")
                              - have[seq]).clamp(0, pages - 1)]
        s["slots"] = (torch.where(fresh, extra, page_of) * page + pos % page).to(torch.int32)
        return s
    s["q"] = torch.randn((T, case["heads"], case["dim"]), device=dev, generator=g, dtype=dt)
    if own and case["op"] == "attend":
        # the work list of a step: a program builds it once and keeps it for every layer
        s["plan"] = _plan(s, s["seq_lens"], s["q_start"])
    return s


def _places(s):
    """Request and position of every new token."""
    start = s["q_start"].long()
    t = torch.arange(s["tokens"], device=start.device)
    seq = torch.searchsorted(start[1:], t, right=True)
    return seq, s["old"].long()[seq] + t - start[seq]


# --------------------------------------------------------------------- the framework's calls
def _mask(s):
    from polyhedral_b200 import masks_gpu
    if s["mask"] == "causal":
        return masks_gpu.CAUSAL, 0, 0, 0
    if s["mask"] == "window":
        return masks_gpu.WINDOW, s["window"], 0, 0
    return masks_gpu.SINKS, s["window"], s["sinks"], 0


def _plan(s, seq_lens, q_start):
    from polyhedral_b200 import paged
    return paged.make_plan(seq_lens, q_start, *_mask(s), tokens=s["tokens"], heads=s["heads"],
                           kv_heads=s["kv_heads"], head_dim=s["dim"], page_size=s["page"],
                           max_new=s["max_new"], max_len=s["max_len"])


def _own_tables(s):
    from polyhedral_b200 import paged
    return paged.make_step(s["table"], s["old"], s["new"], s["free"], s["head"],
                           page_size=s["page"], tokens=s["tokens"])


def _own(s):
    from polyhedral_b200 import paged
    if s["op"] == "tables":
        st = _own_tables(s)
        return [s["table"], st.q_start, st.seq_lens, st.slot_map, st.positions, st.free_head,
                st.missing]
    if s["op"] == "append":
        paged.append_kv(s["k"], s["v"], s["k_cache"], s["v_cache"], s["slots"])
        return [s["k_cache"], s["v_cache"]]
    if s["op"] == "attend":
        return list(paged.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["table"],
                                          s["seq_lens"], s["q_start"], *_mask(s),
                                          scale=s["scale"], plan=s["plan"], return_lse=True))
    st = _own_tables(s)
    paged.append_kv(s["k"], s["v"], s["k_cache"], s["v_cache"], st.slot_map)
    plan = _plan(s, st.seq_lens, st.q_start)
    o, lse = paged.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], st.seq_lens,
                                   st.q_start, *_mask(s), scale=s["scale"], plan=plan,
                                   return_lse=True)
    return [s["table"], st.slot_map, s["k_cache"], s["v_cache"], o, lse]


# --------------------------------------------------------------------- plain forms
def _plain_tables(s):
    page, T = s["page"], s["tokens"]
    old, new, table = s["old"].long(), s["new"].long(), s["table"]
    B, width = table.shape
    dev = table.device
    have = torch.div(old + page - 1, page, rounding_mode="floor")
    need = torch.div(old + new + page - 1, page, rounding_mode="floor").clamp(max=width)
    more = (need - have).clamp(min=0)
    base = s["head"].long() + torch.cumsum(more, 0) - more
    col = torch.arange(width, device=dev)
    take = (col >= have[:, None]) & (col < need[:, None])
    at = (base[:, None] + col - have[:, None]).clamp(0, s["free"].numel() - 1)
    table.copy_(torch.where(take, s["free"][at], table))
    q_start = torch.cat([new.new_zeros(1), torch.cumsum(new, 0)])
    t = torch.arange(T, device=dev)
    seq = torch.searchsorted(q_start[1:], t, right=True)
    pos = old[seq] + t - q_start[seq]
    slot = table.long()[seq, torch.div(pos, page, rounding_mode="floor")] * page + pos % page
    head = s["head"].long() + more.sum()
    missing = torch.zeros(1, dtype=torch.int32, device=dev)
    return [table, q_start.int(), (old + new).int(), slot.int(), pos.int(), head.int(), missing]


def _plain_append(k, v, k_cache, v_cache, slots):
    at = slots.long()
    k_cache.view(-1, *k_cache.shape[2:])[at] = k
    v_cache.view(-1, *v_cache.shape[2:])[at] = v
    return [k_cache, v_cache]


def _plain_attend(s, seq_lens, q_start, table):
    """Every request padded to the longest chunk and to the most keys that a chunk can
    see; scores, softmax and products in 32 bits."""
    T, Hq, D = s["q"].shape
    Hkv, page, dev = s["kv_heads"], s["page"], s["q"].device
    G, B = Hq // Hkv, s["requests"]
    lens, start = seq_lens.long(), q_start.long()
    new = start[1:] - start[:-1]
    old = lens - new
    rows = torch.arange(s["max_new"], device=dev)
    row_ok = rows < new[:, None]                                             # [B, M]
    at = (start[:-1, None] + rows).clamp(max=T - 1)
    i = old[:, None] + rows                                                  # positions [B, M]
    if s["mask"] == "causal":
        j = torch.arange(s["max_len"], device=dev).expand(B, -1)
        key_ok = j < lens[:, None]
    else:                              # the sinks, then the keys that any new token sees
        lo = (old - s["window"] + 1).clamp(min=0)
        span = min(s["max_len"], s["window"] + s["max_new"] - 1)
        sink = torch.arange(s["sinks"], device=dev).expand(B, -1)
        band = lo[:, None] + torch.arange(span, device=dev)
        j = torch.cat([sink, band], 1)
        key_ok = torch.cat([sink < torch.minimum(lo, lens)[:, None], band < lens[:, None]], 1)
    jc = torch.where(key_ok, j, torch.zeros_like(j))
    page_of = torch.gather(table.long(), 1, torch.div(jc, page, rounding_mode="floor"))
    k = s["k_cache"][page_of, jc % page].float().masked_fill_(~key_ok[:, :, None, None], 0.0)
    q = s["q"][at].float().view(B, -1, Hkv, G, D).permute(0, 2, 3, 1, 4)     # [B, Hkv, G, M, D]
    x = torch.matmul(q.reshape(B, Hkv, -1, D), k.permute(0, 2, 3, 1))
    x = x.view(B, Hkv, G, -1, j.shape[1]).mul_(s["scale"])
    del k
    d = i[:, :, None] - j[:, None, :]
    live = (d >= 0) & key_ok[:, None, :]
    if s["mask"] == "window":
        live &= d < s["window"]
    elif s["mask"] == "sinks":
        live &= (d < s["window"]) | (j[:, None, :] < s["sinks"])
    x.masked_fill_(~live[:, None, None], float("-inf"))
    m = x.amax(-1, keepdim=True)
    m = torch.where(m == float("-inf"), torch.zeros_like(m), m)
    p = x.sub_(m).exp_()
    total = p.sum(-1, keepdim=True)
    v = s["v_cache"][page_of, jc % page].float().masked_fill_(~key_ok[:, :, None, None], 0.0)
    o = torch.matmul(p.view(B, Hkv, -1, j.shape[1]), v.permute(0, 2, 1, 3))
    o = o.view(B, Hkv, G, -1, D) / torch.where(total > 0, total, torch.ones_like(total))
    lse = (m + torch.log(total)).squeeze(-1)                                 # [B, Hkv, G, M]
    o = o.permute(0, 3, 1, 2, 4).reshape(B, -1, Hq, D)[row_ok]
    lse = lse.permute(0, 3, 1, 2).reshape(B, -1, Hq)[row_ok]
    return [o.to(s["q"].dtype), lse.t().contiguous()]


def run(state):
    s = state
    if own:
        return _own(s)
    if s["op"] == "tables":
        return _plain_tables(s)
    if s["op"] == "append":
        return _plain_append(s["k"], s["v"], s["k_cache"], s["v_cache"], s["slots"])
    if s["op"] == "attend":
        return _plain_attend(s, s["seq_lens"], s["q_start"], s["table"])
    table, q_start, seq_lens, slots = _plain_tables(s)[:4]
    caches = _plain_append(s["k"], s["v"], s["k_cache"], s["v_cache"], slots)
    return [table, slots] + caches + _plain_attend(s, seq_lens, q_start, table)


# --------------------------------------------------------------------- floors
def _seen(case, old, new):
    """(live query-key pairs, keys that some new token sees) of one request, per head."""
    w = case["window"] if case["mask"] != "causal" else old + new
    pairs = 0
    for i in range(old, old + new):
        near = min(i + 1, w)
        pairs += near + min(case["sinks"], i + 1 - near)
    lo = max(0, old - w + 1)
    return pairs, old + new - lo + min(case["sinks"], lo)


def work(case):
    old, new = _lengths(case)
    T, page = sum(new), case["page"]
    fresh = sum(_pages(o + n, page) - _pages(o, page) for o, n in zip(old, new))
    tables = 8 * case["requests"] + 8 * fresh + 8 * T + 8 * case["requests"]
    rows = 2 * T * case["kv_heads"] * case["dim"] * 2
    append = 2 * rows + 4 * T
    if case["op"] == "tables":
        return {"bytes": tables, "flops": 0}
    if case["op"] == "append":
        return {"bytes": append, "flops": 0}
    pairs = keys = 0
    for o, n in zip(old, new):
        a, b = _seen(case, o, n)
        pairs, keys = pairs + a, keys + b
    attend = (keys * case["kv_heads"] * case["dim"] * 4          # K and V rows
              + T * case["heads"] * (case["dim"] * 4 + 4)        # q, o, lse
              + 4 * _pages(keys, page))
    flops = 4 * case["dim"] * case["heads"] * pairs
    if case["op"] == "step":
        attend += tables + append
    return {"bytes": attend, "flops": flops}


# --------------------------------------------------------------------- 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] in ("tables", "append"):
        return None
    T, Hq, D = s["q"].shape
    page, Hkv = s["page"], s["kv_heads"]
    old, new = _lengths(case)
    kc, vc, table = s["k_cache"].clone(), s["v_cache"].clone(), s["table"].cpu()
    free = s["free"].cpu()
    nxt, t0 = int(s["head"].item()), 0
    o = torch.zeros(T, Hq, D, dtype=torch.float64, device=s["q"].device)
    lse = torch.zeros(Hq, T, dtype=torch.float64, device=s["q"].device)
    for b, (c, n) in enumerate(zip(old, new)):
        if s["op"] == "step":
            for x in range(_pages(c, page), _pages(c + n, page)):
                table[b, x] = free[nxt]
                nxt += 1
        pages = table[b, :_pages(c + n, page)].long().to(kc.device)
        for t in range(n if s["op"] == "step" else 0):
            at = pages[(c + t) // page]
            kc[at, (c + t) % page] = s["k"][t0 + t]
            vc[at, (c + t) % page] = s["v"][t0 + t]
        i = torch.arange(c, c + n, device=kc.device)[:, None]
        near = 0 if s["mask"] == "causal" else max(0, c + 1 - s["window"])
        j = torch.arange(c + n, device=kc.device)
        j = j[(j < s["sinks"]) | (j >= near)]                   # the others no row sees
        seen = j <= i
        if s["mask"] != "causal":
            seen &= (i - j < s["window"]) | (j < s["sinks"])
        for h in range(Hkv):
            kh = kc[pages, :, h].reshape(-1, D)[j].double()
            vh = vc[pages, :, h].reshape(-1, D)[j].double()
            for a in range(h * (Hq // Hkv), (h + 1) * (Hq // Hkv)):
                z = s["q"][t0:t0 + n, a].double() @ kh.t() * s["scale"]
                z = torch.where(seen, z, torch.full_like(z, -math.inf))
                lse[a, t0:t0 + n] = torch.logsumexp(z, 1)
                o[t0:t0 + n, a] = torch.softmax(z, 1) @ vh
        t0 += n
    if s["op"] == "step":
        return [None, None, None, None, o, lse]
    return [o, lse]
