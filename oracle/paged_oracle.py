"""CPU statements of the paged-cache operators: the tables of a serving step (numpy,
request by request) and the attention of new tokens over a paged cache (64-bit)."""
import math

import numpy as np
import torch


def step_tables(block_table, old, new, free, head, page_size, tokens):
    """(block_table, q_start, seq_lens, slot_map, positions, free_head, missing) of one
    step; the arrays given are not changed."""
    table = np.array(block_table, dtype=np.int64)
    width, P = table.shape[1], page_size
    q_start, lens, slots, pos = [0], [], [], []
    missing = 0
    for b, (c, n) in enumerate(zip(old, new)):
        c, n = max(int(c), 0), max(int(n), 0)
        for col in range(-(-c // P), -(-(c + n) // P)):
            if col >= width:
                missing += 1
            elif head < len(free):
                table[b, col] = free[head]
                head += 1
            else:
                table[b, col] = -1
                missing += 1
        for p in range(c, c + n):
            col = p // P
            page = int(table[b, col]) if col < width else -1
            ok = page >= 0 and (page + 1) * P <= 2**31 - 1
            slots.append(page * P + p % P if ok else -1)
            pos.append(p)
        lens.append(c + n)
        q_start.append(q_start[-1] + n)
    slots = (slots + [-1] * tokens)[:tokens]
    pos = (pos + [-1] * tokens)[:tokens]
    return table, q_start, lens, slots, pos, head, missing


def live(kind, p0, p1, p2, i, j):
    """[len(i), len(j)] bool: the mask on absolute positions."""
    d = i[:, None] - j[None, :]
    kv = j[None, :]
    m = d >= 0
    if kind == 1:
        m &= d < p0
    elif kind == 2:
        m &= d % p0 == 0
    elif kind == 3:
        m &= (d < p0) | (d % p1 == 0)
    elif kind == 4:
        m &= (d < p0) | ((d >= p1) & (d < p1 + p2))
    elif kind == 5:
        m &= (d < p0) | (kv < p1)
    elif kind == 6:
        m &= (d >= p0) & (d % p1 == 0)
    elif kind != 0:
        raise ValueError(kind)
    return m


def paged_attention(q, k_cache, v_cache, block_table, seq_lens, q_start, kind, p0, p1, p2,
                    scale=None):
    """o [tokens, heads, D] and lse [heads, tokens] in float64 on the CPU; rows of no
    request are NaN.  Keys on pages outside the cache do not count."""
    q, kc, vc = (t.double().cpu() for t in (q, k_cache, v_cache))
    table = torch.as_tensor(block_table).long().cpu()
    T, Hq, D = q.shape
    P, Hkv = kc.shape[1], kc.shape[2]
    scale = scale or 1.0 / math.sqrt(D)
    o = torch.full((T, Hq, D), math.nan, dtype=torch.float64)
    lse = torch.full((Hq, T), math.nan, dtype=torch.float64)
    for b, n in enumerate(int(x) for x in seq_lens):
        t0, t1 = int(q_start[b]), int(q_start[b + 1])
        if t1 <= t0:
            continue
        i = torch.arange(n - (t1 - t0), n)
        j = torch.arange(max(n, 0))
        page = table[b][j // P] if n > 0 else j
        j, page = j[(page >= 0) & (page < kc.shape[0])], page[(page >= 0) & (page < kc.shape[0])]
        m = live(kind, p0, p1, p2, i, j)
        for a in range(Hq):
            h = a // (Hq // Hkv)
            k, v = kc[page, j % P, h], vc[page, j % P, h]
            z = q[t0:t1, a] @ k.t() * scale
            z = torch.where(m, z, torch.full_like(z, -math.inf))
            top = z.max(1, keepdim=True).values if j.numel() else z.new_full((t1 - t0, 1), -math.inf)
            top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
            e = torch.where(m, torch.exp(z - top), torch.zeros_like(z))
            s = e.sum(1, keepdim=True)
            # a masked key's value takes no part, whatever it is
            vz = torch.where(m.any(0)[:, None], v, torch.zeros_like(v))
            if torch.isfinite(vz).all():
                num = e @ vz
            else:
                num = torch.stack([(e[r][:, None] * v)[m[r]].sum(0) for r in range(t1 - t0)])
            o[t0:t1, a] = num / torch.where(s > 0, s, torch.ones_like(s))
            lse[a, t0:t1] = (top + torch.log(s)).squeeze(1)
    return o, lse
