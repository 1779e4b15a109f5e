"""Inputs of the paged-attention tests: ragged requests over scattered pages, with NaN in
every cache row that holds no token, and the bound that the outputs keep."""
import numpy as np
import torch

from oracle import paged_oracle as PO

CAUSAL, WINDOW, DILATED, LOCAL_STRIDED, TWOBAND, SINKS, FAR_STRIDED = range(7)

# half a step of the output's type relative to the value
HALF_STEP = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}


def make(old, new, heads, kv_heads, D, page, dtype, seed=0, tail=0, spare=3, nan=True):
    """Tensors on the CPU: q [tokens, heads, D] with `tail` rows behind the last request,
    caches, table, lengths.  Rows of no token hold NaN, spare table entries page ids of
    another request's or none at all."""
    r = np.random.RandomState(seed)
    g = torch.Generator().manual_seed(seed)
    old, new = np.asarray(old), np.asarray(new)
    total = old + new
    need = -(-total // page)
    pages = int(need.sum()) + spare
    ids = r.permutation(pages)
    width = int(need.max()) + 2
    table = np.where(r.rand(len(old), width) < 0.5, -1, r.randint(0, pages, (len(old), width)))
    kc, vc = (torch.randn(pages, page, kv_heads, D, generator=g).to(dtype) for _ in range(2))
    n = 0
    used = torch.zeros(pages, page, dtype=torch.bool)
    for b in range(len(old)):
        table[b, :need[b]] = ids[n:n + need[b]]
        n += need[b]
        for x in range(need[b]):
            used[table[b, x], :min(page, total[b] - x * page)] = True
    if nan:
        kc[~used] = float("nan")
        vc[~used] = float("nan")
    T = int(new.sum()) + tail
    q = torch.randn(T, heads, D, generator=g).to(dtype)
    q_start = np.concatenate([[0], np.cumsum(new)])
    return dict(q=q, k_cache=kc, v_cache=vc, block_table=torch.from_numpy(table).int(),
                seq_lens=torch.from_numpy(total).int(), q_start=torch.from_numpy(q_start).int(),
                tokens=int(new.sum()))


def bounds(c, spec, o_ref, scale=None):
    """Largest error of o and lse against 64 bits, from the roundings:

    - o is rounded once: u |o|, u half a step of the type;
    - every softmax weight is rounded once to the type before the product with V: u A,
      A = sum p_j |v_j| / sum p_j, and, where the type is fp16, weights below 2^-14 of
      the largest lose up to 2^-25 each: n 2^-25 max |v|;
    - a score is a sum of D products in 32 bits: off by at most (D + 2) 2^-24 sum |q k| scale.
      Here |q|, |k| ~ |N(0, 1)|: sum |q k| scale < 16 for D = 64, 128 (mean 7, and its
      deviation below 1), so the error is below 130 * 2^-24 * 16 = 1.3e-4 = e; a weight is
      then off by at most 2 e relative, and so is A's share;
    - partial results of a split request are joined in 32 bits: 2^-20 A covers them and
      the exponential's own error (2 units of 2^-23) many times over;
    - lse: e, plus the sum's relative error and the logarithm's: 2e-5 together."""
    e = 1.3e-4
    u = HALF_STEP[c["q"].dtype]
    va = c["v_cache"].double().abs()
    A, _ = PO.paged_attention(c["q"], c["k_cache"], va, c["block_table"], c["seq_lens"],
                              c["q_start"], *spec, scale=scale)
    n = int(c["seq_lens"].max())
    flush = n * 2.0**-25 * 8 if c["q"].dtype == torch.float16 else 0.0
    return u * (o_ref.abs() + A) + (2 * e + 2.0**-20) * A + flush + 1e-30, e + 2e-5


def check(c, spec, o, lse, scale=None):
    o_ref, lse_ref = PO.paged_attention(c["q"], c["k_cache"], c["v_cache"], c["block_table"],
                                        c["seq_lens"], c["q_start"], *spec, scale=scale)
    T = c["tokens"]
    bo, bl = bounds(c, spec, o_ref, scale)
    o, lse = o.double().cpu()[:T], lse.double().cpu()[:, :T]
    o_ref, lse_ref, bo = o_ref[:T], lse_ref[:, :T], bo[:T]
    dead = torch.isneginf(lse_ref)
    assert torch.equal(torch.isneginf(lse), dead)
    assert (o[dead.t()] == 0).all()
    assert torch.isfinite(o).all()
    err = (o - o_ref).abs()
    assert (err <= bo).all(), f"o off by {err.max():.3e}, {(err / bo).max():.2f} of its bound"
    el = (lse - lse_ref)[~dead].abs()
    assert el.numel() == 0 or el.max() <= bl, f"lse off by {el.max():.3e}"
    return float((err / bo).max()) if err.numel() else 0.0


def run(c, spec, **kw):
    from polyhedral_b200 import paged
    d = {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in c.items()}
    return paged.paged_attention(d["q"], d["k_cache"], d["v_cache"], d["block_table"],
                                 d["seq_lens"], d["q_start"], *spec, return_lse=True, check=True,
                                 **kw)
