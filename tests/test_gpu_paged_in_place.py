"""Results written over q."""
import pytest
import torch

from tests import paged_cases as C

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


@pytest.mark.parametrize("hints", [dict(max_new=1), dict(), dict(max_new=300, max_len=128)],
                         ids=["few", "chunk", "whole"])
@pytest.mark.parametrize("heads,kv_heads,D,dtype", [(4, 2, 64, BF), (6, 2, 128, HF), (8, 8, 128, BF),
                                                    (48, 2, 64, HF)])
@pytest.mark.parametrize("bad", [None, float("nan"), float("inf")])
def test_in_place(bad, heads, kv_heads, D, dtype, hints):
    """The same bits as into a tensor of its own: also where rows that the window has left, and
    the last token's value, are not finite, so that rows are computed again from their q; the
    rows behind the last request's and the other columns of a wider buffer stay."""
    from polyhedral_b200 import paged
    spec = (C.WINDOW, 30, 0, 0)
    old, new = [0, 70, 130, 0, 600, 250], [1, 70, 33, 0, 300, 1]
    c = C.make(old, new, heads, kv_heads, D, 16, dtype, seed=81, tail=5)
    if bad is not None:
        for b, (x, n) in enumerate(zip(old, new)):
            t = c["block_table"][b].long()
            for j in list(range(max(x - 30 + 1, 0))) + ([x + n - 1] if n > 1 else []):
                c["v_cache"][t[j // 16], j % 16] = bad
    d = {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in c.items()}
    T = d["q"].shape[0]
    wide = torch.full((T, heads + 1, 2 * D), 7.0, dtype=dtype, device="cuda")
    q = wide[:, :heads, D:]

    def call(q, **kw):
        return paged.paged_attention(q, d["k_cache"], d["v_cache"], d["block_table"], d["seq_lens"],
                                     d["q_start"], *spec, return_lse=True, check=True, **hints, **kw)

    out = torch.full_like(d["q"], 7.0)
    o_ref, lse_ref = call(d["q"], out=out)
    if bad is None:
        C.check(c, spec, o_ref, lse_ref)
    for _ in range(3):
        q.copy_(d["q"])
        o, lse = call(q, out=q)
        n = c["tokens"]
        same = lambda x, y: torch.equal(x.isnan(), y.isnan()) and torch.equal(  # noqa: E731
            x.nan_to_num(1.0), y.nan_to_num(1.0))
        assert same(o[:n], o_ref[:n]) and same(lse[:, :n], lse_ref[:, :n])
        assert torch.equal(q[n:], d["q"][n:])
        assert (wide[:, heads:] == 7).all() and (wide[:, :, :D] == 7).all()
