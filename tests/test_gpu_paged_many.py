"""Paged attention of very many requests at once."""
import pytest
import torch

from tests import paged_cases as C

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B", [1023, 1024, 1025, 3000, 65536])
@pytest.mark.parametrize("most,hints", [(1, dict(max_new=1)), (1, dict(max_new=1, max_len=24)), (9, {}),
                                        (9, dict(max_new=9, max_len=24))],
                         ids=["one", "one whole", "chunk", "chunk whole"])
def test_many_requests(B, most, hints):
    """Requests of 0 to 24 tokens, up to `most` of them new, idle ones among them, against
    64-bit sums over all requests at once; the bound is that of paged_cases.bounds, with
    A <= max |v| < 6."""
    from polyhedral_b200 import paged
    H, Hkv, D, page = 4, 2, 64, 16
    g = torch.Generator(device="cuda").manual_seed(B)
    kw = dict(device="cuda", generator=g)
    lens = torch.randint(0, 25, (B,), **kw)
    new = torch.minimum(torch.randint(0, most + 1, (B,), **kw), lens)
    start = torch.cat([new.new_zeros(1), new.cumsum(0)])
    T = int(start[-1])
    kc, vc = (torch.randn(2 * B, page, Hkv, D, dtype=torch.bfloat16, **kw) for _ in range(2))
    table = torch.randperm(2 * B, **kw).view(B, 2)
    q = torch.randn(T, H, D, dtype=torch.bfloat16, **kw)
    o, lse = paged.paged_attention(q, kc, vc, table.int(), lens.int(), start.int(), C.CAUSAL, 0, 0, 0,
                                   return_lse=True, check=True, **hints)
    t = torch.arange(T, device="cuda")
    b = torch.searchsorted(start[1:], t, right=True)
    i = lens[b] - new[b] + t - start[b]
    j = torch.arange(32, device="cuda")
    worst = 0.0
    for part in t.split(16384):
        k, v = (x[table[b[part]]].reshape(-1, 32, Hkv, D).double().repeat_interleave(2, 2)
                for x in (kc, vc))
        z = torch.einsum("thd,tjhd->thj", q[part].double(), k) / D**0.5
        z = z.masked_fill((j > i[part][:, None])[:, None], -torch.inf)
        ref = torch.einsum("thj,tjhd->thd", torch.softmax(z, 2), v)
        err = (o[part].double() - ref).abs()
        tol = 2.0**-8 * (ref.abs() + 6.0) + (2 * 1.3e-4 + 2.0**-20) * 6.0
        worst = max(worst, float((err / tol).max()))
        assert (lse[:, part].double().t() - torch.logsumexp(z, 2)).abs().max() <= 1.5e-4
        # no larger error is common to many elements
        assert err.norm() <= 2.0**-7 * ref.norm()
    assert worst <= 1.0
