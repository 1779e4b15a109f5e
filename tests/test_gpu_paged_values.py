"""What the paged attention makes of values that are not finite in keys and queries that do
count, at every column of a super-tile, and how exact its exponentials are."""
import math

import numpy as np
import pytest
import torch

from oracle import paged_oracle as PO
from tests import paged_cases as C

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16
CAUSAL = (C.CAUSAL, 0, 0, 0)
# 34 query rows per key head: the tensor-core kernel; told one token, the few-rows kernel
HINTS = [pytest.param({}, id="chunk"), pytest.param(dict(max_new=1), id="few")]


def _compare(c, o, lse):
    """Rows whose result is no number in 64 bits are none here; the others keep their bound."""
    o_ref, lse_ref = PO.paged_attention(c["q"], c["k_cache"], c["v_cache"], c["block_table"],
                                        c["seq_lens"], c["q_start"], *CAUSAL)
    o, lse = o.double().cpu(), lse.double().cpu()
    gone = ~torch.isfinite(lse_ref.t())
    assert gone.any() and not gone.all()
    assert torch.isnan(o_ref[gone]).all()
    assert torch.isnan(o[gone]).all(), f"{int((~torch.isnan(o[gone])).any(1).sum())} rows lost a key"
    assert not torch.isfinite(lse[gone.t()]).any()
    ok = dict(c, q=c["q"].clone(), k_cache=c["k_cache"].nan_to_num(0.0, 0.0, 0.0))
    ok["q"][gone] = 0
    bo, bl = C.bounds(ok, CAUSAL, torch.where(gone[..., None], 0.0, o_ref))
    # an infinite key of weight 0 stands as one of score 0 in `ok`: up to a factor 2 of the sums
    assert ((o - o_ref).abs() <= 2 * bo)[~gone].all()
    assert (lse - lse_ref)[~gone.t()].abs().max() <= bl


@pytest.mark.parametrize("hints", HINTS)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_keys_that_are_seen(bad, dtype, D, hints):
    """Request x: the key at column x of the second super-tile has a NaN or an infinity in its
    first place, which makes its score a NaN, or +inf or -inf by the sign of q's.  A NaN and a
    +inf reach o and lse of every row; a -inf is a weight of 0.  The odd requests stay whole."""
    B, n = 256, 17
    c = C.make([283] * B, [n] * B, 2, 1, D, 64, dtype, seed=31, nan=False)
    for x in range(128):
        j = 128 + x
        c["k_cache"][c["block_table"][2 * x, j // 64].long(), j % 64, 0, 0] = bad
    o, lse = C.run(c, CAUSAL, **hints)
    _compare(c, o, lse)


@pytest.mark.parametrize("hints", HINTS)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_queries_that_are_not_finite(bad, D, hints):
    """A row of q that is no number has no result; the rows beside it do."""
    c = C.make([40, 283, 0], [30, 17, 9], 2, 1, D, 16, BF, seed=32)
    for t, a in ((0, 0), (7, 1), (30, 0), (46, 1), (47, 0), (55, 1)):
        c["q"][t, a, 3] = bad
    o, lse = C.run(c, CAUSAL, **hints)
    gone = ~torch.isfinite(c["q"]).all(2)
    o, lse = o.double().cpu(), lse.double().cpu()
    # an infinite query's scores are infinities: a row of -inf alone has weights of 0, one with
    # a +inf no result
    o_bad, lse_bad = PO.paged_attention(c["q"], c["k_cache"], c["v_cache"], c["block_table"],
                                        c["seq_lens"], c["q_start"], *CAUSAL)
    none = torch.isneginf(lse_bad.t())
    assert torch.isnan(o[gone & ~none]).all() and not torch.isfinite(lse.t()[gone]).any()
    assert (o[none] == 0).all() and torch.isneginf(lse.t()[none]).all()
    rest = dict(c, q=torch.where(gone[..., None], 0.0, c["q"].float()).to(BF))
    o_ref, lse_ref = PO.paged_attention(rest["q"], c["k_cache"], c["v_cache"], c["block_table"],
                                        c["seq_lens"], c["q_start"], *CAUSAL)
    bo, bl = C.bounds(rest, CAUSAL, o_ref)
    assert ((o - o_ref).abs() <= bo)[~gone].all()
    assert (lse - lse_ref)[~gone.t()].abs().max() <= bl


@pytest.mark.parametrize("hints", HINTS)
@pytest.mark.parametrize("D", [64, 128])
def test_exponentials(D, hints):
    """One row sees a key of score 0 and, at column x of the second super-tile, one of score z:
    lse = log(1 + e^z) in 32 bits.  z goes through [-20, 5.5]: above 0 too, since the maximum
    that is subtracted lags by up to 2^8.  With w = e^z / (1 + e^z) the error is at most

    - w times the weight's: 2.7e-6 of the polynomial, which is the larger one's, and 2^-23
      |z log2 e| of an exponent that is a product rounded once with a constant rounded once;
    - 2^-24 for each of the sum, log2's own (1 unit in the last place, at most 2^-23 of its
      value and of 1) and the final product: 2^-22 (1 + |lse|) together."""
    B = 128
    z = torch.linspace(-20.0, 5.5, B).to(HF)
    z = z[torch.randperm(B, generator=torch.Generator().manual_seed(1))]
    c = C.make([239] * B, [17] * B, 2, 1, D, 64, HF, seed=33, nan=False)
    c["k_cache"][:] = 0
    c["k_cache"][..., 0] = -200.0                   # weight 0
    t = c["block_table"].long()
    c["k_cache"][t[:, 0], 0, 0, 0] = 0.0
    for x in range(B):
        j = 128 + x
        c["k_cache"][t[x, j // 64], j % 64, 0, 0] = z[x]
    c["q"][:] = 0
    c["q"][..., 0] = 1.0
    o, lse = C.run(c, CAUSAL, scale=1.0, **hints)
    lse = lse.double().cpu()[:, 16::17]             # the last token sees every key
    zd = z.double()
    ref = torch.log1p(torch.exp(zd))
    w = torch.exp(zd - ref)
    tol = w * (2.7e-6 + 2.0**-23 * (zd / math.log(2)).abs()) + 2.0**-22 * (1 + ref)
    err = (lse - ref).abs()
    assert (err <= tol).all(), f"{float((err / tol).max()):.2f} of the bound, {np.argmax((err / tol).amax(0))}"
