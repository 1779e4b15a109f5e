"""Lengths and offsets outside the buffers, against the 64-bit statement."""
import pytest
import torch

from tests import paged_cases as C

pytestmark = pytest.mark.gpu

CAUSAL = (C.CAUSAL, 0, 0, 0)


@pytest.mark.parametrize("hints", [dict(max_new=1), dict()], ids=["few", "chunk"])
@pytest.mark.parametrize("end,lens", [(999, (80, 6, 34)), (999, (80, 6, 1007)), (45, (80, 6, 34)), (31, (80, 6, 34))])
def test_new_tokens_beyond_q(end, lens, hints):
    """The last request's offset says more new tokens than q has rows: those rows that exist are
    the first of them, at the positions that the lengths give, and nothing else is read or
    written."""
    from polyhedral_b200 import paged
    T, B = 30, 3
    c = C.make([60, 0, 1000], [20, 6, 7], 4, 2, 64, 16, torch.bfloat16, seed=51, nan=False)
    c["q"] = c["q"][:T].contiguous()
    c["seq_lens"] = torch.tensor(lens, dtype=torch.int32)
    start = torch.tensor([0, 20, 26, end], dtype=torch.int32)
    out = torch.full((T + 9, 4, 64), 5.0, dtype=torch.bfloat16, device="cuda")
    lse = torch.full((4, T + 9), 5.0, device="cuda")
    d = {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in c.items()}
    paged.paged_attention(d["q"], d["k_cache"], d["v_cache"], d["block_table"], d["seq_lens"],
                          start.cuda(), *CAUSAL, out=out[:T], lse_out=lse[:, :T], check=True, **hints)
    # the statement's request of all its tokens, cut off behind the rows that exist
    full = dict(c, q=torch.cat([c["q"], torch.zeros(end - T, 4, 64).bfloat16()]), q_start=start,
                tokens=T)
    C.check(full, CAUSAL, torch.cat([out[:T], out.new_zeros(end - T, 4, 64)]),
            torch.cat([lse[:, :T], lse.new_zeros(4, end - T)], 1))
    assert (out[T:] == 5).all() and (lse[:, T:] == 5).all()
