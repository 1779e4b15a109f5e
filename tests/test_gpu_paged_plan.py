"""A plan belongs to the lengths that it was built from: a forward with others says so."""
import pytest
import torch

from tests import paged_cases as C

pytestmark = pytest.mark.gpu

BF = torch.bfloat16
CAUSAL = (C.CAUSAL, 0, 0, 0)
LONGEST = 4200


def _setup(total, new, seed=41):
    """Requests of `total` tokens, the last `new` of which are the step's, over a cache that
    holds all of LONGEST."""
    B = len(total)
    c = C.make([LONGEST] * B, [0] * B, 8, 2, 64, 16, BF, seed=seed, nan=False)
    T = sum(new)
    g = torch.Generator().manual_seed(seed)
    c["q"] = torch.randn(T, 8, 64, generator=g).to(BF)
    c["tokens"] = T
    return _lengths(c, total, new)


def _lengths(c, total, new):
    start = torch.tensor([0] + new).cumsum(0)
    return dict(c, seq_lens=torch.tensor(total).int(), q_start=start.int())


def _plan(c, spec, **hints):
    from polyhedral_b200 import paged
    return paged.make_plan(c["seq_lens"].cuda(), c["q_start"].cuda(), *spec, tokens=c["q"].shape[0],
                           heads=8, kv_heads=2, head_dim=64, page_size=16, **hints)


# (tokens, new ones) of the plan's step and of the call's: the next decode step; the next chunks;
# new tokens moved from one request to another; a request that had nothing to do and now
# has; a plan of a step with nothing to do
STALE = [pytest.param(([3000, 40, 700], [1, 1, 1]), ([3001, 41, 701], [1, 1, 1]), id="decode"),
         pytest.param(([400, 90, 2000], [300, 90, 17]), ([700, 180, 2017], [300, 90, 17]), id="chunks"),
         pytest.param(([400, 90, 2000], [3, 1, 1]), ([401, 91, 2001], [1, 3, 1]), id="moved"),
         pytest.param(([0, 90, 2000], [0, 2, 1]), ([1, 91, 2001], [1, 1, 1]), id="woken"),
         pytest.param(([0, 0], [0, 0]), ([50, 60], [2, 3]), id="nothing")]


@pytest.mark.parametrize("plan_step,step", STALE)
@pytest.mark.parametrize("hints", [dict(max_new=1), dict(), dict(max_new=1, max_len=100)],
                         ids=["few", "chunk", "whole"])
def test_another_steps_plan_is_reported(plan_step, step, hints):
    from polyhedral_b200 import _lib
    c = _setup(*step)
    old = _lengths(c, *plan_step)
    plan = _plan(old, CAUSAL, **hints)
    with pytest.raises(_lib.PolyattnError, match="other lengths") as e:
        C.run(c, CAUSAL, plan=plan)
    assert e.value.code == _lib.PA_ERR_DEVICE
    assert plan.status() == _lib.DEV_OTHER_LENGTHS
    # built again for these lengths: clean, and right
    o, lse = C.run(c, CAUSAL, plan=_plan(c, CAUSAL, **hints))
    C.check(c, CAUSAL, o, lse)


@pytest.mark.parametrize("hints", [dict(max_new=1), dict()], ids=["few", "chunk"])
def test_lengths_overwritten_in_place_are_reported(hints):
    """A loop that fills one pair of length tensors step after step, and forgets the plan."""
    from polyhedral_b200 import _lib
    c = _setup([3000, 40, 700], [1, 1, 20])
    d = {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in c.items()}
    from polyhedral_b200 import paged
    plan = paged.make_plan(d["seq_lens"], d["q_start"], *CAUSAL, tokens=22, heads=8, kv_heads=2,
                           head_dim=64, page_size=16, **hints)

    def call():
        return paged.paged_attention(d["q"], d["k_cache"], d["v_cache"], d["block_table"],
                                     d["seq_lens"], d["q_start"], *CAUSAL, plan=plan, check=True)
    call()
    d["seq_lens"] += 1
    with pytest.raises(_lib.PolyattnError, match="other lengths"):
        call()


@pytest.mark.parametrize("hints", [dict(max_new=1), dict()], ids=["few", "chunk"])
def test_equal_lengths_are_not_reported(hints):
    """Idle requests before, between and behind the others; tensors of the same values; a table
    narrower than the lengths."""
    c = _setup([0, 5, 900, 33, 0, 70, 8], [0, 0, 40, 1, 0, 30, 0])
    plan = _plan(c, CAUSAL, **hints)
    o, lse = C.run(c, CAUSAL, plan=plan)
    C.check(c, CAUSAL, o, lse)
    narrow = dict(c, block_table=c["block_table"][:, :20].contiguous())
    C.run(narrow, CAUSAL, plan=plan)
    assert plan.status() == 0


@pytest.mark.parametrize("hints", [dict(max_new=1, max_len=100), dict(max_new=60, max_len=100)],
                         ids=["few", "chunk"])
@pytest.mark.parametrize("woken", [0, 700, 2999])
def test_one_request_woken_among_many(hints, woken):
    """Idle requests before the first share: one of them has tokens in the call, not in the plan.
    Units stay whole here, so that no join runs.  (One that wakes behind the first share is
    read from the arrays, and served.)"""
    from polyhedral_b200 import _lib
    B = 3000
    total, new = [0] * B + [70] * 80, [0] * B + [60] * 80
    old = _lengths(_setup([5], [0]), total, new)
    c = dict(old, block_table=old["block_table"].expand(B + 80, -1).contiguous(),
             q=torch.randn(4800, 8, 64).to(BF), tokens=4800)
    plan = _plan(c, CAUSAL, **hints)
    C.run(c, CAUSAL, plan=plan)
    total[woken], new[woken] = 3, 1
    new[-1] -= 1                                 # q keeps its rows
    with pytest.raises(_lib.PolyattnError, match="other lengths"):
        C.run(_lengths(c, total, new), CAUSAL, plan=plan)
