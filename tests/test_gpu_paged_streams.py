"""The paged-cache operators across streams, eagerly and in captured graphs: kernels that may
begin while the one before them still runs keep every order that events ask for."""
import pytest
import torch

from tests import paged_cases as C

pytestmark = pytest.mark.gpu

BF = torch.bfloat16
SPEC = (C.SINKS, 200, 3, 0)
LENS = [pytest.param(([500, 3, 130], [1, 1, 1]), dict(max_new=1), id="few"),
        pytest.param(([500, 3, 130], [90, 40, 1]), {}, id="chunk")]


class Step:
    """One step of one layer: caches without the new rows, which `append` brings."""

    def __init__(self, lens, seed):
        self.c = c = C.make(*lens, 8, 2, 64, 16, BF, seed=seed)
        self.d = {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in c.items()}
        slots = []
        for b, (x, n) in enumerate(zip(*lens)):
            t = c["block_table"][b].long()
            slots += [int(t[p // 16]) * 16 + p % 16 for p in range(x, x + n)]
        flat = torch.tensor(slots)
        self.k, self.v = (c[n].view(-1, 2, 64)[flat].cuda() for n in ("k_cache", "v_cache"))
        self.slots = flat.int().cuda()
        self.T = len(slots)

    def clear(self):
        for n in ("k_cache", "v_cache"):
            self.d[n].view(-1, 2, 64)[self.slots.long()] = 0.0

    def append(self):
        from polyhedral_b200 import paged
        paged.append_kv(self.k, self.v, self.d["k_cache"], self.d["v_cache"], self.slots)

    def plan(self, hints):
        from polyhedral_b200 import paged
        return paged.make_plan(self.d["seq_lens"], self.d["q_start"], *SPEC, tokens=self.T, heads=8,
                               kv_heads=2, head_dim=64, page_size=16, **hints)

    def attend(self, plan):
        from polyhedral_b200 import paged
        d = self.d
        return paged.paged_attention(d["q"], d["k_cache"], d["v_cache"], d["block_table"],
                                     d["seq_lens"], d["q_start"], *SPEC, plan=plan, return_lse=True)


def _fork(steps, hints):
    """The rows are appended on a second stream behind some waiting, while the first builds the
    plan; the first attends when the second is done, another layer on the second stream."""
    side, main = torch.cuda.Stream(), torch.cuda.current_stream()
    side.wait_stream(main)
    with torch.cuda.stream(side):
        torch.cuda._sleep(400_000)
        for s in steps:
            s.append()
    plan = steps[0].plan(hints)
    main.wait_stream(side)
    side.wait_stream(main)
    with torch.cuda.stream(side):
        second = steps[1].attend(plan)
    first = steps[0].attend(plan)
    main.wait_stream(side)
    return first, second, plan, side


@pytest.mark.parametrize("lens,hints", LENS)
def test_append_on_another_stream(lens, hints):
    steps = [Step(lens, seed) for seed in (71, 72)]
    for _ in range(5):
        for s in steps:
            s.clear()
        first, second, plan, _ = _fork(steps, hints)
        torch.cuda.synchronize()
        for s, (o, lse) in zip(steps, (first, second)):
            C.check(s.c, SPEC, o, lse)
        assert plan.status() == 0


@pytest.mark.parametrize("lens,hints", LENS)
def test_captured_fork_and_join(lens, hints):
    steps = [Step(lens, seed) for seed in (73, 74)]
    _fork(steps, hints)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        first, second, plan, side = _fork(steps, hints)
    for _ in range(5):
        for s in steps:
            s.clear()
        for t in first + second:
            t.fill_(9.0)
        graph.replay()
        torch.cuda.synchronize()
        for s, (o, lse) in zip(steps, (first, second)):
            C.check(s.c, SPEC, o, lse)
        assert plan.status() == 0


@pytest.mark.parametrize("lens,hints", LENS)
def test_captured_first_and_last(lens, hints):
    """A graph whose only nodes are the forward's, one behind a copy and one before a fill, and
    replays beside eager calls on the same plan."""
    s = Step(lens, 75)
    s.append()
    plan = s.plan(hints)
    ref = s.attend(plan)
    torch.cuda.synchronize()
    q = s.d["q"].clone()
    graphs = []
    for mode in range(3):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            if mode == 1:
                s.d["q"].copy_(q)
            out = s.attend(plan)
            kept = out[0].clone() if mode == 2 else out[0]
            if mode == 2:
                out[0].fill_(3.0)
        graphs.append((g, kept, out[1]))
    side = torch.cuda.Stream()
    for _ in range(10):
        for g, o, lse in graphs:
            g.replay()
            with torch.cuda.stream(side):
                eager = s.attend(plan)
        torch.cuda.synchronize()
        for o, lse in [x[1:] for x in graphs] + [eager]:
            assert torch.equal(o, ref[0]) and torch.equal(lse, ref[1])
    C.check(s.c, SPEC, *ref)
