"""The paged-cache operators together, as a serving loop runs them: prompts in chunks, then
single tokens, against the framework's whole-sequence attention; captured steps; several
streams; caches beyond 32-bit offsets."""
import numpy as np
import pytest
import torch

from oracle import paged_oracle as PO
from tests import paged_cases as C

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


class Loop:
    """One layer's serving state: a block table, a free list and a cache for `B` requests."""

    def __init__(self, B, longest, heads, kv_heads, D, page, dtype=BF, seed=0, nan=True):
        self.B, self.page, self.shape = B, page, (heads, kv_heads, D)
        pages = B * (-(-longest // page)) + 2
        g = torch.Generator().manual_seed(seed)
        self.table = torch.full((B, -(-longest // page)), -1, dtype=torch.int32, device="cuda")
        self.free = torch.randperm(pages, generator=g).int().cuda()
        self.head = torch.zeros(1, dtype=torch.int32, device="cuda")
        fill = float("nan") if nan else 0.0
        self.kc, self.vc = (torch.full((pages, page, kv_heads, D), fill, dtype=dtype, device="cuda")
                            for _ in range(2))
        self.old = torch.zeros(B, dtype=torch.int32, device="cuda")

    def step(self, q, k, v, new, spec, **hints):
        from polyhedral_b200 import paged
        T = q.shape[0]
        st = paged.make_step(self.table, self.old, new, self.free, self.head, page_size=self.page,
                             tokens=T)
        plan = paged.make_plan(st.seq_lens, st.q_start, *spec, tokens=T, heads=self.shape[0],
                               kv_heads=self.shape[1], head_dim=self.shape[2], page_size=self.page,
                               **hints)
        paged.append_kv(k, v, self.kc, self.vc, st.slot_map)
        o, lse = paged.paged_attention(q, self.kc, self.vc, self.table, st.seq_lens, st.q_start,
                                       *spec, plan=plan, return_lse=True)
        self.old, self.head = st.seq_lens, st.free_head
        return o, lse, st, plan


@pytest.mark.parametrize("spec", [(C.CAUSAL, 0, 0, 0), (C.WINDOW, 128, 0, 0), (C.SINKS, 256, 4, 0),
                                  (C.DILATED, 4, 0, 0), (C.LOCAL_STRIDED, 64, 8, 0)])
def test_chunks_then_single_tokens_equal_the_whole_sequence(spec):
    """Two sequences of 1024 tokens, cut into chunks and single tokens in different ways,
    give what block_sparse_attention gives on the whole: the two round in different places
    (weights and results to bf16 once each), so they agree within twice the bound that each
    keeps against 64 bits."""
    from polyhedral_b200 import attention, blockindex, masks
    N, H, D, B = 1024, 4, 128, 2
    g = torch.Generator().manual_seed(21)
    q, k, v = (torch.randn(B, H, N, D, generator=g).to(BF).cuda() for _ in range(3))
    flat = [t.reshape(B * H, N, D) for t in (q, k, v)]

    class Spec(masks.Mask):
        def __init__(self):
            self.spec = spec

    dbi = blockindex.build_device(Spec(), N, 128, 64, device="cuda")
    o_ref, lse_ref = attention.block_sparse_attention(*flat, dbi.kv_idx, dbi.kv_num, dbi.kv_partial,
                                                      *spec, 128, 64, return_lse=True, check=True)
    o_ref, lse_ref = o_ref.view(B, H, N, D), lse_ref.view(B, H, N)

    loop = Loop(B, N, H, H, D, 64)
    cuts = [[300, 1, 211, 0, 500, 1, 1, 10], [1, 1, 600, 77, 0, 1, 300, 44]]
    done = [0, 0]
    for n in zip(*cuts):
        rows = [slice(done[b], done[b] + n[b]) for b in range(B)]
        part = [torch.cat([t[b, :, rows[b]].transpose(0, 1) for b in range(B)]) for t in (q, k, v)]
        new = torch.tensor(n, dtype=torch.int32, device="cuda")
        o, lse, st, plan = loop.step(*part, new, spec, max_new=max(n))
        assert plan.status() == 0 and int(st.missing) == 0
        at = 0
        for b in range(B):
            ob, lb = o[at:at + n[b]].transpose(0, 1), lse[:, at:at + n[b]]
            at += n[b]
            r = o_ref[b][:, rows[b]].float()
            # A <= max |v| bounds sum p |v| / sum p
            tol = 2 * (2.0**-8 * (r.abs() + 4.0) + 4e-4 * 4.0)
            assert ((ob.float() - r).abs() <= tol).all()
            assert ((ob.float() - r).norm() <= 2.0**-7 * r.norm() + 1e-6)
            assert (lb - lse_ref[b][:, rows[b]]).abs().nan_to_num(0.0).max() <= 2 * 1.5e-4 if n[b] else True
            done[b] += n[b]
    assert done == [N, N]


def test_captured_step_replays_with_new_lengths():
    """A whole step captured once: its lengths, tables and free list change between replays;
    a longer batch is padded with requests that have nothing to do."""
    from polyhedral_b200 import paged
    B, T, H, Hkv, D, page = 5, 24, 8, 2, 64, 16
    spec = (C.SINKS, 40, 3, 0)
    longest = 400
    loop = Loop(B, longest, H, Hkv, D, page, seed=3)
    g = torch.Generator().manual_seed(4)
    q, k, v = (torch.zeros(T, h, D, dtype=BF, device="cuda") for h in (H, Hkv, Hkv))
    old, new = (torch.zeros(B, dtype=torch.int32, device="cuda") for _ in range(2))
    head = torch.zeros(1, dtype=torch.int32, device="cuda")
    st = paged.PagedStep(B, T, q.device)
    out = torch.full((T, H, D), 5.0, dtype=BF, device="cuda")
    lse = torch.full((H, T), 5.0, device="cuda")

    def run():
        paged.make_step(loop.table, old, new, loop.free, head, page_size=page, tokens=T, out=st)
        plan = paged.make_plan(st.seq_lens, st.q_start, *spec, tokens=T, heads=H, kv_heads=Hkv,
                               head_dim=D, page_size=page)
        paged.append_kv(k, v, loop.kc, loop.vc, st.slot_map)
        paged.paged_attention(q, loop.kc, loop.vc, loop.table, st.seq_lens, st.q_start, *spec,
                              plan=plan, out=out, lse_out=lse)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        run()                                  # nothing to do: all lengths are 0
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    lens = np.zeros(B, dtype=np.int64)
    for n in ([7, 0, 9, 1, 0], [1, 1, 1, 1, 1], [0, 24, 0, 0, 0], [2, 3, 1, 5, 8], [0] * 5,
              [1, 1, 1, 1, 20]):
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, generator=g).to(BF))
        old.copy_(torch.from_numpy(lens).int())
        new.copy_(torch.tensor(n, dtype=torch.int32))
        out.fill_(5.0)
        lse.fill_(5.0)
        graph.replay()
        torch.cuda.synchronize()
        head.copy_(st.free_head)
        lens += np.array(n)
        assert int(st.missing) == 0
        total = sum(n)
        c = dict(q=q.cpu(), k_cache=loop.kc.cpu(), v_cache=loop.vc.cpu(), block_table=loop.table.cpu(),
                 seq_lens=torch.from_numpy(lens).int(), q_start=st.q_start.cpu(), tokens=total)
        if total:
            C.check(c, spec, out, lse)
        assert (out[total:] == 5).all() and (lse[:, total:] == 5).all()


@pytest.mark.parametrize("lens,hint", [(([3000, 900, 50], [1, 1, 1]), 1), (([700, 0, 90], [300, 200, 1]), 0)])
def test_one_plan_on_two_streams_and_two_graphs(lens, hint):
    """Layers on different streams share a plan; so do two captured graphs that replay at
    the same time (every call has scratch memory of its own)."""
    from polyhedral_b200 import paged
    spec = (C.CAUSAL, 0, 0, 0)
    H, Hkv, D, page = 8, 2, 64, 16
    cases = [C.make(*lens, H, Hkv, D, page, BF, seed=s) for s in (1, 2)]
    dev = [{k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in c.items()} for c in cases]
    T = dev[0]["q"].shape[0]
    plan = paged.make_plan(dev[0]["seq_lens"], dev[0]["q_start"], *spec, tokens=T, heads=H,
                           kv_heads=Hkv, head_dim=D, page_size=page, max_new=hint)

    def call(d):
        return paged.paged_attention(d["q"], d["k_cache"], d["v_cache"], d["block_table"],
                                     d["seq_lens"], d["q_start"], *spec, plan=plan, return_lse=True)

    ref = [call(d) for d in dev]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(20):
        for s, d in zip(streams, dev):
            with torch.cuda.stream(s):
                got.append(call(d))
    torch.cuda.synchronize()
    for i, (o, lse) in enumerate(got):
        assert torch.equal(o, ref[i % 2][0]) and torch.equal(lse, ref[i % 2][1])
    graphs, outs = [], []
    for d in dev:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call(d))
        graphs.append(g)
    for _ in range(20):
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for i, (o, lse) in enumerate(outs):
        assert torch.equal(o, ref[i][0]) and torch.equal(lse, ref[i][1])
    for c, (o, lse) in zip(cases, ref):
        C.check(c, spec, o, lse)


@pytest.mark.parametrize("lens,hint", [(([500, 33], [1, 1]), 1), (([70, 200], [130, 9]), 0)])
def test_cache_beyond_32_bit_offsets(lens, hint):
    """Pages behind the 2^32-nd byte of K and of V."""
    spec = (C.CAUSAL, 0, 0, 0)
    H, Hkv, D, page = 8, 4, 128, 16
    c = C.make(*lens, H, Hkv, D, page, BF, seed=8, nan=False)
    extra = 2**32 // (page * Hkv * D * 2) + 5
    big = {}
    for name in ("k_cache", "v_cache"):
        t = torch.zeros(extra + c[name].shape[0], page, Hkv, D, dtype=BF, device="cuda")
        t[extra:] = c[name].cuda()
        big[name] = t
    from polyhedral_b200 import paged
    table = torch.where(c["block_table"] >= 0, c["block_table"] + extra, c["block_table"])
    o, lse = paged.paged_attention(c["q"].cuda(), big["k_cache"], big["v_cache"], table.int().cuda(),
                                   c["seq_lens"].cuda(), c["q_start"].cuda(), *spec, return_lse=True,
                                   check=True, max_new=hint)
    C.check(c, spec, o, lse)


def test_nothing_to_do():
    from polyhedral_b200 import paged
    z = torch.zeros(0, 4, 64, dtype=BF, device="cuda")
    kc = torch.zeros(3, 16, 2, 64, dtype=BF, device="cuda")
    i = torch.zeros(2, dtype=torch.int32, device="cuda")
    o, lse = paged.paged_attention(z, kc, kc, torch.zeros(2, 1, dtype=torch.int32, device="cuda"), i,
                                   torch.zeros(3, dtype=torch.int32, device="cuda"), 0, 0, 0, 0,
                                   return_lse=True, check=True)
    assert o.shape == (0, 4, 64) and lse.shape == (4, 0)
    # rows, but no request has any
    q = torch.ones(5, 4, 64, dtype=BF, device="cuda")
    out = torch.full_like(q, 3.0)
    for hint in (0, 1):
        paged.paged_attention(q, kc, kc, torch.zeros(2, 1, dtype=torch.int32, device="cuda"), i,
                              torch.zeros(3, dtype=torch.int32, device="cuda"), 0, 0, 0, 0, out=out,
                              check=True, max_new=hint)
        assert (out == 3).all()


@pytest.mark.parametrize("hint", [0, 1])
def test_lengths_that_do_not_fit(hint):
    """More tokens than the table has room for: the tokens behind its end are not there;
    more new tokens than tokens: the first of them see nothing; offsets outside q are not
    followed."""
    from polyhedral_b200 import paged
    spec = (C.CAUSAL, 0, 0, 0)
    c = C.make([60, 0, 30], [20, 6, 4], 4, 2, 64, 16, BF, seed=10)
    d = {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in c.items()}
    table = d["block_table"].clone()
    lens = d["seq_lens"].clone()
    lens[1] = 4                                # 6 new tokens, 4 in all: positions -2 .. 3
    narrow = table[:, :4].contiguous()         # 64 of request 0's 80 tokens
    o, lse = paged.paged_attention(d["q"], d["k_cache"], d["v_cache"], narrow, lens, d["q_start"], *spec,
                                   return_lse=True, check=True, max_new=hint)
    assert torch.isneginf(lse[:, 20:22]).all() and not o[20:22].any()
    assert torch.isfinite(o).all() and torch.isfinite(lse[:, :20]).all()
    ref = dict(c)
    ref["block_table"] = torch.full((3, 6), -1, dtype=torch.int32)
    ref["block_table"][:, :4] = narrow.cpu()
    ref["seq_lens"] = lens.cpu()
    C.check(ref, spec, o, lse)
    start = torch.tensor([0, 20, 26, 999], dtype=torch.int32, device="cuda")
    before = o.clone()
    o2 = paged.paged_attention(d["q"], d["k_cache"], d["v_cache"], table, d["seq_lens"], start, *spec,
                               check=True, max_new=hint)
    assert o2.shape == before.shape


def test_wide_masks():
    """Widths near the largest int are as good as no limit."""
    c = C.make([100, 3], [40, 5], 4, 2, 64, 16, BF, seed=12)
    big = 2**31 - 1
    a, la = C.run(c, (C.CAUSAL, 0, 0, 0))
    for spec in ((C.WINDOW, big, 0, 0), (C.SINKS, big, big, 0), (C.SINKS, 1, big, 0),
                 (C.TWOBAND, big, 5, 5), (C.TWOBAND, 0, 0, big), (C.LOCAL_STRIDED, big, 8, 0),
                 (C.DILATED, 1, 0, 0)):
        for hint in (0, 1):
            o, lse = C.run(c, spec, max_new=hint)
            C.check(c, (C.CAUSAL, 0, 0, 0), o, lse)


@pytest.mark.parametrize("lens", [([300, 70], [1, 1]), ([200, 33], [90, 40])])
def test_parts_join_with_lse_merge(lens):
    """Disjoint masks over one cache (the near band, everything behind it) joined by
    ``merge.lse_merge`` are the causal attention: each part is within its bound, and the
    merge rounds once more, so 2.5 bounds cover the three."""
    from polyhedral_b200 import merge
    c = C.make(*lens, 8, 2, 128, 16, BF, seed=14)
    parts = [C.run(c, spec) for spec in ((C.WINDOW, 40, 0, 0), (C.FAR_STRIDED, 40, 1, 0))]
    (o1, l1), (o2, l2) = ((o.transpose(0, 1), lse) for o, lse in parts)
    o, lse = merge.lse_merge(o1, l1, o2, l2)
    spec = (C.CAUSAL, 0, 0, 0)
    o_ref, lse_ref = PO.paged_attention(c["q"], c["k_cache"], c["v_cache"], c["block_table"],
                                        c["seq_lens"], c["q_start"], *spec)
    bo, bl = C.bounds(c, spec, o_ref)
    # a part's own mean of |v| may exceed the whole's: 4 bounds |v| < 4 as well
    bo = 2.5 * (bo + 2.0**-7 * 4.0 * 0.25)
    err = (o.transpose(0, 1).double().cpu() - o_ref).abs()
    assert (err <= bo).all(), float((err / bo).max())
    assert (lse.double().cpu() - lse_ref).abs().max() <= 2.5 * bl
