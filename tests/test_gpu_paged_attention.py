"""Attention over a paged cache against the 64-bit statement, with bounds derived from the
roundings (paged_cases.bounds)."""
import pytest
import torch

from tests import paged_cases as C

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16
SPECS = [(C.CAUSAL, 0, 0, 0), (C.WINDOW, 37, 0, 0), (C.SINKS, 20, 4, 0), (C.DILATED, 4, 0, 0),
         (C.DILATED, 5, 0, 0), (C.LOCAL_STRIDED, 24, 8, 0), (C.TWOBAND, 17, 40, 9),
         (C.FAR_STRIDED, 16, 8, 0)]
# (old, new) lengths: single tokens, first tokens, chunks, requests with nothing to do,
# page ends inside and at the chunk's end
DECODE = ([0, 15, 16, 99, 300, 0, 511], [1, 1, 1, 1, 1, 0, 1])
FEW = ([0, 3, 100, 255, 40], [4, 3, 2, 4, 0])
MIXED = ([0, 7, 130, 0, 64, 250, 1], [1, 70, 33, 0, 300, 1, 17])


@pytest.mark.parametrize("spec", SPECS)
@pytest.mark.parametrize("lens", [DECODE, FEW, MIXED], ids=["decode", "few", "mixed"])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_masks(spec, lens, dtype):
    c = C.make(*lens, 4, 2, 64, 16, dtype, seed=1)
    o, lse = C.run(c, spec)
    C.check(c, spec, o, lse)


@pytest.mark.parametrize("spec", SPECS)
@pytest.mark.parametrize("lens,longest", [(([0, 33, 90, 0], [17, 5, 30, 0]), 120), (MIXED, 364)],
                         ids=["short", "mixed"])
@pytest.mark.parametrize("heads,kv_heads,D", [(4, 2, 64), (6, 2, 128), (24, 1, 64)])
def test_small_chunks_with_known_lengths(spec, lens, longest, heads, kv_heads, D):
    """With few keys in all the few-rows kernel takes chunks too, units that begin and end
    inside a token among them."""
    c = C.make(*lens, heads, kv_heads, D, 16, BF, seed=11)
    o, lse = C.run(c, spec, max_new=max(lens[1]), max_len=longest)
    C.check(c, spec, o, lse)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (6, 2), (5, 5), (7, 1), (16, 2), (24, 2), (48, 2),
                                            (128, 1)])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lens", [DECODE, MIXED], ids=["decode", "mixed"])
def test_head_layouts(heads, kv_heads, D, lens):
    spec = (C.CAUSAL, 0, 0, 0)
    c = C.make(*lens, heads, kv_heads, D, 32, BF, seed=heads)
    o, lse = C.run(c, spec)
    C.check(c, spec, o, lse)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256, 1024])
@pytest.mark.parametrize("spec", [(C.CAUSAL, 0, 0, 0), (C.SINKS, 100, 5, 0), (C.WINDOW, 1, 0, 0)])
@pytest.mark.parametrize("lens", [DECODE, MIXED], ids=["decode", "mixed"])
def test_pages(page, spec, lens):
    c = C.make(*lens, 8, 2, 128, page, HF, seed=page)
    o, lse = C.run(c, spec)
    C.check(c, spec, o, lse)


@pytest.mark.parametrize("old,new,hint", [([4095], [1], 1), ([5000, 3], [1, 1], 1), ([4000], [64], 0),
                                          ([2000, 2500], [1, 200], 0), ([6000], [3], 3)])
@pytest.mark.parametrize("spec", [(C.CAUSAL, 0, 0, 0), (C.WINDOW, 1000, 0, 0),
                                  (C.SINKS, 900, 130, 0), (C.LOCAL_STRIDED, 64, 16, 0)])
def test_long_contexts_are_split(old, new, hint, spec):
    c = C.make(old, new, 4, 2, 128, 64, BF, seed=7)
    o, lse = C.run(c, spec, max_new=hint)
    C.check(c, spec, o, lse)


@pytest.mark.parametrize("old,new", [(3000, 900), (2945, 1000), (2900, 1055), (500, 1210), (0, 1300)])
@pytest.mark.parametrize("spec", [(C.SINKS, 300, 4, 0), (C.SINKS, 1, 70, 0), (C.WINDOW, 257, 0, 0),
                                  (C.TWOBAND, 100, 400, 60), (C.CAUSAL, 0, 0, 0)])
def test_shares_cut_units_anywhere(old, new, spec):
    """Enough units that the shares' cuts fall on every super-tile of some unit, super-tiles
    that one half skips among them; twice the same bits."""
    c = C.make([old, 17], [new, 40], 24, 24, 64, 64, BF, seed=9)
    o, lse = C.run(c, spec)
    C.check(c, spec, o, lse)
    o2, lse2 = C.run(c, spec)
    assert torch.equal(o, o2) and torch.equal(lse, lse2)


@pytest.mark.parametrize("spec", [(C.WINDOW, 0, 0, 0), (C.FAR_STRIDED, 10**6, 4, 0),
                                  (C.SINKS, 0, 0, 0)])
@pytest.mark.parametrize("lens", [DECODE, MIXED], ids=["decode", "mixed"])
def test_rows_that_see_nothing(spec, lens):
    c = C.make(*lens, 4, 2, 64, 16, BF, seed=2)
    o, lse = C.run(c, spec)
    assert not o.any() and torch.isneginf(lse).all()


def test_scale_and_hints_do_not_change_results():
    """The hints choose the kernel, never the result's meaning, even where they are wrong."""
    spec = (C.SINKS, 50, 3, 0)
    c = C.make(*MIXED, 8, 2, 128, 16, BF, seed=3)
    for hints in (dict(), dict(max_new=1), dict(max_new=300, max_len=364), dict(max_len=5),
                  dict(max_new=1, max_len=1)):
        o, lse = C.run(c, spec, scale=0.05, **hints)
        C.check(c, spec, o, lse, scale=0.05)


def test_rows_behind_the_last_request_and_strides():
    """A padded batch; q cut from a fused projection, o and lse into larger buffers, the
    caches interleaved in one tensor with the heads before the rows."""
    from polyhedral_b200 import paged
    spec = (C.WINDOW, 60, 0, 0)
    for lens in (DECODE, MIXED):
        c = C.make(*lens, 6, 2, 64, 16, BF, seed=4, tail=37)
        T, H, D = c["q"].shape
        kc = c["k_cache"]
        both = torch.full((kc.shape[0], 2, 2, 16, D), float("nan"), dtype=BF, device="cuda")
        both[:, 0] = kc.cuda().transpose(1, 2)
        both[:, 1] = c["v_cache"].cuda().transpose(1, 2)
        wide = torch.randn(T, H + 4, D, dtype=BF, device="cuda")
        q = wide[:, 2:2 + H]
        q.copy_(c["q"])
        out = torch.full((T, H, 2 * D), 7.0, dtype=BF, device="cuda")
        lse = torch.full((H, T + 9), 7.0, device="cuda")
        tab = torch.full((len(lens[0]), c["block_table"].shape[1] + 3), 10**6, dtype=torch.int32,
                         device="cuda")
        tab[:, :-3] = c["block_table"]
        paged.paged_attention(q, both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2),
                              tab[:, :-3], c["seq_lens"].cuda(), c["q_start"].cuda(), *spec,
                              out=out[..., :D], lse_out=lse[:, :T], check=True)
        C.check(c, spec, out[..., :D], lse[:, :T])
        n = c["tokens"]
        assert (out[n:] == 7).all() and (out[..., D:] == 7).all()
        assert (lse[:, n:] == 7).all()


@pytest.mark.parametrize("lens", [DECODE, MIXED], ids=["decode", "mixed"])
def test_pages_outside_the_cache_hold_no_keys(lens):
    spec = (C.CAUSAL, 0, 0, 0)
    c = C.make(*lens, 4, 2, 64, 16, BF, seed=5)
    t = c["block_table"]
    t[3, 1] = -1
    t[4, 2] = c["k_cache"].shape[0]
    t[5, 0] = 2**31 - 1
    t[6, 0] = -2**31
    o, lse = C.run(c, spec)
    C.check(c, spec, o, lse)


@pytest.mark.parametrize("bad", [float("inf"), float("nan"), float("-inf")])
@pytest.mark.parametrize("lens", [DECODE, MIXED], ids=["decode", "mixed"])
def test_non_finite_values_in_masked_places(bad, lens):
    """Rows that the window has left behind hold no numbers any more; a token's own
    future neither."""
    for spec in ((C.WINDOW, 30, 0, 0), (C.SINKS, 30, 2, 0), (C.CAUSAL, 0, 0, 0)):
        c = C.make(*lens, 4, 2, 64, 16, BF, seed=6)
        old, new = lens
        for b, (x, n) in enumerate(zip(old, new)):
            t = c["block_table"][b].long()
            gone = range(2, x - 30 + 1) if spec[0] != C.CAUSAL else []
            for j in gone:
                c["k_cache"][t[j // 16], j % 16] = bad
                c["v_cache"][t[j // 16], j % 16] = bad
        o, lse = C.run(c, spec)
        C.check(c, spec, o, lse)
        if max(new) > 1:      # the last token of a chunk breaks down: no earlier one does
            b = new.index(max(new))
            j = old[b] + new[b] - 1
            c["v_cache"][c["block_table"][b, j // 16].long(), j % 16] = bad
            o2, lse2 = C.run(c, spec)
            last = int(c["q_start"][b + 1]) - 1
            rest = torch.arange(c["tokens"]) != last
            assert torch.isfinite(o2[: c["tokens"]][rest.cuda()]).all()
            assert not torch.isfinite(o2[last]).any()
            err = (o2.float() - o.float())[: c["tokens"]][rest.cuda()].abs().max()
            assert err <= 2.0**-7 * o.float().abs().max()
            # the rows may be summed in another order now; each sum keeps the bound of
            # paged_cases.bounds (e + 2e-5, e = 1.3e-4), so two are within twice that
            assert (lse2 - lse)[:, : c["tokens"]].abs().max() <= 2 * (1.3e-4 + 2e-5)


@pytest.mark.parametrize("old,new,hint", [([3000], [3], 3), ([2500, 60], [90, 1], 0)])
def test_non_finite_values_in_split_requests(old, new, hint):
    """The last token's value breaks down in a request that is divided among workers: only the
    last row does; and a value that every row sees reaches all of them."""
    spec = (C.CAUSAL, 0, 0, 0)
    c = C.make(old, new, 4, 2, 128, 16, BF, seed=15)
    o, lse = C.run(c, spec, max_new=hint)
    C.check(c, spec, o, lse)
    j = old[0] + new[0] - 1
    t = c["block_table"][0].long()
    c["v_cache"][t[j // 16], j % 16] = float("nan")
    o2, lse2 = C.run(c, spec, max_new=hint)
    last = new[0] - 1
    assert torch.isnan(o2[last]).all() and torch.isfinite(o2[:last]).all()
    assert torch.isfinite(o2[new[0]:]).all()
    # both are within paged_cases.bounds of the same 64-bit result
    bo, bl = C.bounds(c, spec, torch.zeros(o.shape, dtype=torch.float64))
    tol = 2 * (bo[:last] + 2.0**-8 * o[:last].double().cpu().abs())
    assert ((o2 - o).double().cpu().abs()[:last] <= tol).all()
    assert (lse2 - lse).abs().max() <= 2 * bl
    c["v_cache"][t[7], 3] = float("inf")
    o3, _ = C.run(c, spec, max_new=hint)
    assert torch.isinf(o3[:last]).all() and torch.isfinite(o3[new[0]:]).all()
