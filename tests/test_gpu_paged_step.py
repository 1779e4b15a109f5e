"""Tables of a serving step and the cache append, on the GPU, against request-by-request
statements on the CPU (whole numbers and copies: exact)."""
import numpy as np
import pytest
import torch

from oracle import paged_oracle as PO

pytestmark = pytest.mark.gpu


def _i32(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


def _run(table, old, new, free, head, P, tokens, out=None):
    from polyhedral_b200 import paged
    t = table.cuda() if isinstance(table, torch.Tensor) else _i32(table)
    st = paged.make_step(t, _i32(old), _i32(new), _i32(free), _i32([head]), page_size=P,
                         tokens=tokens, out=out)
    return t, st


def _same(t, st, ref):
    table, q_start, lens, slots, pos, head, missing = ref
    assert np.array_equal(t.cpu().numpy(), table)
    assert st.q_start.tolist() == q_start
    assert st.seq_lens.tolist() == lens
    assert st.slot_map.tolist() == slots
    assert st.positions.tolist() == pos
    assert st.free_head.tolist() == [head] and st.missing.tolist() == [missing]


def _case(B, P, lo, hi, old_hi, seed, spare=3):
    r = np.random.RandomState(seed)
    old, new = r.randint(0, old_hi + 1, B), r.randint(lo, hi + 1, B)
    width = int(max(-(-(old + new) // P))) + 1
    have = -(-old // P)
    total = int((-(-(old + new) // P)).sum()) + spare
    ids = r.permutation(total + 7)
    table = np.full((B, width), -1)
    n = 0
    for b in range(B):
        table[b, :have[b]] = ids[n:n + have[b]]
        n += have[b]
    return table, old, new, ids, n


@pytest.mark.parametrize("B,P,lo,hi,old_hi", [
    (1, 16, 1, 1, 0), (1, 16, 1, 1, 15), (1, 16, 1, 1, 16), (3, 1, 0, 4, 9), (8, 16, 1, 1, 2000),
    (5, 24, 0, 100, 60), (511, 16, 0, 3, 200), (512, 32, 1, 1, 64), (513, 64, 0, 40, 129),
    (1500, 16, 0, 9, 300)])
def test_step_matches_statement(B, P, lo, hi, old_hi):
    table, old, new, ids, n = _case(B, P, lo, hi, old_hi, B + P)
    for extra in (0, 5):                       # entries behind the last token
        tokens = int(new.sum()) + extra
        t, st = _run(table, old, new, ids, n, P, tokens)
        _same(t, st, PO.step_tables(table, old, new, ids, n, P, tokens))


def test_many_requests():
    table, old, new, ids, n = _case(16384, 16, 0, 2, 40, 3)
    t, st = _run(table, old, new, ids, n, 16, int(new.sum()))
    _same(t, st, PO.step_tables(table, old, new, ids, n, 16, int(new.sum())))


def test_free_list_and_table_run_out():
    """Too few free pages, a table too narrow, entries that are no pages, negative
    lengths, fewer slots than tokens."""
    table, old, new, ids, n = _case(40, 16, 0, 90, 50, 11)
    for head, width, cut in ((len(ids) - 9, table.shape[1], 0), (len(ids), table.shape[1], 0),
                             (n, 3, 0), (n, table.shape[1], 100), (len(ids) - 4, 2, 33)):
        tab = table[:, :width]
        tokens = int(new.sum()) - cut
        t, st = _run(tab, old, new, ids, head, 16, tokens)
        _same(t, st, PO.step_tables(tab, old, new, ids, head, 16, tokens))
    bad = table.copy()
    bad[::3, 0] = -7
    bad[1::3, 0] = 2**31 - 1                  # its slots would not fit in 32 bits
    old2, new2 = old.copy(), new.copy()
    old2[2], new2[5] = -4, -3
    tokens = int(np.maximum(new2, 0).sum())
    t, st = _run(bad, old2, new2, ids, n, 16, tokens)
    _same(t, st, PO.step_tables(bad, old2, new2, ids, n, 16, tokens))


def test_step_strided_table_and_out_reuse():
    from polyhedral_b200 import paged
    table, old, new, ids, n = _case(9, 16, 1, 40, 100, 5)
    wide = torch.full((9, table.shape[1] + 6), -5, dtype=torch.int32, device="cuda")
    view = wide[:, 2:2 + table.shape[1]]
    view.copy_(_i32(table))
    tokens = int(new.sum())
    out = paged.PagedStep(9, tokens, view.device)
    st = paged.make_step(view, _i32(old), _i32(new), _i32(ids), _i32([n]), page_size=16,
                         tokens=tokens, out=out)
    assert st is out
    _same(view, st, PO.step_tables(table, old, new, ids, n, 16, tokens))
    assert (wide[:, :2] == -5).all() and (wide[:, 2 + table.shape[1]:] == -5).all()
    with pytest.raises(Exception, match="free_head_out is free_head"):
        paged.make_step(view, _i32(old), _i32(new), _i32(ids), out.free_head, page_size=16,
                        tokens=tokens, out=out)


def _rows(T, H, D, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(T, H, D, generator=g).to(dtype).cuda() for _ in range(2)]


@pytest.mark.parametrize("T,H,D,P", [(1, 1, 64, 16), (61, 8, 128, 16), (7, 3, 64, 32), (300, 16, 128, 64),
                                     (5, 5, 40, 8), (1000, 1, 128, 1), (33, 32, 256, 16)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_append_matches_copy(T, H, D, P, dtype):
    from polyhedral_b200 import paged
    k, v = _rows(T, H, D, dtype, T)
    pages = -(-T // P) + 3
    g = torch.Generator().manual_seed(1)
    slots = torch.randperm(pages * P, generator=g)[:T].to(torch.int32)
    slots[::5] = -1
    if T > 3:
        slots[3] = pages * P                  # one past the end: skipped
    kc, vc = (torch.full((pages, P, H, D), float("nan"), dtype=dtype, device="cuda")
              for _ in range(2))
    paged.append_kv(k, v, kc, vc, slots.cuda())
    ok = (slots >= 0) & (slots < pages * P)
    for got, rows in ((kc, k), (vc, v)):
        ref = torch.full((pages * P, H, D), float("nan"), dtype=dtype)
        ref[slots[ok].long()] = rows.cpu()[ok]
        assert torch.equal(got.cpu().view(torch.int16), ref.view(pages, P, H, D).view(torch.int16))


def test_append_strided():
    """Rows cut out of a fused projection, caches interleaved in one tensor and with the
    heads before the rows."""
    from polyhedral_b200 import paged
    T, H, D, P, pages = 29, 4, 64, 16, 5
    g = torch.Generator().manual_seed(2)
    qkv = torch.randn(T, 3 * H * D, generator=g).bfloat16().cuda()
    k, v = (qkv[:, i * H * D:(i + 1) * H * D].view(T, H, D) for i in (1, 2))
    slots = torch.randperm(pages * P, generator=g)[:T].to(torch.int32).cuda()
    both = torch.zeros(pages, 2, P, H, D, dtype=torch.bfloat16, device="cuda")
    paged.append_kv(k, v, both[:, 0], both[:, 1], slots)
    heads_first = torch.zeros(2, pages, H, P, D, dtype=torch.bfloat16, device="cuda")
    paged.append_kv(k, v, heads_first[0].transpose(1, 2), heads_first[1].transpose(1, 2), slots)
    for i, rows in enumerate((k, v)):
        ref = torch.zeros(pages * P, H, D, dtype=torch.bfloat16, device="cuda")
        ref[slots.long()] = rows
        ref = ref.view(pages, P, H, D)
        assert torch.equal(both[:, i], ref)
        assert torch.equal(heads_first[i].transpose(1, 2), ref)


def test_append_offsets_beyond_32_bits():
    """Rows behind the 2^32-nd byte of a cache."""
    from polyhedral_b200 import paged
    H, D, P = 8, 128, 16
    pages = (2**32 // 2 // (P * H * D)) + 40          # elements past 2^31, bytes past 2^32
    kc = torch.zeros(pages, P, H, D, dtype=torch.bfloat16, device="cuda")
    k, v = _rows(6, H, D, torch.bfloat16, 4)
    slots = torch.tensor([0, pages * P - 1, pages * P - 20, 17, (pages - 3) * P, 5],
                         dtype=torch.int32, device="cuda")
    vc = kc[:, :, :, :]                                # one buffer for both: V written too
    paged.append_kv(v, v, kc, vc, slots)
    flat = kc.view(pages * P, H, D)
    assert torch.equal(flat[slots.long()], v)
    flat[slots.long()] = 0
    assert not flat.any()


def test_append_nothing():
    from polyhedral_b200 import paged
    kc = torch.zeros(2, 16, 1, 64, dtype=torch.bfloat16, device="cuda")
    z = torch.zeros(0, 1, 64, dtype=torch.bfloat16, device="cuda")
    paged.append_kv(z, z, kc, kc.clone(), torch.zeros(0, dtype=torch.int32, device="cuda"))
    assert not kc.any()
