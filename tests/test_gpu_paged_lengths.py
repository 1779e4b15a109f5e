"""Tables of a step for lengths at the end of 32 bits."""
import numpy as np
import pytest
import torch

from oracle import paged_oracle as PO

pytestmark = pytest.mark.gpu

TOP = 2**31 - 1


def _i32(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("P", [1, 16, 24, 1024])
@pytest.mark.parametrize("old,new", [([TOP, 5, 0], [1, 20, 3]), ([TOP - 2, TOP, 7, TOP], [9, 0, 2, 30]),
                                     ([40, TOP - 700, 3], [2, 1500, 1])])
def test_tokens_behind_the_last_position(P, old, new):
    """They have no slot and no position, and disturb no other request's."""
    from polyhedral_b200 import paged
    B, width = len(old), 60
    r = np.random.RandomState(3)
    ids = r.permutation(200)
    table = np.full((B + 2, width), -7)
    table[1:-1] = -1
    n = 0
    for b in range(B):
        if old[b] < 1000:
            have = -(-old[b] // P)
            table[1 + b, :have] = ids[n:n + have]
            n += have
        else:
            table[1 + b] = 199                  # a page at every column
    whole = _i32(table)
    T = sum(new) + 4
    st = paged.make_step(whole[1:-1], _i32(old), _i32(new), _i32(ids), _i32([n]), page_size=P,
                         tokens=T)
    ref = PO.step_tables(table[1:-1], old, new, ids, n, P, T)
    gone = [p > TOP for p in ref[4]]
    assert np.array_equal(whole[1:-1].cpu().numpy(), ref[0])
    assert (whole[0] == -7).all() and (whole[-1] == -7).all()
    assert st.q_start.tolist() == ref[1]
    assert st.seq_lens.tolist() == [min(x, TOP) for x in ref[2]]
    assert st.slot_map.tolist() == [-1 if g else s for g, s in zip(gone, ref[3])]
    assert st.positions.tolist() == [-1 if g else p for g, p in zip(gone, ref[4])]
    assert st.free_head.tolist() == [ref[5]] and st.missing.tolist() == [ref[6]]


def test_slot_map_of_all_32_bits():
    """2^31 - 1 entries, of which six tokens fill the first."""
    from polyhedral_b200 import paged
    T = TOP
    table = torch.full((2, 3), -1, dtype=torch.int32, device="cuda")
    guard = torch.full((3, 1000), 77, dtype=torch.int32, device="cuda")
    st = paged.make_step(table, _i32([0, 15]), _i32([2, 4]), _i32([4, 9, 2]), _i32([0]), page_size=16,
                         tokens=T)
    assert st.slot_map[:6].tolist() == [64, 65, -1, 144, 145, 146]
    assert st.positions[:6].tolist() == [0, 1, 15, 16, 17, 18]
    for t in (st.slot_map, st.positions):
        for part in t[6:].split(2**28):
            assert bool((part == -1).all())
    assert st.q_start.tolist() == [0, 2, 6] and st.seq_lens.tolist() == [2, 19]
    assert st.free_head.tolist() == [2] and st.missing.tolist() == [0]
    assert (guard == 77).all()
