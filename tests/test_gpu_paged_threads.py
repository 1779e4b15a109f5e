"""Paged-cache entry points from several host threads at once."""
import threading

import pytest
import torch

from oracle import paged_oracle as PO

pytestmark = pytest.mark.gpu


def test_steps_of_many_requests_from_two_threads():
    """Batches whose prefix sums need different amounts of shared memory beyond 48 KB; every
    call is launched, and gives its own tables."""
    from polyhedral_b200 import paged
    errors = []

    def work(B, n):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                table = torch.full((B, 2), -1, dtype=torch.int32, device="cuda")
                old = torch.zeros(B, dtype=torch.int32, device="cuda")
                new = (torch.arange(B, device="cuda") % 3).int()
                free = torch.arange(B, dtype=torch.int32, device="cuda").flip(0).contiguous()
                head = torch.zeros(1, dtype=torch.int32, device="cuda")
                T = int(new.sum())
                for _ in range(n):
                    st = paged.make_step(table, old, new, free, head, page_size=16, tokens=T)
                ref = PO.step_tables(torch.full((B, 2), -1).numpy(), old.tolist(), new.tolist(),
                                     free.tolist(), 0, 16, T)
                assert (table.cpu().numpy() == ref[0]).all()
                assert st.slot_map.tolist() == ref[3] and st.missing.tolist() == [0]
        except Exception as e:              # noqa: BLE001  (shown by the assert below)
            errors.append((B, e))

    threads = [threading.Thread(target=work, args=a) for a in ((16384, 3000), (6000, 3000), (7000, 3000))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
