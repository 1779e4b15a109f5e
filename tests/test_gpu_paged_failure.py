"""Failure detection of the paged attention, exercised without a GPU fault: as for the
whole-sequence forward, a test hook never loads one Q tile, so that a bounded wait runs out;
the kernel records it, drains and ends, and the next forward is clean."""
import ctypes

import pytest
import torch

from tests import paged_cases as C

pytestmark = pytest.mark.gpu

DEV_TIMEOUT_Q = 1
# (old, new): whole and cut units of one and of two halves; one unit of one half; hints that
# keep units whole, so that no join runs
RAGGED = ([300, 0, 64, 5000], [200, 77, 1, 300])
LENS = [pytest.param(RAGGED, {}, id="ragged"), pytest.param(([3], [40]), {}, id="half"),
        pytest.param(RAGGED, dict(max_new=300, max_len=128), id="whole")]


def _captured(monkeypatch, c, spec, **hints):
    """Arguments of the forward's C call, plan and results of an ordinary call."""
    from polyhedral_b200 import paged
    d = {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in c.items()}
    T, H, D = d["q"].shape
    plan = paged.make_plan(d["seq_lens"], d["q_start"], *spec, tokens=T, heads=H,
                           kv_heads=d["k_cache"].shape[2], head_dim=D,
                           page_size=d["k_cache"].shape[1], **hints)
    calls, launch = [], paged._launch

    def keep(name, device, *args):
        calls.append((name, args))
        launch(name, device, *args)
    monkeypatch.setattr(paged, "_launch", keep)
    out = paged.paged_attention(d["q"], d["k_cache"], d["v_cache"], d["block_table"], d["seq_lens"],
                                d["q_start"], *spec, plan=plan, return_lse=True, check=True)
    monkeypatch.undo()
    (name, args), = calls
    assert name == "pa_paged_attn"
    return d, plan, args, out


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lens,hints", LENS)
def test_bounded_wait_runs_out_and_reports(monkeypatch, lens, D, hints):
    from polyhedral_b200 import _lib, paged
    lib = _lib.load()
    spec = (C.SINKS, 90, 4, 0)
    c = C.make(*lens, 8, 2, D, 32, torch.bfloat16, seed=61)
    d, plan, args, ref = _captured(monkeypatch, c, spec, **hints)
    C.check(c, spec, *ref)
    scratch = torch.zeros(max(plan.scratch_bytes, 256), dtype=torch.uint8, device="cuda")
    o, lse = torch.zeros_like(ref[0]), torch.zeros_like(ref[1])
    a = _lib.PaPagedAttnArgs.from_buffer_copy(args[0] + bytes(ctypes.sizeof(_lib.PaPagedAttnArgs) - len(args[0])))
    a.o, a.lse = o.data_ptr(), lse.data_ptr()
    for _ in range(2):
        assert plan.status() == 0
        rc = lib.pa_paged_attn_withheld(ctypes.byref(a), plan.buffer.data_ptr(), plan.nbytes,
                                        scratch.data_ptr(), plan.scratch_bytes, 2_000_000,
                                        _lib.stream_handle(o.device))
        assert rc == 0, lib.pa_last_error()
        assert plan.status() == DEV_TIMEOUT_Q
        with pytest.raises(_lib.PolyattnError, match="bounded wait"):
            paged.paged_attention(d["q"], d["k_cache"], d["v_cache"], d["block_table"],
                                  d["seq_lens"], d["q_start"], *spec, plan=plan, check=True)
        # the context is usable, and a forward on a plan built anew clean
        plan = paged.make_plan(d["seq_lens"], d["q_start"], *spec, tokens=o.shape[0], heads=8,
                               kv_heads=2, head_dim=D, page_size=32, **hints)
        again = paged.paged_attention(d["q"], d["k_cache"], d["v_cache"], d["block_table"],
                                      d["seq_lens"], d["q_start"], *spec, plan=plan,
                                      return_lse=True, check=True)
        assert torch.equal(again[0], ref[0]) and torch.equal(again[1], ref[1])


def test_withheld_refusals(monkeypatch):
    from polyhedral_b200 import _lib
    lib = _lib.load()
    spec = (C.CAUSAL, 0, 0, 0)
    c = C.make([30], [40], 4, 2, 64, 16, torch.bfloat16, seed=62)
    for hints, limit, code in ((dict(), 999, _lib.PA_ERR_ARG), (dict(), 1_000_000_001, _lib.PA_ERR_ARG),
                               (dict(max_new=1), 2_000_000, _lib.PA_ERR_UNSUPPORTED)):
        _, plan, args, _ = _captured(monkeypatch, c, spec, **hints)
        rc = lib.pa_paged_attn_withheld(args[0], plan.buffer.data_ptr(), plan.nbytes, args[3],
                                        plan.scratch_bytes, limit, None)
        assert rc == code, lib.pa_last_error()
        assert plan.status() == 0
