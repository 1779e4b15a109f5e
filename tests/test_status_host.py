"""Reading a plan's device status when CUDA itself fails, without a GPU: the C entry point is
replaced by one that reports the error."""
import contextlib
import ctypes
import types

import pytest
import torch

from polyhedral_b200 import _lib, attention, paged


@pytest.fixture
def answers(monkeypatch):
    """Makes both status entry points return a code and write a word."""
    monkeypatch.setattr(_lib, "on_device", lambda device: contextlib.nullcontext())
    monkeypatch.setattr(_lib, "stream_handle", lambda device=None: ctypes.c_void_p(0))

    def set_to(rc, word):
        def status(ptr, out, stream):
            out._obj.value = word
            return rc
        fake = types.SimpleNamespace(pa_paged_status=status, pa_attn_status=status,
                                     pa_last_error=lambda: b"copy failed: unspecified launch failure")
        monkeypatch.setattr(_lib, "load", lambda: fake)
    return set_to


def _plans():
    p = object.__new__(paged.PagedPlan)
    p.buffer, p.device = torch.zeros(4, dtype=torch.uint8), 0
    a = object.__new__(attention.AttnPlan)
    a.workspace = torch.zeros(4, dtype=torch.uint8)
    return p, a


@pytest.mark.parametrize("which", [0, 1], ids=["paged", "whole"])
def test_a_status_that_cannot_be_read_is_an_error(answers, which):
    plan = _plans()[which]
    for rc in (_lib.PA_ERR_CUDA, _lib.PA_ERR_ARG):
        answers(rc, 0)
        with pytest.raises(_lib.PolyattnError, match="copy failed") as e:
            plan.status()
        assert e.value.code == rc


@pytest.mark.parametrize("which", [0, 1], ids=["paged", "whole"])
def test_a_recorded_code_is_returned(answers, which):
    plan = _plans()[which]
    answers(_lib.PA_OK, 0)
    assert plan.status() == 0
    answers(_lib.PA_ERR_DEVICE, 5)
    assert plan.status() == 5
