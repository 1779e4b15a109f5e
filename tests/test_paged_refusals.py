"""More refusals of the paged-cache entry points, without GPU work."""
import ctypes

import pytest

from polyhedral_b200 import _lib
from tests.test_paged_host import PTR, _attn_args, lib  # noqa: F401


@pytest.mark.parametrize("field,word", [("q", b"over q with other strides"), ("k_cache", b"over a cache"),
                                        ("v_cache", b"over a cache")])
def test_results_over_the_inputs(lib, field, word):  # noqa: F811
    a = _attn_args()
    a.o, a.o_token_stride = 4096, 128
    setattr(a, field, 4096)
    for call in (lambda: lib.pa_paged_attn(ctypes.byref(a), PTR, 1 << 30, PTR, 1 << 40, None),
                 lambda: lib.pa_paged_attn_withheld(ctypes.byref(a), PTR, 1 << 30, PTR, 1 << 40,
                                                    2_000_000, None)):
        assert call() == _lib.PA_ERR_ARG
        assert word in lib.pa_last_error()


@pytest.mark.parametrize("limit", [0, -1, 999, 10**9 + 1])
def test_withheld_limits(lib, limit):  # noqa: F811
    a = _attn_args()
    rc = lib.pa_paged_attn_withheld(ctypes.byref(a), PTR, 1 << 30, PTR, 1 << 40, limit, None)
    assert rc == _lib.PA_ERR_ARG and b"wait_limit_ns" in lib.pa_last_error()
