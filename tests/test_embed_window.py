"""What EmbedOps.attention makes of a window and first keys before it calls the
library (no GPU)."""

import ctypes
from types import SimpleNamespace

import pytest
import torch

from browservec_amd import EmbedOps
from browservec_amd import _lib as L


@pytest.fixture
def ops():
    """An EmbedOps whose device is the CPU (get_device() -1) and whose calls end ahead of
    the library."""
    e = object.__new__(EmbedOps)
    e._ordinal, e._int32, e._empty, e._empty_like = -1, torch.int32, torch.empty, torch.empty_like
    e._dtypes = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
    a = L.AttentionArgs(ctypes.sizeof(L.AttentionArgs))
    e._attention, e.lib, e.handle = (a, ctypes.addressof(a)), SimpleNamespace(bv_embed_attention=None), None
    e.calls = []
    e._call = lambda fn, address: e.calls.append((a.window, a.window_left, a.window_right, a.sinks))
    return e


def attend(ops, **kw):
    q = torch.zeros(4, 2, 8, dtype=torch.float16)
    return ops.attention(q, q, q, torch.tensor([0, 4], dtype=torch.int32), **kw)


@pytest.mark.parametrize("window", [None, (3, 0)])
def test_first_keys_are_checked_with_and_without_a_window(ops, window):
    for sinks in (-1, -2 ** 40):
        with pytest.raises(L.BVError) as e:
            attend(ops, window=window, sinks=sinks)
        assert e.value.code == L.BV_E_INVALID and str(e.value)
    for sinks in (1.5, "four", (1,)):
        with pytest.raises(TypeError):
            attend(ops, window=window, sinks=sinks)
    assert not ops.calls
    for sinks in (0, 5, 2 ** 40, None):
        attend(ops, window=window, sinks=sinks)
    most = 2 ** 32 - 1
    if window is None:
        assert [c[0] for c in ops.calls] == [0] * 4
    else:
        assert ops.calls == [(1, 3, 0, s) for s in (0, 5, most, most)]
