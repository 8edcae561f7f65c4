"""The embedding operators' host side: the rotary table and the binding (no GPU)."""

import ctypes
import math
import os
import re

import numpy as np
import pytest

from browservec_amd import _lib as L
from browservec_amd import rotary_table

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def want(rows, freq, mag=1.0):
    a = np.arange(rows, dtype=np.float64)[:, None] * freq
    return np.stack([mag * np.cos(a), mag * np.sin(a)], -1)


@pytest.mark.parametrize("rot", [2, 6, 64, 128])
def test_rotary_table(rot):
    f = 10000.0 ** (-np.arange(0, rot, 2) / rot)
    rows = 70000
    # 64-bit frequencies off by a few 2^-53: angles up to 7e4 by 1e-10
    tol = dict(rtol=2.0 ** -23, atol=1e-9)
    np.testing.assert_allclose(rotary_table(rows, rot), want(rows, f), **tol)
    np.testing.assert_allclose(rotary_table(500, rot, scaling="linear", factor=8.0), want(500, f / 8), **tol)
    np.testing.assert_allclose(rotary_table(500, rot, base=500.0, magnitude=1.25), want(500, 500.0 ** (-np.arange(0, rot, 2) / rot), 1.25), **tol)
    if rot > 2:
        b = 10000.0 * 4.0 ** (rot / (rot - 2))
        np.testing.assert_allclose(rotary_table(500, rot, scaling="base", factor=4.0), want(500, b ** (-np.arange(0, rot, 2) / rot)), **tol)
    turns = 2048 * f / (2 * math.pi)
    g = np.clip((turns - 1) / (32 - 1), 0, 1)
    got = rotary_table(500, rot, scaling="parts", factor=4.0, original_rows=2048, low_turns=1, high_turns=32)
    np.testing.assert_allclose(got, want(500, f * (g + (1 - g) / 4)), **tol)


def test_rotary_table_empty_and_refusals():
    assert rotary_table(0, 8).shape == (0, 4, 2) and rotary_table(3, 0).shape == (3, 0, 2)
    for kw in (dict(rot_dim=3), dict(base=0.0), dict(base=float("nan")), dict(scaling="other"), dict(scaling="linear", factor=0.0),
               dict(scaling="base", rot_dim=2, factor=2.0), dict(scaling="parts", factor=2.0), dict(rows=-1),
               dict(scaling="parts", factor=2.0, original_rows=100, low_turns=5, high_turns=5), dict(magnitude=float("inf"))):
        with pytest.raises(L.BVError) as e:
            rotary_table(**{"rows": 4, "rot_dim": 8, **kw})
        assert e.value.code == L.BV_E_INVALID and str(e.value)


def test_argument_structs_match_the_header():
    text = open(os.path.join(ROOT, "include", "browservec_hip.h")).read()
    ctype = {"uint32_t": ctypes.c_uint32, "uint64_t": ctypes.c_uint64, "float": ctypes.c_float, "double": ctypes.c_double}
    for struct, cls in (("linear_args", L.LinearArgs), ("rotary_args", L.RotaryArgs), ("rotary_scaling", L.RotaryScaling),
                        ("attention_args", L.AttentionArgs), ("norm_args", L.NormArgs)):
        body = re.search(r"typedef struct bv_embed_%s \{(.*?)\} bv_embed_%s;" % (struct, struct), text, re.S).group(1)
        fields = re.findall(r"([\w ]+?\s*\*?)(\w+);", re.sub(r"/\*.*?\*/", "", body, flags=re.S))
        assert [n for _, n in fields] == [n for n, _ in cls._fields_], struct
        for (t, n), (_, got) in zip(fields, cls._fields_):
            assert got is (ctypes.c_void_p if "*" in t else ctype[t.strip()]), (struct, n)


def test_refusals_before_any_device():
    lib = L.load()
    for fn in (lib.bv_embed_linear, lib.bv_embed_rotary, lib.bv_embed_attention, lib.bv_embed_norm):
        assert fn(None, None) == L.BV_E_INVALID and lib.bv_last_error()
    assert lib.bv_embed_create(None, None) == L.BV_E_INVALID
    assert lib.bv_embed_destroy(None) == L.BV_OK
    assert lib.bv_embed_sync(None) == L.BV_E_INVALID and lib.bv_embed_set_stream(None, None) == L.BV_E_INVALID
