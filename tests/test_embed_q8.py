"""The host side of the operators in 8 bits and of windows (no GPU)."""

import ctypes
import os
import re

import pytest

from browservec_amd import _lib as L
from browservec_amd import embed

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_argument_structs_match_the_header():
    text = open(os.path.join(ROOT, "include", "browservec_hip.h")).read()
    ctype = {"uint32_t": ctypes.c_uint32, "uint64_t": ctypes.c_uint64, "float": ctypes.c_float}
    for struct, cls in (("linear_q8_args", L.LinearQ8Args), ("add_norm_args", L.AddNormArgs)):
        body = re.search(r"typedef struct bv_embed_%s \{(.*?)\} bv_embed_%s;" % (struct, struct), text, re.S).group(1)
        fields = re.findall(r"([\w ]+?\s*\*?)(\w+);", re.sub(r"/\*.*?\*/", "", body, flags=re.S))
        assert [n for _, n in fields] == [n for n, _ in cls._fields_], struct
        for (t, n), (_, got) in zip(fields, cls._fields_):
            assert got is (ctypes.c_void_p if "*" in t else ctype[t.strip()]), (struct, n)
    before = int(re.search(r"#define BV_EMBED_ATTENTION_ARGS_V1 (\d+)", text).group(1))
    assert L.AttentionArgs.window.offset == before


def test_refusals_before_any_device():
    lib = L.load()
    for fn in (lib.bv_embed_linear_q8, lib.bv_embed_add_norm):
        assert fn(None, None) == L.BV_E_INVALID and lib.bv_last_error()


def test_numbers_of_keys():
    assert [embed._keys(n) for n in (0, 5, 2 ** 32 - 1, 2 ** 32, 2 ** 70, None)] == [0, 5] + [2 ** 32 - 1] * 4
    with pytest.raises(L.BVError) as e:
        embed._keys(-1)
    assert e.value.code == L.BV_E_INVALID
    with pytest.raises(TypeError):
        embed._keys(1.5)
