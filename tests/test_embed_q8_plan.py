"""Which shapes of tile linear_q8's plan chooses for the sizes that the GPU tests run
(no GPU: the plan is plain C++, compiled here by itself)."""

import ctypes
import os
import subprocess

import pytest

from tests.test_gpu_embed_q8_tiles import TILES

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SOURCE = """
#include "%s"
extern "C" int shapes(uint32_t (*out)[3]) {
    for (int i = 0; i < bvk::Q8_SHAPES; i++) out[i][0] = bvk::q8_shapes[i].bm, out[i][1] = bvk::q8_shapes[i].bn, out[i][2] = bvk::q8_shapes[i].bk;
    return bvk::Q8_SHAPES;
}
extern "C" void plan(uint64_t m, uint32_t n, uint32_t k, int act, uint64_t *out) {
    const bvk::Q8Plan p = bvk::q8_plan(m, n, k, act);
    out[0] = p.shape, out[1] = p.rows, out[2] = p.then;
}
"""


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    at = tmp_path_factory.mktemp("plan")
    (at / "plan.cpp").write_text(SOURCE % os.path.join(ROOT, "browservec_amd", "csrc", "bv_linear_q8_plan.h"))
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Wextra", "-Werror", "-shared", "-fPIC", str(at / "plan.cpp"), "-o", str(at / "plan.so")],
                   check=True)
    lib = ctypes.CDLL(str(at / "plan.so"))
    lib.plan.argtypes = [ctypes.c_uint64, ctypes.c_uint32, ctypes.c_uint32, ctypes.c_int, ctypes.c_void_p]
    return lib


def shapes_of(lib):
    out = (ctypes.c_uint32 * 3 * 64)()
    return [tuple(s) for s in out[:lib.shapes(out)]]


def plan(lib, m, n, k, act):
    out = (ctypes.c_uint64 * 3)()
    lib.plan(m, n, (k + 15) // 16 * 16, {"none": 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}[act], out)
    return list(out)


def test_every_shape_is_run_and_ragged(lib):
    shapes = shapes_of(lib)
    alone, first, then = set(), set(), set()
    steps = {i: set() for i in range(len(shapes))}
    for m, n, k, act in TILES:
        shape, rows, behind = plan(lib, m, n, k, act)
        assert 0 < rows <= m
        last = shape if rows == m else behind
        bm, bn, bk = shapes[last]
        if (m - (0 if rows == m else rows)) % bm and n % bn and n % 8 and k % 16 and (k + 15) // 16 * 16 % bk:
            (alone if rows == m else then).add(last)
        if rows < m:
            first.add(shape)
            assert rows % shapes[shape][0] == 0
        steps[shape].add(-(-k // shapes[shape][2]))
        steps[last].add(-(-k // bk))
    assert alone == set(range(len(shapes))), alone
    assert len(first) >= 4 and len(then) >= 5, (first, then)
    # loops that end as they begin, and loops that use every buffer again
    assert all(max(s) >= 5 for s in steps.values()), steps
    assert sum(min(s) <= 2 for s in steps.values()) >= 6, steps


def test_the_plan_covers_all_rows(lib):
    for m in (33, 64, 100, 2037, 16492, 20011, 32768, 2 ** 24 + 5, 2 ** 31):
        for n in (1, 17, 768, 1000, 4096, 2 ** 20 + 1, 2 ** 32 - 1):
            for k in (0, 1, 768, 4096, 131071):
                for act in ("none", "gelu"):
                    shape, rows, behind = plan(lib, m, n, k, act)
                    assert shape < 8 and behind < 8 and 0 < rows <= m
