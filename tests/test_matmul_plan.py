"""The launch rule of the fine-tuning operators' matrix product, and what its test entry refuses (host code only)."""
import ctypes

import pytest

from interior_amd import _lib
from test_finetune import FAKE, linear_args


def plan(m, n, k):
    """[(rows, tile, slices, k-tiles a slice)] of C [m, n] over k."""
    parts, count = (_lib.MatmulPart * 2)(), ctypes.c_int()
    _lib.check(_lib.lib().clipvit_matmul_plan_test(m, n, k, parts, ctypes.byref(count)))
    return [(p.rows, p.tile, p.slices, p.kslice) for p in parts[:count.value]]


# rows, in and out features of a Linear, and the launches of y, dx and dw. tests/test_gpu_matmul_tiles.py runs these, and needs
# 256-wide tiles of many k-tiles, unequal slices and remaining rows: a rule that no longer gives them there needs other sizes.
RULE = {
    "rest in slices": (4160, 2040, 4096, [(4096, 256, 1, 32), (64, 64, 4, 8)], [(4160, 256, 1, 64)], [(4096, 128, 1, 65)]),
    "rest in slices, back": (4160, 4096, 2040, [(4160, 256, 1, 64)], [(4096, 256, 1, 32), (64, 64, 4, 8)], [(2040, 128, 1, 65)]),
    "hidden layer": (12608, 1024, 4096, [(12288, 256, 1, 16), (320, 64, 1, 16)], [(12608, 256, 1, 64)], [(4096, 256, 4, 50)]),
    "hidden layer, back": (12608, 4096, 1024, [(12608, 256, 1, 64)], [(12288, 256, 1, 16), (320, 64, 1, 16)], [(1024, 256, 4, 50)]),
    "ragged everywhere": (4104, 4088, 4072, [(4096, 256, 1, 64), (8, 64, 8, 8)], [(4096, 256, 1, 64), (8, 64, 8, 8)], [(4072, 256, 1, 65)]),
}


@pytest.mark.parametrize("name", RULE)
def test_rule(name):
    m, k, n, y, dx, dw = RULE[name]
    assert plan(m, n, k) == y and plan(m, k, n) == dx and plan(n, k, m) == dw


def test_rule_covers_every_row_and_k_tile():
    for m in (1, 63, 64, 257, 5000, 36928):
        for n in (1, 437, 1024, 4096):
            for k in (0, 1, 64, 513, 4096, 36928):
                parts = plan(m, n, k)
                assert sum(p[0] for p in parts) == m and all(p[0] % 256 == 0 for p in parts[:-1])
                for _, tile, slices, kslice in parts:
                    nk = (k + 63) // 64
                    assert tile in (64, 128, 256) and (slices - 1) * kslice < max(nk, 1) <= max(slices * kslice, 1)


@pytest.mark.parametrize("parts", [[], [(4, 32, 1)], [(4, 64, 0)], [(4, 64, 65)], [(0, 64, 1)], [(5, 64, 1)], [(2, 64, 1), (2, 64, 1)], [(256, 64, 1), (4, 64, 1)]])
def test_chosen_launches_are_checked(parts):
    L, need = _lib.lib(), ctypes.c_size_t()
    chosen = (_lib.MatmulPart * 2)(*(_lib.MatmulPart(*p, 0) for p in parts))
    for out in (ctypes.byref(need), None):
        assert L.clipvit_linear_test(None, ctypes.byref(linear_args()), chosen, len(parts), FAKE, 1 << 20, out) == _lib.E_INVALID
    assert L.clipvit_linear_test(None, ctypes.byref(linear_args()), None, 1, FAKE, 1 << 20, ctypes.byref(need)) == _lib.E_INVALID
    assert L.clipvit_matmul_plan_test(-1, 4, 4, chosen, ctypes.byref(ctypes.c_int())) == _lib.E_INVALID
    assert L.clipvit_matmul_plan_test(4, 4, 4, None, ctypes.byref(ctypes.c_int())) == _lib.E_INVALID


def test_chosen_launches_need_their_workspace():
    L, need = _lib.lib(), ctypes.c_size_t()
    chosen = (_lib.MatmulPart * 1)(_lib.MatmulPart(4, 64, 2, 0))
    a = linear_args(K=128, x_row=128, w_row=128)
    assert L.clipvit_linear_test(None, ctypes.byref(a), chosen, 1, None, 0, ctypes.byref(need)) == 0 and need.value >= 2 * 4 * 8 * 4
    assert L.clipvit_linear_test(None, ctypes.byref(a), chosen, 1, FAKE, need.value - 1, None) == _lib.E_INVALID
    assert L.clipvit_linear_test(None, ctypes.byref(a), chosen, 1, None, need.value, None) == _lib.E_INVALID
