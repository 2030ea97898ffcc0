"""Which kernel a product with 4-bit weights takes: the rules of w4_rules.hpp, compiled for
the host (no GPU)."""
import ctypes
import random
import subprocess

import pytest

from baracuda_amd import build as B
from tests import w4_forms

SOURCE = r"""
#include "w4_rules.hpp"
using namespace bk::w4;
extern "C" {
void linear_form(int m, int n, int k, int gated, int *out) {
    out[0] = rows_pay(m, n);
    const int held = rows_held(m);
    const RowsShape s = rows_shape(held, (m + held - 1) / held, n, k, gated);
    out[1] = held, out[2] = s.blocks, out[3] = s.waves, out[4] = tile_shape(m, 0, n, k);
}
void moe_form(int pairs, int experts, int n, int k, int gated, int *out) {
    out[0] = moe_rows_pay(pairs, experts, n);
    const int held = moe_rows_held(pairs, experts);
    const RowsShape s = rows_shape(held, moe_rows_likely(pairs, experts, held), n, k, gated);
    out[1] = held, out[2] = s.blocks, out[3] = s.waves, out[4] = tile_shape(pairs, experts, n, k);
}
int64_t workgroups(int shape, int64_t rows, int experts, int n) {
    const TileCost &c = kTileCost[shape];
    return most_tile_rows(rows, experts, c.tm) * ((n + c.tn - 1) / c.tn);
}
}
"""


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    d = tmp_path_factory.mktemp("w4_rules")
    (d / "rules.cpp").write_text(SOURCE)
    cmd = [B.CXX, "-O1", "-std=c++17", "-fPIC", "-shared", f"-I{B.CSRC}", str(d / "rules.cpp"), "-o", str(d / "rules.so")]
    res = subprocess.run(cmd, capture_output=True, text=True)
    assert res.returncode == 0, res.stderr
    lib = ctypes.CDLL(str(d / "rules.so"))
    lib.workgroups.restype = ctypes.c_int64
    lib.workgroups.argtypes = [ctypes.c_int, ctypes.c_int64, ctypes.c_int, ctypes.c_int]
    return lib


def _form(f, *sizes):
    out = (ctypes.c_int * 5)()
    f(*sizes, out)
    return ("rows", *out[1:4]) if out[0] else ("tile", out[4])


def _linear(rules, m, n, k, gated):
    return _form(rules.linear_form, m, n, k, int(gated))


def _moe(rules, pairs, experts, n, k, gated):
    return _form(rules.moe_form, pairs, experts, n, k, int(gated))


def test_cases_take_their_forms(rules):
    for form, (m, n, k, gated) in w4_forms.LINEAR.items():
        assert _linear(rules, m, n, k, gated) == form, (m, n, k, gated)
    for form, (pairs, experts, n, k, gated) in w4_forms.MOE.items():
        assert _moe(rules, pairs, experts, n, k, gated) == form, (pairs, experts, n, k, gated)


@pytest.mark.parametrize("experts,pairs", [(3, 65), (5, 64), (9, 256), (2, 200), (7, 63)])
def test_few_pairs_of_wide_experts_take_tiles(rules, experts, pairs):
    assert _moe(rules, pairs, experts, 4161, 96, False)[0] == _moe(rules, pairs, experts, 4224, 160, True)[0] == "tile"


def test_forms_are_all_there_are(rules):
    """No sizes take a form that the cases lack, and none of the launches is too large."""
    rng = random.Random(1)

    def spread(lo, hi, step=1):
        return max(lo, int(2 ** rng.uniform(0, hi)) // step * step)

    found = {"linear": set(), "moe": set()}
    for _ in range(40000):
        m, n, k, gated = spread(1, 13), spread(64, 16, 64), spread(32, 14, 32), rng.random() < 0.4
        found["linear"].add(_linear(rules, m, n, k, gated))
        pairs, experts = spread(1, 15), spread(1, 9)
        found["moe"].add(_moe(rules, pairs, experts, n, k, gated))
        for rows, e in ((m, 0), (pairs, experts)):
            form = _moe(rules, rows, e, n, k, gated) if e else _linear(rules, rows, n, k, gated)
            if form[0] == "tile":
                assert rules.workgroups(form[1], rows, e, n) <= 1 << 21
            else:
                assert -(-rows // form[1]) + min(e, rows) <= 65535
    assert found["linear"] <= set(w4_forms.LINEAR)
    assert found["moe"] <= set(w4_forms.MOE)
