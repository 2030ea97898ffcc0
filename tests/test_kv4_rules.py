"""Which kernel attention over 4-bit pages takes: the rules of kv4_rules.hpp, compiled for
the host (no GPU), on the cases that the GPU tests run and against the library's sizes."""
import ctypes
import random
import subprocess

import pytest

from baracuda_amd import build as B
from baracuda_amd import ffi
from tests import kv4_forms
from tests.kv4_forms import CASES, FORMS, HK, case_id

SOURCE = r"""
#include "kv4_rules.hpp"
extern "C" {
void cut_of(int num_seqs, int max_q, int64_t max_kv, int ratio, int hk, int D, int window, int64_t *out) {
    const bk::kv4::Cut c = bk::kv4::cut_of(num_seqs, max_q, max_kv, ratio, hk, D, window);
    out[0] = c.rows, out[1] = c.wide, out[2] = c.slots, out[3] = (int64_t)c.bytes, out[4] = c.row_blocks, out[5] = c.grid;
}
}
"""


@pytest.fixture(scope="module")
def cut_of(tmp_path_factory):
    d = tmp_path_factory.mktemp("kv4_rules")
    (d / "rules.cpp").write_text(SOURCE)
    cmd = [B.CXX, "-O1", "-std=c++17", "-fPIC", "-shared", f"-I{B.CSRC}", str(d / "rules.cpp"), "-o", str(d / "rules.so")]
    res = subprocess.run(cmd, capture_output=True, text=True)
    assert res.returncode == 0, res.stderr
    lib = ctypes.CDLL(str(d / "rules.so"))
    lib.cut_of.argtypes = [ctypes.c_int, ctypes.c_int, ctypes.c_int64, *[ctypes.c_int] * 4, ctypes.POINTER(ctypes.c_int64)]

    def f(*sizes):
        out = (ctypes.c_int64 * 6)()
        lib.cut_of(*sizes, out)
        return dict(zip(("rows", "wide", "slots", "bytes", "row_blocks", "grid"), out))

    return f


@pytest.mark.parametrize("case", CASES, ids=case_id)
def test_case_takes_its_form(cut_of, case):
    form, d, (_, _, windowed), _ = case
    window = form.window() if windowed else 0
    c = cut_of(form.seqs, form.max_q, form.max_kv, form.ratio, HK, d, window)
    assert (c["rows"], bool(c["wide"]), c["slots"] > 0) == (form.block_rows(d), form.wide, form.cut)
    assert ffi.lib().kv4_attention_gfx950_workspace_size(form.seqs, form.max_q, form.max_kv, HK * form.ratio, HK, d,
                                                         window) == c["bytes"]


def test_forms_are_all_there_are(cut_of):
    """No sizes take a form that the cases lack."""
    known = {(f.block_rows(d), f.wide, f.cut, d) for f in FORMS for d in (64, 128, 256)}
    rng = random.Random(1)
    found = set()
    for _ in range(60000):
        d, hk = rng.choice((64, 128, 256)), rng.choice((1, 2, 8))
        sizes = (int(2 ** rng.uniform(0, 12)), int(2 ** rng.uniform(0, 12)), int(2 ** rng.uniform(0, 18)), rng.randint(1, 16), hk, d,
                 rng.choice((0, 0, int(2 ** rng.uniform(0, 14)))))
        c = cut_of(*sizes)
        found.add((c["rows"], bool(c["wide"]), c["slots"] > 0, d))
        assert c["grid"] >= sizes[0] * c["row_blocks"] * hk and (not c["slots"] or c["grid"] % hk == 0)
        assert ffi.lib().kv4_attention_gfx950_workspace_size(*sizes[:3], hk * sizes[3], hk, d, sizes[6]) == c["bytes"]
    assert found == known


def test_refills_lie_within_the_longest_sequence():
    for f in FORMS:
        for tokens in f.refill.values():
            assert f.lens[0] > tokens + 100 and not f.cut
    assert {(f.rows, f.wide) for f in FORMS if not f.cut} == {(f.rows, f.wide) for f in FORMS if f.refill}
    assert len({case_id(c) for c in CASES}) == len(CASES) and kv4_forms.HK == 2
