"""The kernels of few rows with 4-bit weights that are compiled are those that some sizes
take: the rules of w4_rules.hpp, compiled for the host (no GPU)."""
import ctypes
import subprocess

import pytest

from baracuda_amd import build as B

SOURCE = r"""
#include "w4_rules.hpp"
using namespace bk::w4;
// Every held, slots, N and K: workgroups of 16 weight rows and 256-value words alone decide.
extern "C" void taken(int gated, int most, int *out) {      // out: [5 log held][3 log blocks][5 log waves]
    const int words[] = {1, 4, 5, 8, 31, 32, 33, 64};
    for (int held : {2, 4, 8, 16})
        for (int slots : {1, 2, 3, 5, 16})
            for (int n = gated ? 64 : 16; (n / 16) * (int64_t)slots <= most; n += gated ? 64 : 16)
                for (int w : words) {
                    const RowsShape s = rows_shape(held, slots, n, 256 * w, gated);
                    out[(__builtin_ctz(held) * 3 + __builtin_ctz(s.blocks)) * 5 + __builtin_ctz(s.waves)] = 1;
                }
}
extern "C" int form(int held, int blocks, int waves, int gated) { return rows_form(held, blocks, waves, gated); }
"""


@pytest.mark.parametrize("gated", [0, 1])
def test_compiled_forms_are_those_taken(tmp_path, gated):
    (tmp_path / "forms.cpp").write_text(SOURCE)
    cmd = [B.CXX, "-O2", "-std=c++17", "-fPIC", "-shared", f"-I{B.CSRC}", str(tmp_path / "forms.cpp"), "-o", str(tmp_path / "forms.so")]
    res = subprocess.run(cmd, capture_output=True, text=True)
    assert res.returncode == 0, res.stderr
    lib = ctypes.CDLL(str(tmp_path / "forms.so"))
    out = (ctypes.c_int * 75)()
    lib.taken(gated, 5000, out)
    found = {(1 << h, 1 << b, 1 << w) for h in range(5) for b in range(3) for w in range(5) if out[(h * 3 + b) * 5 + w]}
    forms = {(h, b, w) for h in (2, 4, 8, 16) for b in (1, 2, 4) for w in (1, 2, 4, 8, 16) if lib.form(h, b, w, gated)}
    assert found == forms
    assert len(forms) == (21 if gated else 29)
