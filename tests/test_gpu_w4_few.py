"""Few pairs of a mixture in tiles of every shape, found from the ids: each pair has its row."""
import pytest
import torch

from tests import w4_few
from tests import w4_plain as plain
from tests.test_gpu_w4 import BF, F16, _grouped

pytestmark = pytest.mark.gpu

ALL = [(shape, case) for shape, cases in w4_few.CASES.items() for case in cases]


@pytest.mark.parametrize("shape,case", ALL, ids=lambda v: str(v) if isinstance(v, int) else "-".join(map(str, (*v[0], *v[1:]))))
def test_every_pair_has_its_row(gpu, shape, case):
    counts, none, n, k = case
    ok, why = plain.close(*_grouped(counts, n, k, BF, False, 1, False, n % 2 == 0, seed=n + k, none=none))
    assert ok, why
    ok, why = plain.close(*_grouped(counts, n // 64 * 64, k, F16, True, min(2, len(counts)), True, n % 2 == 1, seed=n, none=none))
    assert ok, why
