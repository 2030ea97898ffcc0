"""How a few sorted pairs are cut into tiles from their experts' ids: the arithmetic of
w4_rules.hpp, compiled for the host and replayed lane by lane (no GPU)."""
import ctypes
import random
import subprocess

import pytest

from baracuda_amd import build as B
from tests import w4_few

SOURCE = r"""
#include "w4_rules.hpp"
using namespace bk::w4;

// Every tile that a kernel of TB rows finds: expert, first position and rows.
template <int TB>
static int tiles(const int *ids, int size_m, int experts, int *out) {
    int id[kFewPairs], from = 0, n = 0;
    uint64_t head[kFewChunks] = {};
    for (int p = 0; p < kFewPairs; ++p) id[p] = p < size_m ? ids[p] : -1;
    for (int p = 0; p < kFewPairs; ++p)
        if (id[p] != (p ? id[p - 1] : -2)) head[p / 64] |= 1ull << (p % 64);
    for (int i = 0; i < kFewChunks; ++i) {
        for (int l = 0; l < 64; ++l) {
            const int p = 64 * i + l;
            if ((unsigned)id[p] >= (unsigned)experts || (p - run_began(head[i], i, l, from)) % TB) continue;
            out[3 * n] = id[p], out[3 * n + 1] = p;
            out[3 * n++ + 2] = std::min(std::min(TB, run_left<TB>(head, i, l)), size_m - p);
        }
        from = run_began(head[i], i, 63, from);
    }
    return n;
}

extern "C" int tiles_of(int tb, const int *ids, int size_m, int experts, int *out) {
    switch (tb) {
        case 2: return tiles<2>(ids, size_m, experts, out);
        case 4: return tiles<4>(ids, size_m, experts, out);
        case 8: return tiles<8>(ids, size_m, experts, out);
        case 16: return tiles<16>(ids, size_m, experts, out);
        case 32: return tiles<32>(ids, size_m, experts, out);
        case 64: return tiles<64>(ids, size_m, experts, out);
        case 128: return tiles<128>(ids, size_m, experts, out);
        case 192: return tiles<192>(ids, size_m, experts, out);
        case 256: return tiles<256>(ids, size_m, experts, out);
    }
    return -1;
}

extern "C" int few_pairs() { return kFewPairs; }
// The shape that few pairs take; -1 where they take the kernel of few rows.
extern "C" int tile_of(int pairs, int experts, int n, int k) {
    return moe_rows_pay(pairs, experts, n) ? -1 : (int)tile_shape(pairs, experts, n, k);
}
extern "C" int tile_rows_of(int shape) { return kTileCost[shape].tm; }
"""


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    d = tmp_path_factory.mktemp("w4_few")
    (d / "few.cpp").write_text(SOURCE)
    cmd = [B.CXX, "-O1", "-std=c++17", "-fPIC", "-shared", f"-I{B.CSRC}", str(d / "few.cpp"), "-o", str(d / "few.so")]
    res = subprocess.run(cmd, capture_output=True, text=True)
    assert res.returncode == 0, res.stderr
    return ctypes.CDLL(str(d / "few.so"))


def _tiles(rules, tb, ids, experts):
    out = (ctypes.c_int * (3 * 256))()
    n = rules.tiles_of(tb, (ctypes.c_int * len(ids))(*ids), len(ids), experts, out)
    return [tuple(out[3 * i:3 * i + 3]) for i in range(n)]


def _expected(tb, counts):
    """Each expert's run in pieces of tb rows."""
    tiles, at = [], 0
    for e, c in enumerate(counts):
        tiles += [(e, at + i, min(tb, c - i)) for i in range(0, c, tb)]
        at += c
    return tiles


def _ids(counts, none=0):
    return [e for e, c in enumerate(counts) for _ in range(c)] + [len(counts)] * none


def _splits():
    yield from (([c], 0) for c in range(1, 257))
    yield from (([a, b], 0) for a in range(0, 257, 3) for b in range(0, 257 - a, 7) if a + b)
    rng = random.Random(3)
    for _ in range(4000):
        experts, pairs, none = rng.randint(1, 12), rng.randint(1, 256), rng.choice((0, 0, 0, 5, 70))
        pairs = min(pairs, 256 - none)
        cuts = sorted(rng.randint(0, pairs) for _ in range(experts - 1))
        yield [b - a for a, b in zip([0, *cuts], [*cuts, pairs])], none
    yield [0] * 1023 + [256], 0
    yield [1 if i % 4 == 0 else 0 for i in range(1024)], 0


@pytest.mark.parametrize("tb", [2, 4, 8, 16, 32, 64, 128, 192, 256])
def test_every_pair_is_in_one_tile(rules, tb):
    for counts, none in _splits():
        assert _tiles(rules, tb, _ids(counts, none), len(counts)) == _expected(tb, counts), (counts, none)


def test_cases_take_their_shapes(rules):
    for shape, cases in w4_few.CASES.items():
        for counts, none, n, k in cases:
            assert rules.tile_of(sum(counts) + none, len(counts), n, k) == shape, (counts, n, k)


def test_runs_reach_far_chunks(rules):
    """Each height of more than 64 rows has a tile that begins inside a chunk and ends
    behind the next one, or would if it were cut there."""
    for shape, cases in w4_few.CASES.items():
        tb = rules.tile_rows_of(shape)
        ends = [(p, p + r) for counts, none, *_ in cases for _, p, r in _tiles(rules, tb, _ids(counts, none), len(counts))]
        assert tb <= 64 or any(p % 64 and end > p // 64 * 64 + 128 for p, end in ends), shape


def test_shapes_are_all_there_are(rules):
    """No sizes of few pairs take a shape that the cases lack, nor a height not replayed."""
    rng, found = random.Random(2), set()
    for _ in range(60000):
        pairs, experts = rng.randint(1, 256), int(2 ** rng.uniform(0, 6))
        n, k = int(2 ** rng.uniform(6, 16.5)), max(32, int(2 ** rng.uniform(0, 14)) // 32 * 32)
        found.add(rules.tile_of(pairs, experts, n, k))
    assert found - {-1} <= set(w4_few.CASES)
    assert {rules.tile_rows_of(shape) for shape in found - {-1}} <= {32, 64, 128, 192, 256}
    assert rules.few_pairs() == 256
