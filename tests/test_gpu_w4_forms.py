"""Every form of the kernels of products with 4-bit weights on a case of its own."""
import random

import pytest
import torch

from tests import w4_forms
from tests import w4_plain as plain
from tests.test_gpu_w4 import BF, F16, _grouped, _linear

pytestmark = pytest.mark.gpu


def _id(item):
    return "-".join(map(str, item[0]))


@pytest.mark.parametrize("item", w4_forms.LINEAR.items(), ids=_id)
def test_linear_form(gpu, item):
    form, (m, n, k, gated) = item
    dtype = F16 if sum(map(int, form[1:])) % 2 else BF
    ok, why = plain.close(*_linear(m, n, k, dtype, gated, True, seed=m + n + k))
    assert ok, why
    if form[0] == "tile":       # the shape goes by the sizes: the other end of the product too
        ok, why = plain.close(*_linear(m, n if gated else -(-n // 64) * 64, k, BF, not gated, False, seed=m + n))
        assert ok, why


def _counts(pairs, experts, rng):
    """An uneven split, the last expert's and about a fifth of the others' share empty."""
    share = [rng.random() ** 3 * (rng.random() > 0.2) for _ in range(experts)]
    if experts > 1:
        share[-1] = 0.0
    share[0] += 0.1
    counts = [int(pairs * s / sum(share)) for s in share]
    counts[0] += pairs - sum(counts)
    return counts


@pytest.mark.parametrize("item", w4_forms.MOE.items(), ids=_id)
def test_moe_form(gpu, item):
    form, (pairs, experts, n, k, gated) = item
    dtype = F16 if sum(map(int, form[1:])) % 2 else BF
    counts = _counts(pairs, experts, random.Random(pairs))
    mix = not gated and form[1] % 2 == 0
    ok, why = plain.close(*_grouped(counts, n, k, dtype, gated, min(2, experts), mix, True, seed=n + k))
    assert ok, why
    if form[0] == "tile":
        ok, why = plain.close(*_grouped(counts, n if gated else -(-n // 64) * 64, k, BF, not gated, 1, gated, False, seed=n))
        assert ok, why


@pytest.mark.parametrize("experts,pairs", [(3, 65), (5, 64), (9, 256), (200, 255), (1024, 130), (2, 200), (7, 63)])
def test_few_pairs_found_from_the_ids(gpu, experts, pairs):
    """Runs of an expert that end at, begin at and pass every boundary of 64 positions."""
    rng = random.Random(experts)
    counts = _counts(pairs, experts, rng)
    ok, why = plain.close(*_grouped(counts, 33, 96, BF, False, 1, False, False, seed=experts))
    assert ok, why
    one = [0] * (experts - 1) + [pairs]
    ok, why = plain.close(*_grouped(one, 33, 96, BF, False, 1, False, False, seed=experts))
    assert ok, why
    if experts < 50:      # wide enough for tiles
        ok, why = plain.close(*_grouped(counts, 4161, 96, BF, False, 1, False, True, seed=experts, none=min(3, 256 - pairs)))
        assert ok, why
        ok, why = plain.close(*_grouped(one, 4224, 160, F16, True, 1, True, False, seed=experts))
        assert ok, why


@pytest.mark.parametrize("m", [0, 1])
def test_nothing_to_do(gpu, m):
    """No tokens, no pairs: no output, but the counts."""
    from baracuda_amd import w4
    packed = torch.zeros(4, w4.packed_bytes(64, 64), dtype=torch.uint8, device=gpu)
    w4.W4LinearPlan.select(w4.W4LinearDescriptor(0, 64, 64)).run(torch.empty(0, 64, dtype=BF, device=gpu), packed[0],
                                                                 torch.empty(0, 64, dtype=BF, device=gpu))
    counts, offsets = (torch.full((c,), 7, dtype=torch.int32, device=gpu) for c in (4, 5))
    ids = torch.full((m,), 4, dtype=torch.int32, device=gpu)
    out = torch.full((m, 64), 3.0, dtype=BF, device=gpu)
    w4.MoeW4GroupedPlan.select(w4.MoeW4GroupedDescriptor(4, 1, m, 64, 64)).run(
        torch.zeros(m, 64, dtype=BF, device=gpu), packed, torch.zeros(m, dtype=torch.int32, device=gpu), ids, out, counts, offsets)
    assert not counts.any() and not offsets.any() and bool((out == 3).all())


def test_two_streams_at_once(gpu):
    """One plan's calls on two streams, with other inputs each."""
    from baracuda_amd import w4
    from tests.test_gpu_w4 import _gen, _packed, _randn
    n, k, m, g = 1024, 2048, 90, _gen(4)
    codes, scales = plain.checkpoint(g, 1, n, k)
    packed, xs = _packed(codes, scales), [_randn(g, m, k).to(BF) for _ in range(8)]
    outs = [torch.zeros(m, n, dtype=BF, device=gpu) for _ in xs]
    plan = w4.W4LinearPlan.select(w4.W4LinearDescriptor(m, n, k))
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for i, (x, out) in enumerate(zip(xs, outs)):
        plan.run(x, packed, out, stream=streams[i % 2])
    torch.cuda.synchronize()
    for x, out in zip(xs, outs):
        ok, why = plain.close(out, *plain.product(x, plain.values(codes, scales)[0]))
        assert ok, why


def test_output_past_32_bits(gpu):
    """More than 2^31 elements of output; the last rows are the last rows' product."""
    from baracuda_amd import w4
    from tests.test_gpu_w4 import _gen, _packed, _randn
    m, n, k, g = 66001, 33000, 32, _gen(5)
    codes, scales = plain.checkpoint(g, 1, n, k)
    x = _randn(g, m, k).to(BF)
    out = torch.empty(m, n, dtype=BF, device=gpu)
    w4.W4LinearPlan.select(w4.W4LinearDescriptor(m, n, k)).run(x, _packed(codes, scales), out)
    for rows in (slice(0, 3), slice(m // 2, m // 2 + 3), slice(m - 40, m)):
        ok, why = plain.close(out[rows], *plain.product(x[rows], plain.values(codes, scales)[0]))
        assert ok, why


@pytest.mark.parametrize("pairs", [3, 400])
def test_weights_past_32_bits(gpu, pairs):
    """An expert that lies behind 4 GiB of others."""
    from baracuda_amd import w4
    from tests.test_gpu_w4 import _gen, _packed, _randn
    e, n, k, g = 3, 131072, 32768, _gen(6)
    codes, scales = plain.checkpoint(g, e, n, k)
    packed = _packed(codes, scales)
    assert 2 * packed.shape[1] > 2 ** 32
    x = _randn(g, pairs, k).to(BF)
    i32 = dict(dtype=torch.int32, device=gpu)
    ids = torch.full((pairs,), 2, **i32)
    out = torch.empty(pairs, n, dtype=BF, device=gpu)
    w4.MoeW4GroupedPlan.select(w4.MoeW4GroupedDescriptor(e, 1, pairs, n, k)).run(
        x, packed, torch.arange(pairs, **i32), ids, out, torch.empty(e, **i32), torch.empty(e + 1, **i32))
    for rows in (slice(0, 50), slice(n - 50, n)):
        want, error = plain.product(x, plain.values(codes[2, rows], scales[2, rows]))
        ok, why = plain.close(out[:, rows], want, error)
        assert ok, why
