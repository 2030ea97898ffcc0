"""The operators around a 4-bit key-value cache at the ends of what they take."""
import pytest
import torch

from baracuda_amd import kv4
from tests import kv4_plain as plain
from tests.gpu_util import sync
from tests.test_gpu_kv4 import (BF, FL, HF, KIND, _check_attention, _dev, _near, _on_gpu, _plain_rows, _rotation, _rows, _same,
                                _scene)

pytestmark = pytest.mark.gpu


def _attend(scene, hk, max_q, max_kv, causal=True, window=0):
    cache, tables, lens, cu, q = scene
    total, hq, d = q.shape
    plan = kv4.Kv4AttentionPlan.select(kv4.Kv4AttentionDescriptor(
        len(lens), total, max_q, max_kv, hq, hk, d, cache.shape[2] // (d + d // 16), cache.shape[0], tables.shape[1],
        KIND[q.dtype], causal, window))
    ws = torch.full((plan.workspace_size(),), 0x7f, dtype=torch.uint8, device="cuda:0")
    out = torch.full((total, hq, d), 3.0, dtype=q.dtype, device="cuda:0")
    plan.run(_dev(q), _dev(cache), _dev(tables), _dev(lens), out, cu_q=_dev(cu), workspace=ws)
    sync()
    return out.cpu()


# ---- sequences longer than max_q ----------------------------------------------
PAST = [  # sequences, max_q, new tokens of the long one, max_kv, hq, hk, D, causal, window
    (32, 64, 200, 1100, 32, 8, 128, True, 0), (6, 300, 400, 512, 64, 4, 64, True, 0),     # large blocks from both ends
    (32, 64, 200, 1100, 32, 8, 128, True, 80), (32, 64, 150, 1100, 32, 8, 128, False, 0),
    (32, 40, 150, 1100, 32, 8, 256, True, 0), (2, 70, 200, 100000, 8, 2, 128, True, 0),   # the last one cut
    (3, 20, 50, 200, 4, 2, 128, True, 0), (2, 5, 30, 100000, 4, 2, 64, True, 0),          # blocks of 16
    (32, 5, 30, 1100, 32, 8, 128, True, 0)]                                               # blocks of 32


@pytest.mark.parametrize("case", PAST, ids=str)
def test_attention_of_a_sequence_longer_than_max_q(gpu, case):
    """The rows before max_q of every sequence are computed, whatever a sequence has past it."""
    seqs, max_q, n, max_kv, hq, hk, d, causal, window = case
    print(f"past max_q {case}", flush=True)
    qs = [i % 3 for i in range(seqs)]
    qs[1] = n
    lens = [x + 7 * i % 50 for i, x in enumerate(qs)]
    scene = _scene(torch.Generator().manual_seed(n), lens, qs, hq, hk, d, 16, BF)
    cache, tables, lens_t, cu, q = scene
    got = _attend(scene, hk, max_q, max_kv, causal, window)
    past = slice(int(cu[1]) + max_q, int(cu[2]))
    want, size, _ = plain.attention(q, cache, tables, lens_t, cu, causal, window, d ** -0.5)
    # the rows past max_q are not the call's: take them out of the comparison
    got[past] = want[past].to(BF)
    _check_attention(got, q, cache, tables, lens_t, cu, causal, window, d ** -0.5)


# ---- heads and weights at the ends of the range -------------------------------
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("dt", [BF, FL], ids=str)
@pytest.mark.parametrize("t", [5, 520])
def test_qk_products_out_of_range(gpu, dt, t, inter):
    # values and their products with the weights past the largest number, where the
    # normed values are of ordinary size, and heads of the smallest numbers there are
    d, rope = 128, 64
    g = torch.Generator().manual_seed(16)
    x = _rows(g, t, 6, d, FL)
    x[:, 0] = x[:, 0].sign() * 3e38 * (0.5 + 0.5 * torch.rand(t, d, generator=g))
    x[:, 1, ::7] = 3.3e38
    x[:, 3] = x[:, 3].sign() * torch.finfo(dt).max
    x[:, 4] = x[:, 4].sign() * (torch.finfo(dt).tiny * torch.finfo(dt).eps) * torch.randint(1, 9, (t, d), generator=g)
    x[:, 5] *= 1e-30
    x = x.to(dt)
    assert torch.isfinite(x).all()
    w = (1.3 + 0.2 * torch.randn(d, generator=g)).to(dt)
    rot = _rotation(g, t, rope, 1)
    out = [torch.empty(t, 3, d, dtype=dt, device=gpu) for _ in range(2)]
    kv4.QkNormRopePlan.select(kv4.QkNormRopeDescriptor(t, 3, 3, d, rope, KIND[dt], interleaved=inter, eps=0.0)).run(
        _dev(x[:, :3]), _dev(x[:, 3:]), *out, q_weight=_dev(w), k_weight=_dev(w), **_on_gpu(rot))
    for got, part in ((out[0], x[:, :3]), (out[1], x[:, 3:])):
        want, size = _plain_rows(part, w, 0.0, rope, rot, inter)
        _near(got, want, size, dt)


@pytest.mark.parametrize("t", [5, 520])
def test_qk_weights_out_of_range(gpu, t):
    # ordinary heads under large weights, and large ones under those
    d, eps = 128, 1e-6
    g = torch.Generator().manual_seed(17)
    x = _rows(g, t, 2, d, FL)
    x[:, 1] *= 1e16
    x = x.to(BF)
    w = ((1 + 0.2 * torch.randn(d, generator=g)) * 1e25).to(BF)
    rot = _rotation(g, t, 64, 1)
    out = [torch.empty(t, 1, d, dtype=BF, device=gpu) for _ in range(2)]
    kv4.QkNormRopePlan.select(kv4.QkNormRopeDescriptor(t, 1, 1, d, 64, eps=eps)).run(
        _dev(x[:, :1]), _dev(x[:, 1:]), *out, q_weight=_dev(w), k_weight=_dev(w), **_on_gpu(rot))
    for got, part in ((out[0], x[:, :1]), (out[1], x[:, 1:])):
        want, size = _plain_rows(part, w, eps, 64, rot, False)
        _near(got, want, size, BF)


@pytest.mark.parametrize("d,rope,inter", [(64, 64, False), (128, 64, True), (256, 0, False)])
@pytest.mark.parametrize("t", [5, 520])
def test_append_products_out_of_range(gpu, t, d, rope, inter):
    hq, hk, ps = 1, 4, 16
    g = torch.Generator().manual_seed(18)
    x = _rows(g, t, hq + 2 * hk, d, FL)
    x[:, 0] = x[:, 0].sign() * 3e38
    x[:, 1] = x[:, 1].sign() * 3e38 * (0.3 + 0.7 * torch.rand(t, d, generator=g))
    x[:, 2, ::5] = 3.3e38
    x[:, 3] *= 1e-37
    x[:, 4] = x[:, 4].sign() * 2.0 ** -133 * torch.randint(1, 9, (t, d), generator=g)
    x = x.to(BF)
    assert torch.isfinite(x).all()
    w = (1.3 + 0.2 * torch.randn(d, generator=g)).to(BF)
    rot = _rotation(g, t, rope, 1)
    pages = -(-t // ps)
    cache = torch.zeros(pages, hk, kv4.head_bytes(ps, d), dtype=torch.uint8)
    got, q_out = _dev(cache), torch.empty(t, hq, d, dtype=BF, device=gpu)
    kv4.Kv4AppendPlan.select(kv4.Kv4AppendDescriptor(t, hq, hk, d, ps, pages, rope, interleaved=inter, eps=0.0)).run(
        _dev(x[:, hq:hq + hk]), _dev(x[:, hq + hk:]), got, _dev(torch.arange(t)), q=_dev(x[:, :hq]), q_out=q_out,
        q_weight=_dev(w), k_weight=_dev(w), **_on_gpu(rot))
    want, size = _plain_rows(x[:, :hq], w, 0.0, rope, rot, inter)
    _near(q_out, want, size, BF)
    k = _plain_rows(x[:, hq:hq + hk], w, 0.0, rope, rot, inter)[0].float().to(BF)
    for i in range(t):
        for h in range(hk):
            plain.put(cache, i, h, k[i, h], x[i, hq + hk + h], plain.most(BF))
    _same(got, cache, "cache")


# ---- windows --------------------------------------------------------------------
WINDOWS = [([40], [64], 4, 2, 64, 200), ([40], [64], 4, 2, 64, 2_000_000), ([3, 0, 30], [9, 5, 30], 16, 2, 128, 900),
           ([600, 5], [257, 129], 8, 2, 256, 2_000_000)]


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 60])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("case", WINDOWS, ids=str)
def test_attention_windows_that_hide_nothing(gpu, case, causal, window):
    """The widest windows, also with more new tokens than the cache holds."""
    lens, qs, hq, hk, d, max_kv = case
    scene = _scene(torch.Generator().manual_seed(sum(qs)), lens, qs, hq, hk, d, 16, BF)
    cache, tables, lens_t, cu, q = scene
    got = _attend(scene, hk, max(qs), max_kv, causal, window)
    _check_attention(got, q, cache, tables, lens_t, cu, causal, 0, d ** -0.5)


@pytest.mark.parametrize("d,dt", [(64, HF), (128, BF), (256, BF)], ids=str)
@pytest.mark.parametrize("seqs,max_q,max_kv", [(1, 1, 300), (1, 1, 100000), (2, 1, 600), (32, 20, 1100), (2, 64, 2_000_000)])
def test_attention_window_without_causal(gpu, d, dt, seqs, max_q, max_kv):
    """A window w hides what lies w or more positions before the row's own; the
    positions after it are hidden by `causal` alone.  The same tokens are hidden here
    by taking their pages out of the table, without a window."""
    ps, hq, hk, n = 16, 8, 2, 3
    lens, qs = [410] + [0] * (seqs - 1), [n] + [0] * (seqs - 1)
    if max_q == 1:
        n = qs[0] = 1
    cache, tables, lens_t, cu, q = _scene(torch.Generator().manual_seed(d), lens, qs, hq, hk, d, ps, dt)
    for i in range(n):           # row i stands at 410 - n + i: windows that begin with a page
        first = 11 * ps
        window = lens[0] - n + i - first + 1
        got = _attend((cache, tables, lens_t, cu, q), hk, max_q, max_kv, causal=False, window=window)
        cut = tables.clone()
        cut[0, :11] = -1
        one = torch.tensor([0, 1] + [1] * (seqs - 1), dtype=torch.int32)
        _check_attention(got[i:i + 1], q[i:i + 1], cache, cut, lens_t, one, False, 0, d ** -0.5)


# ---- sums of large values ---------------------------------------------------------
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("ratio,n,max_kv", [(1, 1, 200), (4, 1, 600), (4, 1, 100000), (4, 5, 2_000_000), (8, 9, 2_000_000),
                                            (32, 70, 2_000_000)])
def test_attention_of_values_near_the_largest(gpu, d, ratio, n, max_kv):
    """Values whose weighted sum is in range where the sum of their products with
    weights that are not divided yet is not; and others that are all very small."""
    lens, qs, ps = [700], [n], 16
    cache, tables, lens_t, cu, q = _scene(torch.Generator().manual_seed(d), lens, qs, 2 * ratio, 2, d, ps, BF)
    vs = plain.places(ps, d)[3]
    for byte in (252, 45):
        cache[:, :, vs] = byte
        cache[:, :, vs[:, ::2]] = byte - 3
        scene = cache, tables, lens_t, cu, q
        got = _attend(scene, 2, n, max_kv)
        assert torch.isfinite(got).all(), byte
        _check_attention(got, q, cache, tables, lens_t, cu, True, 0, d ** -0.5)


def test_attention_of_the_largest_value_everywhere(gpu):
    lens, qs, ps, d = [3000, 20], [1, 1], 16, 128
    cache, tables, lens_t, cu, q = _scene(torch.Generator().manual_seed(1), lens, qs, 8, 2, d, ps, BF, garbage=False)
    cache[:, :, ps * d // 2:ps * d] = 0x77
    cache[:, :, plain.places(ps, d)[3]] = 252
    got = _attend((cache, tables, lens_t, cu, q), 2, 1, 3000).double()
    most = 6 * 2.0 ** 125
    assert ((got - most).abs() <= 2 * plain.half_step(BF) * most).all()


# ---- pages -------------------------------------------------------------------------
@pytest.mark.parametrize("size", [32, 20000])
def test_pages_fork_of_a_row_that_is_a_child_too(gpu, size):
    """Which the caller must not ask for: what the two rows hold then is open, but nothing
    past the tables is read and no page but the one handed out is written."""
    g = torch.Generator().manual_seed(size)
    cache = torch.randint(0, 256, (2, 9, size), generator=g, dtype=torch.uint8)
    tables = torch.tensor([[0, 1], [-1, -1], [4, 5]], dtype=torch.int32)
    lens, refs = torch.tensor([8, 0, 5], dtype=torch.int32), torch.tensor([1, 1, 0, 0, 1, 1, 0, 0, 0], dtype=torch.int32)
    dev = [_dev(x) for x in (cache, tables, lens, refs)]
    fresh = torch.empty(2, dtype=torch.int32, device=gpu)
    # the last row is read by the first fork and becomes a full one by the second
    kv4.KvPagesPlan.select(kv4.KvPagesDescriptor(2, 9, size, 4, 3, 2)).fork(
        *dev, _dev(torch.tensor([2, 0], dtype=torch.int32)), _dev(torch.tensor([1, 2], dtype=torch.int32)), fresh)
    sync()
    assert fresh.tolist() == [2, -1]
    got = dev[0].cpu()
    rest = [p for p in range(9) if p != 2]
    _same(got[:, rest], cache[:, rest], "pages")
    assert int(dev[1].min()) >= -1 and int(dev[1].max()) < 9 and dev[1][0].tolist() == [0, 1] and int(dev[3].min()) >= 0
