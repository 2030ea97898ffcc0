"""The operators around a 4-bit key-value cache at the ends of what they take."""
import pytest
import torch

from baracuda_amd import kv4
from tests import kv4_plain as plain
from tests.gpu_util import sync
from tests.test_gpu_kv4 import BF, KIND, _check_attention, _dev, _scene

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
