"""Attention over 4-bit pages: every kernel, way to cut the work, size of heads, type and
mask, in sequences long enough that a wave looks up further pages on its way.

The tokens that a wrong page or a lost part would change carry the weights: around
every such place, and here and there, K points along the queries' signs, so that a
row's result is about the mean of those tokens' V.  tests/test_kv4_rules.py holds the
cases to the forms that they name."""
import pytest
import torch

from baracuda_amd import kv4
from tests import kv4_plain as plain
from tests.gpu_util import sync
from tests.kv4_forms import CASES, HK, case_id
from tests.test_gpu_kv4 import KIND, _check_attention, _dev, _scene

pytestmark = pytest.mark.gpu

PS = 16


def _spread(form):
    """The sequences of the longest list that have tokens, and all sequences' lengths and new tokens."""
    lens, new = [0] * form.seqs, [0] * form.seqs
    at = [i * (form.seqs - 1) // max(1, len(form.lens) - 1) for i in range(len(form.lens))]
    for i, n, q in zip(at, form.lens, form.new):
        lens[i], new[i] = n, q
    return at, lens, new


def _boundaries(form, d, windowed):
    """Tokens of the longest sequence at which a wave of its first block looks up pages."""
    if not form.refill:
        return []
    first = max(0, form.lens[0] - form.new[0] - form.window() + 1) // 16 * 16 if windowed else 0
    return list(range(first + form.refill[d], form.lens[0], form.refill[d]))


@pytest.mark.parametrize("case", CASES, ids=case_id)
def test_attention_form(gpu, case):
    form, d, (_, causal, windowed), dt = case
    print(case_id(case), flush=True)
    g = torch.Generator().manual_seed(d + form.max_kv)
    window = form.window() if windowed else 0
    at, lens, new = _spread(form)
    hq = HK * form.ratio
    cache, tables, lens_t, cu, q = _scene(g, lens, new, hq, HK, d, PS, dt)
    sign = torch.randint(0, 2, (HK, d), generator=g)
    q = (q.abs().float() * (1 - 2 * sign.repeat_interleave(form.ratio, 0))).to(dt)
    where = plain.places(PS, d)
    along = sign * 8 + 5                                   # 3 with the queries' signs
    along = (along[:, 0::2] | along[:, 1::2] << 4).to(torch.uint8)

    def point(b, token):
        if 0 <= token < lens[b]:
            page = int(tables[b, token // PS])
            cache[page][:, where[0][token % PS]] = along
            cache[page][:, where[2][token % PS]] = 127

    for b in at:
        for token in torch.randint(0, lens[b], (min(24, lens[b]),), generator=g).tolist():
            point(b, token)
    edges = _boundaries(form, d, windowed)
    for e in edges:
        for page in range(e // PS - 2, e // PS + 3):
            point(at[0], page * PS)
            point(at[0], page * PS + PS - 1)
    plan = kv4.Kv4AttentionPlan.select(kv4.Kv4AttentionDescriptor(
        form.seqs, q.shape[0], form.max_q, form.max_kv, hq, HK, d, PS, cache.shape[0], tables.shape[1], KIND[dt], causal, window))
    assert (plan.workspace_size() > 0) == form.cut
    ws = torch.full((plan.workspace_size(),), 0x7f, dtype=torch.uint8, device=gpu)
    held = [_dev(x) for x in (q, cache, lens_t, cu)]

    def run(tables):
        out = torch.full(q.shape, 3.0, dtype=dt, device=gpu)
        plan.run(held[0], held[1], _dev(tables), held[2], out, cu_q=held[3], workspace=ws)
        sync()
        return out

    _check_attention(run(tables), q, cache, tables, lens_t, cu, causal, window, d ** -0.5)
    if edges or form.cut:         # and with pages missing right after those places
        missing = tables.clone()
        for e in edges or [form.lens[0] // 2]:
            missing[at[0], e // PS] = -1
        _check_attention(run(missing), q, cache, missing, lens_t, cu, causal, window, d ** -0.5)


@pytest.mark.parametrize("case", [c for c in CASES if c[0].new[0] > 4 and c[2][1]], ids=case_id)
def test_nan_reaches_the_rows_that_see_it(gpu, case):
    """A NaN in V of the third last token: the rows before it keep their values, the
    others have it in its group of values alone."""
    form, d, (_, causal, windowed), dt = case
    print(case_id(case), flush=True)
    window = form.window() if windowed else 0
    at, lens, new = _spread(form)
    hq = HK * form.ratio
    cache, tables, lens_t, cu, q = _scene(torch.Generator().manual_seed(d), lens, new, hq, HK, d, PS, dt)
    plan = kv4.Kv4AttentionPlan.select(kv4.Kv4AttentionDescriptor(
        form.seqs, q.shape[0], form.max_q, form.max_kv, hq, HK, d, PS, cache.shape[0], tables.shape[1], KIND[dt], causal, window))
    ws = torch.full((plan.workspace_size(),), 0x7f, dtype=torch.uint8, device=gpu)
    held = [_dev(x) for x in (tables, lens_t)]

    def run():
        out = torch.full(q.shape, 3.0, dtype=dt, device=gpu)
        plan.run(_dev(q), _dev(cache), *held, out, cu_q=_dev(cu), workspace=ws)
        sync()
        return out.cpu()

    clean = run()
    assert not torch.isnan(clean).any()
    token = form.lens[0] - 3
    cache[int(tables[at[0], token // PS]), :, plain.places(PS, d)[3][token % PS, 1]] = 255
    got = run()
    first = new[at[0]] - 3        # the first row that sees it
    assert torch.isnan(got[first:first + 3, :, 32:64]).all()
    got[first:first + 3, :, 32:64] = clean[first:first + 3, :, 32:64]
    assert torch.equal(got, clean)
