"""What the plans and C entries of the 4-bit cache refuse, before any launch (no GPU)."""
import pytest
import torch

from baracuda_amd import ffi, kv4
from baracuda_amd.plans import ElementKind, InvalidProblem, Misaligned, Unsupported, WorkspaceTooSmall
from tests import kv4_plain as plain

BF = torch.bfloat16


def _raises(error, f, *args, **kw):
    with pytest.raises(error):
        f(*args, **kw)


def _qk(**kw):
    return kv4.QkNormRopeDescriptor(**{**dict(tokens=2, num_heads=4, num_kv_heads=2, head_dim=64, rope_dim=32), **kw})


@pytest.mark.parametrize("error,kw", [
    (InvalidProblem, dict(tokens=-1)), (InvalidProblem, dict(num_heads=-1)), (InvalidProblem, dict(num_kv_heads=0)),
    (InvalidProblem, dict(head_dim=0)), (InvalidProblem, dict(rope_dim=-16)), (InvalidProblem, dict(rope_dim=80)),
    (InvalidProblem, dict(axes=0)), (Unsupported, dict(head_dim=72)), (Unsupported, dict(head_dim=512)),
    (Unsupported, dict(rope_dim=24)), (Unsupported, dict(element=ElementKind.F64)), (InvalidProblem, dict(eps=-1.0)),
    (Unsupported, dict(tokens=2 ** 40))], ids=str)
def test_qk_descriptors(error, kw):
    _raises(error, kv4.QkNormRopePlan.select, _qk(**kw))


def test_qk_operands():
    plan = kv4.QkNormRopePlan.select(_qk())
    good = dict(q=torch.zeros(2, 4, 64, dtype=BF), k=torch.zeros(2, 2, 64, dtype=BF), q_out=torch.zeros(2, 4, 64, dtype=BF),
                k_out=torch.zeros(2, 2, 64, dtype=BF), q_weight=torch.ones(64, dtype=BF), k_weight=torch.ones(64, dtype=BF),
                positions=torch.zeros(1, 2, dtype=torch.int32), cos=torch.ones(5, 16), sin=torch.ones(5, 16), stream=0)
    bad = dict(q=[None, torch.zeros(2, 4, 64), torch.zeros(2, 3, 64, dtype=BF), torch.zeros(2, 4, 128, dtype=BF)[..., ::2]],
               k_out=[torch.zeros(1, 2, 64, dtype=BF).expand(2, 2, 64), torch.zeros(2, 1, 64, dtype=BF).expand(2, 2, 64)],
               q_weight=[None, torch.ones(64), torch.ones(128, dtype=BF)[::2]],
               positions=[None, torch.zeros(1, 2, dtype=torch.int64), torch.zeros(2, 2, dtype=torch.int32)],
               cos=[None, torch.ones(5, 17), torch.ones(4, 16), torch.ones(5, 32)[:, ::2], torch.ones(0, 16)],
               sin=[None, torch.ones(5, 16, dtype=torch.float64)], pair_axis=[torch.zeros(16, dtype=torch.int32)])
    for name, values in bad.items():
        for v in values:
            _raises(InvalidProblem, plan.run, **{**good, name: v})
    with pytest.raises(InvalidProblem, match="GPU"):
        plan.run(**good)
    plain_plan = kv4.QkNormRopePlan.select(_qk(norm=False, rope_dim=0))
    for name in ("q_weight", "positions", "cos"):
        none = {k: None if k in ("q_weight", "k_weight", "positions", "cos", "sin") else v for k, v in good.items()}
        _raises(InvalidProblem, plain_plan.run, **{**none, name: good[name]})
    three = kv4.QkNormRopePlan.select(_qk(axes=3))
    _raises(InvalidProblem, three.run, **{**good, "positions": torch.zeros(3, 2, dtype=torch.int32)})   # no pair_axis


def _append(**kw):
    return kv4.Kv4AppendDescriptor(**{**dict(tokens=2, num_heads=4, num_kv_heads=2, head_dim=64, page_size=16, num_pages=3),
                                      **kw})


@pytest.mark.parametrize("error,kw", [
    (Unsupported, dict(head_dim=96)), (Unsupported, dict(page_size=8)), (Unsupported, dict(page_size=48)),
    (Unsupported, dict(page_size=2048)), (InvalidProblem, dict(num_pages=0)), (Unsupported, dict(element=ElementKind.F32)),
    (InvalidProblem, dict(tokens=-1)), (InvalidProblem, dict(rope_dim=128))], ids=str)
def test_append_descriptors(error, kw):
    _raises(error, kv4.Kv4AppendPlan.select, _append(**kw))
    if "rope_dim" not in kw and kw.get("element") != ElementKind.F32:
        d = _append(**kw)
        _raises(error, kv4.Kv4ReadPlan.select, kv4.Kv4ReadDescriptor(d.tokens, d.num_kv_heads, d.head_dim, d.page_size, d.num_pages))


def test_append_and_read_operands():
    n = kv4.head_bytes(16, 64)
    assert n == 16 * 32 + 16 * 32 + 16 * 2 + 16 * 2
    good = dict(k=torch.zeros(2, 2, 64, dtype=BF), v=torch.zeros(2, 2, 64, dtype=BF),
                cache=torch.zeros(3, 2, n, dtype=torch.uint8), slots=torch.zeros(2, dtype=torch.int64),
                q=torch.zeros(2, 4, 64, dtype=BF), q_out=torch.zeros(2, 4, 64, dtype=BF), q_weight=torch.ones(64, dtype=BF),
                k_weight=torch.ones(64, dtype=BF), stream=0)
    plan = kv4.Kv4AppendPlan.select(_append())
    bad = dict(k=[None, torch.zeros(2, 4, 64, dtype=BF)], v=[torch.zeros(2, 2, 64, dtype=torch.float16)],
               cache=[None, torch.zeros(3, 2, n + 1, dtype=torch.uint8), torch.zeros(3, 2, n, dtype=torch.int8),
                      torch.zeros(3, 2, 2 * n, dtype=torch.uint8)[..., ::2]],
               slots=[None, torch.zeros(2, dtype=torch.int32), torch.zeros(3, dtype=torch.int64)], q=[None], q_out=[None])
    for name, values in bad.items():
        for v in values:
            _raises(InvalidProblem, plan.run, **{**good, name: v})
    with pytest.raises(InvalidProblem, match="GPU"):
        plan.run(**good)
    _raises(InvalidProblem, kv4.Kv4AppendPlan.select(_append(num_heads=0)).run, **good)      # a q that it does not take
    read = kv4.Kv4ReadPlan.select(kv4.Kv4ReadDescriptor(2, 2, 64, 16, 3))
    good = dict(cache=good["cache"], slots=good["slots"], k_out=good["k"], v_out=good["v"], stream=0)
    for name, v in (("k_out", None), ("v_out", torch.zeros(2, 2, 64)), ("k_out", good["v_out"][:1].expand(2, 2, 64)),
                    ("slots", torch.zeros(4, dtype=torch.int64)[::2])):
        _raises(InvalidProblem, read.run, **{**good, name: v})


def _attn(**kw):
    return kv4.Kv4AttentionDescriptor(**{**dict(num_seqs=2, total_q=3, max_q=2, max_kv=100, num_heads=4, num_kv_heads=2,
                                                head_dim=64, page_size=16, num_pages=9, max_pages=7), **kw})


@pytest.mark.parametrize("error,kw", [
    (InvalidProblem, dict(num_seqs=-1)), (InvalidProblem, dict(max_kv=-1)), (InvalidProblem, dict(num_heads=5)),
    (InvalidProblem, dict(num_kv_heads=0)), (InvalidProblem, dict(num_heads=1)), (InvalidProblem, dict(window=-1)),
    (InvalidProblem, dict(scale=0.0)), (InvalidProblem, dict(scale=float("nan"))), (InvalidProblem, dict(scale=-1.0)),
    (InvalidProblem, dict(max_pages=0)), (Unsupported, dict(head_dim=80)), (Unsupported, dict(page_size=24)),
    (Unsupported, dict(element=ElementKind.F32)), (Unsupported, dict(max_kv=2 ** 33))], ids=str)
def test_attention_descriptors(error, kw):
    _raises(error, kv4.Kv4AttentionPlan.select, _attn(**kw))


def test_attention_operands():
    n = kv4.head_bytes(16, 64)
    good = dict(q=torch.zeros(3, 4, 64, dtype=BF), cache=torch.zeros(9, 2, n, dtype=torch.uint8),
                tables=torch.zeros(2, 7, dtype=torch.int32), kv_lens=torch.zeros(2, dtype=torch.int32),
                out=torch.zeros(3, 4, 64, dtype=BF), cu_q=torch.zeros(3, dtype=torch.int32), stream=0)
    plan = kv4.Kv4AttentionPlan.select(_attn())
    bad = dict(q=[None, torch.zeros(3, 4, 64)], out=[None, torch.zeros(3, 1, 64, dtype=BF).expand(3, 4, 64)],
               tables=[None, torch.zeros(2, 7, dtype=torch.int64), torch.zeros(7, 2, dtype=torch.int32).t(),
                       torch.zeros(2, 6, dtype=torch.int32)],
               kv_lens=[None, torch.zeros(3, dtype=torch.int32), torch.zeros(2, dtype=torch.int64)],
               cu_q=[None, torch.zeros(2, dtype=torch.int32)], cache=[torch.zeros(9, 2, n, dtype=torch.int8)])
    for name, values in bad.items():
        for v in values:
            _raises(InvalidProblem, plan.run, **{**good, name: v})
    with pytest.raises(InvalidProblem, match="GPU"):
        plan.run(**good)


def test_attention_workspace():
    L, x = ffi.lib(), 4096                 # a pointer that is never followed
    assert kv4.Kv4AttentionPlan.select(_attn()).workspace_size() == 0
    big = _attn(num_seqs=1, total_q=1, max_q=1, max_kv=100000, max_pages=7000)
    need = kv4.Kv4AttentionPlan.select(big).workspace_size()
    assert need > 0
    sizes = kv4.Kv4AttentionPlan._sizes(big)

    def run(ws, n, q=x, cache=x, cu=None):
        return L.kv4_attention_gfx950_run(*sizes, q, 256, 64, cache, x, 7000, x, cu, x, 256, 64, ws, n, None)

    assert run(None, 0) == run(x, need - 1) == WorkspaceTooSmall.status
    assert run(x + 8, need) == run(x, need, q=x + 1) == run(x, need, cache=x + 8) == Misaligned.status
    assert run(x, need, q=None) == InvalidProblem.status
    few = list(sizes)
    few[1] = 2                             # two rows of one sequence without cu_q
    assert L.kv4_attention_gfx950_run(*few, x, 256, 64, x, x, 7000, x, None, x, 256, 64, x, need, None) == 2
    none = list(sizes)
    none[0] = 0                            # nothing to do, nothing read
    assert L.kv4_attention_gfx950_run(*none, None, 0, 0, None, None, 0, None, None, None, 0, 0, None, 0, None) == 0


def test_entries_without_tokens_or_pointers():
    L, x = ffi.lib(), 4096
    zero = (None, 0, 0)
    rot = (None, None, None, None, None, 0, None)
    assert L.qk_norm_rope_gfx950_run(0, 4, 2, 64, 0, 1, 0, 2, 1e-6, *zero * 4, *rot, None) == 0
    assert L.qk_norm_rope_gfx950_run(1, 4, 2, 64, 0, 1, 0, 2, 1e-6, *zero * 4, *rot, None) == 2
    some = (x, 256, 64)
    assert L.qk_norm_rope_gfx950_run(1, 4, 2, 64, 0, 1, 0, 2, 1e-6, (x + 1), 256, 64, *some * 3, *rot, None) == 1
    assert L.qk_norm_rope_gfx950_run(1, 4, 2, 64, 0, 1, 0, 0, 1e-6, (x + 2), 256, 64, *some * 3, *rot, None) == 1
    assert L.qk_norm_rope_gfx950_run(1, 4, 2, 64, 0, 1, 0, 2, 1e-6, *some * 4, x, *rot[1:], None) == 2     # one weight
    assert L.qk_norm_rope_gfx950_run(1, 4, 2, 64, 16, 1, 0, 2, 1e-6, *some * 4, *rot, None) == 2           # no table
    assert L.qk_norm_rope_gfx950_run(1, 4, 2, 64, 16, 2, 0, 2, 1e-6, *some * 4, x, x, x, x, x, 9, None, None) == 2
    assert L.qk_norm_rope_gfx950_run(1, 4, 2, 64, 0, 1, 0, 3, 1e-6, *some * 4, *rot, None) == 2
    assert L.kv4_append_gfx950_run(0, 4, 2, 64, 0, 1, 0, 2, 1e-6, 16, 3, *zero * 4, None, None, *rot, None) == 0
    assert L.kv4_append_gfx950_run(1, 4, 2, 64, 0, 1, 0, 2, 1e-6, 16, 3, *some * 4, None, x, *rot, None) == 2
    assert L.kv4_append_gfx950_run(1, 4, 2, 64, 0, 1, 0, 2, 1e-6, 16, 3, *some * 4, x + 4, x, *rot, None) == 1
    assert L.kv4_append_gfx950_run(1, 4, 2, 64, 0, 1, 0, 2, float("nan"), 16, 3, *some * 4, x, x, *rot, None) == 2
    assert L.kv4_read_gfx950_run(0, 2, 64, 2, 16, 3, None, None, *zero * 2, None) == 0
    assert L.kv4_read_gfx950_run(1, 2, 64, 2, 16, 3, x, None, *some * 2, None) == 2
    assert L.kv4_read_gfx950_run(1, 2, 64, 2, 16, 3, x, x, x + 1, 1, 1, *some, None) == 1


@pytest.mark.parametrize("kw", [dict(layers=0), dict(num_pages=0), dict(page_bytes=0), dict(page_size=0), dict(rows=0),
                                dict(max_pages=0)], ids=str)
def test_pages_descriptors(kw):
    _raises(InvalidProblem, kv4.KvPagesPlan.select, kv4.KvPagesDescriptor(**{**dict(
        layers=2, num_pages=5, page_bytes=32, page_size=4, rows=3, max_pages=6), **kw}))


def test_pages_operands():
    plan = kv4.KvPagesPlan.select(kv4.KvPagesDescriptor(2, 5, 32, 4, 3, 6))
    assert plan.workspace_size() == 16 + 8 * 5
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)
    cache = torch.zeros(2, 5, 32, dtype=torch.uint8)
    with pytest.raises(InvalidProblem, match="GPU"):
        plan.copy(cache, i(2), i(2), stream=0)
    for c, s, d in ((None, i(2), i(2)), (cache[:1], i(2), i(2)), (cache, i(2), i(3)), (cache, i(2).long(), i(2)),
                    (cache, None, i(2)), (cache, i(4)[::2], i(2))):
        _raises(InvalidProblem, plan.copy, c, s, d, stream=0)
    good = dict(cache=cache, tables=i(3, 6), lens=i(3), refs=i(5), parents=i(2), children=i(2), fresh=i(2), stream=0)
    for name, v in (("cache", None), ("tables", i(3, 5)), ("tables", i(6, 3).t()), ("lens", None), ("refs", i(6)),
                    ("children", i(3)), ("fresh", None), ("parents", i(2, 1))):
        _raises(InvalidProblem, plan.fork, **{**good, name: v})
    for name, v in (("tables", None), ("lens", None), ("refs", i(5).long()), ("rows", None), ("rows", i(1, 1))):
        _raises(InvalidProblem, plan.release, **{**dict(tables=i(3, 6), lens=i(3), refs=i(5), rows=i(1), stream=0), name: v})
    good = dict(cache=cache, tables=i(3, 6), refs=i(5), tables_out=i(3, 6), refs_out=i(5), remap=i(5), live=i(1), stream=0)
    for name, v in (("refs_out", good["refs"]), ("remap", i(4)), ("live", i(2)), ("tables_out", None), ("cache", cache.float())):
        _raises(InvalidProblem, plan.compact, **{**good, name: v})
    L, x = ffi.lib(), 4096
    sizes = (2, 5, 32, 4, 3, 6)
    assert L.kv_pages_compact_gfx950_run(*sizes, x, x, x, x, x + 64, x, x, None, 0, None) == 4
    assert L.kv_pages_compact_gfx950_run(*sizes, x, x, x, x, x + 64, x, x, x, 55, None) == 4
    assert L.kv_pages_compact_gfx950_run(*sizes, x, x, x, x, x, x, x, x, 56, None) == 2
    assert L.kv_pages_copy_gfx950_run(2, 5, 32, 0, None, None, None, None) == 0
    assert L.kv_pages_copy_gfx950_run(2, 5, 32, -1, x, x, x, None) == 2
    assert L.kv_pages_copy_gfx950_run(2, 5, 32, 1, x, None, x, None) == 2
    assert L.kv_pages_fork_gfx950_run(*sizes, 0, None, None, None, None, None, None, None, None) == 0
    assert L.kv_pages_fork_gfx950_run(*sizes, 1, x, x, x, x, x, x, None, None) == 2
    assert L.kv_pages_release_gfx950_run(5, 3, 6, 0, None, None, None, None, None) == 0
    assert L.kv_pages_release_gfx950_run(5, 3, 6, 1, x, x, None, x, None) == 2


def test_sizes_past_a_launch():
    L, x = ffi.lib(), 4096
    for tokens in (2 ** 23, 2 ** 31, 2 ** 60):
        _raises(Unsupported, kv4.QkNormRopePlan.select, _qk(tokens=tokens))
        _raises(Unsupported, kv4.Kv4AppendPlan.select, _append(tokens=tokens))
        _raises(Unsupported, kv4.Kv4ReadPlan.select, kv4.Kv4ReadDescriptor(tokens, 2, 64, 16, 3))
    _raises(Unsupported, kv4.Kv4AttentionPlan.select, _attn(num_seqs=2 ** 22, total_q=2 ** 22))
    for name in ("num_heads", "head_dim", "page_size", "max_q", "max_pages"):       # past 32 bits, not cut off to them
        _raises(Unsupported, kv4.Kv4AttentionPlan.select, _attn(**{name: 2 ** 32 + getattr(_attn(), name)}))
    _raises(Unsupported, kv4.KvPagesPlan.select, kv4.KvPagesDescriptor(2, 5, 32, 4, 2 ** 32 + 3, 6))
    assert L.kv_pages_release_gfx950_run(5, 3, 6, 2 ** 24, x, x, x, x, None) == 3
    assert L.kv_pages_fork_gfx950_run(2, 5, 32, 4, 3, 6, 70000, x, x, x, x, x, x, x, None) == 3


def test_plain_codec():
    """The oracle itself: borders, ties, the largest value of a scale, zeros, infinities."""
    x = torch.zeros(32, dtype=torch.float64)
    x[:8] = torch.tensor([6.9, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
    code, byte = plain.encode(x, 125)
    assert code[:8].tolist() == [7, 0, 2, 2, 4, 4, 6, 6] and byte.tolist() == [127]
    x[0] = -7.0
    code, byte = plain.encode(x, 125)
    assert code[:4].tolist() == [14, 0, 1, 1] and byte.tolist() == [128]
    assert plain.encode(torch.zeros(32), 125)[1].tolist() == [2]
    x[3] = float("inf")
    code, byte = plain.encode(x, 125)
    assert not code.any() and byte.tolist() == [255]
    assert torch.isnan(plain.decode(code, byte)).all()
    ps, d = 32, 128
    where = torch.cat([p.flatten() for p in plain.places(ps, d)])
    assert where.sort()[0].tolist() == list(range(kv4.head_bytes(ps, d)))     # every byte once
