"""Sizes of the 4-bit cache's operators at the ends of what a launch holds (no GPU)."""
import pytest

from baracuda_amd import ffi, kv4
from baracuda_amd.plans import Unsupported

TOP = 2 ** 31 - 1


def _attn(**kw):
    return kv4.Kv4AttentionDescriptor(**{**dict(num_seqs=2, total_q=3, max_q=2, max_kv=100, num_heads=4, num_kv_heads=2,
                                                head_dim=64, page_size=16, num_pages=9, max_pages=7), **kw})


@pytest.mark.parametrize("kw", [
    dict(max_q=TOP, num_heads=32768, num_kv_heads=1), dict(max_q=TOP, num_heads=512, num_kv_heads=1),
    dict(max_q=TOP, num_heads=32768, num_kv_heads=1, head_dim=256), dict(max_q=TOP, num_heads=32768, num_kv_heads=1, max_kv=0),
    dict(num_seqs=TOP, max_q=TOP, num_heads=32768, num_kv_heads=1), dict(num_seqs=TOP, max_q=TOP),
    dict(num_seqs=TOP, num_heads=32768, num_kv_heads=32768), dict(num_seqs=2 ** 16, max_q=2 ** 16),
    dict(total_q=TOP, num_heads=32768, num_kv_heads=1), dict(total_q=2 ** 28, num_heads=16)], ids=str)
def test_attention_sizes_past_a_launch(kw):
    d = _attn(**kw)
    with pytest.raises(Unsupported):
        kv4.Kv4AttentionPlan.select(d)
    if "total_q" not in kw:
        assert ffi.lib().kv4_attention_gfx950_workspace_size(d.num_seqs, d.max_q, d.max_kv, d.num_heads, d.num_kv_heads,
                                                             d.head_dim, d.window) == 0


def test_attention_sizes_within_a_launch():
    """The bounds may be larger than what a call has: max_q past total_q, max_kv past the tables."""
    for kw in (dict(max_q=2 ** 20), dict(max_q=2 ** 20, num_heads=64), dict(num_seqs=2 ** 20, total_q=2 ** 20, max_q=1),
               dict(total_q=2 ** 28), dict(max_kv=2 ** 30)):
        plan = kv4.Kv4AttentionPlan.select(_attn(**kw))
        assert 0 <= plan.workspace_size() < 2 ** 40
