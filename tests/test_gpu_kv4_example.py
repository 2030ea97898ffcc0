"""The serving example: rows that share pages, and pages that moved, give what
they would have given."""
import pytest
import torch

from examples import kv4_serving

pytestmark = pytest.mark.gpu


def test_serving_example(gpu):
    out = kv4_serving.main()
    for step in out["samples"]:
        assert torch.equal(step[0], step[2])            # a fork given the same tokens
        assert not torch.equal(step[2], step[3])        # and one given others
        assert all(torch.isfinite(t).all() for t in step)
    assert torch.equal(out["last"][0], out["last"][1])  # the same after the pages have moved
    s = out["server"]
    used = int((s.refs > 0).sum())
    assert used == int((s.refs[:used] > 0).sum()) and int(s.lens[1]) == 0
    # the last step on pages that were never forked or moved
    fresh = kv4_serving.Server()
    g = torch.Generator().manual_seed(1)
    make = lambda n: torch.randn(n, s.hidden, generator=g).to(torch.bfloat16).to(s.dev)
    prompts = [make(45), make(20)]
    assert torch.equal(fresh.step([4], prompts[:1])[0], out["first"][0])
    for step in out["samples"]:
        token, _ = make(1), make(1)
        assert torch.equal(fresh.step([4], [token])[0], step[0])
    assert torch.equal(fresh.step([4], [make(1)])[0], out["last"][0])
