"""The plain form of the page updates in perf/operators.py against the rows taken
one after another (pages_util.py), on the CPU: grants, lengths, counts, tables
and the contents of every page, with page 0 free as well as held."""
import os
import sys

import numpy as np
import pytest
import torch
from torch.overrides import TorchFunctionMode

from pages_util import Plain

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from perf import operators as ops  # noqa: E402


class OnTheCpu(TorchFunctionMode):
    """Tensors that are asked for on the GPU, on the CPU."""

    def __torch_function__(self, func, types, args=(), kwargs=None):
        kwargs = dict(kwargs or {})
        if kwargs.get("device") == "cuda":
            kwargs["device"] = "cpu"
        return func(*args, **kwargs)


@pytest.fixture
def on_the_cpu(monkeypatch):
    monkeypatch.setattr(ops, "own", False)
    monkeypatch.setattr(ops, "_gen", lambda seed: torch.Generator().manual_seed(int(seed)))
    with OnTheCpu():
        yield


@pytest.mark.parametrize("forks,tight", [(0, False), (1, False), (3, False), (4, True), (0, True)])
def test_update(on_the_cpu, forks, tight):
    c = dict(name="x", kind="update", rows=23, page=8, low=3, high=120, forks=forks, bytes=5,
             pools=2, tight=tight)
    copies_to_page_0 = 0
    for seed in range(40):
        s = ops.prepare(c, seed)
        N, (R, P) = s["refs"].numel(), s["table"].shape
        plain = Plain(R, P, c["page"], N)
        plain.table[:] = s["table"].numpy()
        plain.lengths[:], plain.refs[:] = s["lengths"].numpy(), s["refs"].numpy()
        plain.check()
        pools = [p.clone() for p in s["pools"]]
        granted, invalid, _ = plain.update(s["grown"].numpy(), s["parents"].numpy())
        assert not invalid
        copies_to_page_0 += plain.contents[0] != 0
        for _ in range(2):  # the second call begins from the same cache
            got = ops.run(s)
            assert np.array_equal(got["granted"].numpy(), granted)
            assert np.array_equal(got["lengths"].numpy(), plain.lengths)
            assert np.array_equal(got["refs"].numpy(), plain.refs)
            for r in range(R):
                k = plain.pages(plain.lengths[r])
                assert np.array_equal(got["table"][r, :k].numpy(), plain.table[r, :k])
            for before, now in zip(pools, got["pools"]):
                assert torch.equal(now, before[torch.as_tensor(plain.contents)])
    # a copy into page 0 is among the updates with forks
    assert (copies_to_page_0 > 0) == (forks > 0)
