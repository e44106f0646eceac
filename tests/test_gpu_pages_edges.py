"""llmk_pages_* on the GPU at the ends of their documented ranges."""
import numpy as np
import pytest
import torch

import llmk
from llmk import _lib

pytestmark = pytest.mark.gpu


def used_pages(cache):
    words = cache.used.cpu().numpy().view(np.uint32)
    return np.unpackbits(words.view(np.uint8), bitorder="little")[:cache.num_pages].astype(bool)


def test_as_many_rows_and_pages_as_a_cache_holds():
    """2^20 rows and 2^25 pages: rows begin, grow, end and move; too many ask."""
    s = llmk.HipSampler(max_batch=1, max_vocab=1024)
    R, N = 2**20, 2**25
    c = llmk.PageCache(s, R, 40, 1, N)
    row = np.arange(R)
    n = (row % 3 + 1).astype(np.int32)
    assert bool((c.update(torch.as_tensor(n).cuda()) == 1).all())
    first = np.cumsum(n) - n
    table = c.table.cpu().numpy()
    for j in range(3):
        at = n > j
        assert np.array_equal(table[at, j], first[at] + j)
    assert used_pages(c).sum() == n.sum() and used_pages(c)[:n.sum()].all()
    # every second row ends, the pages move down
    end = np.where(row % 2 == 0, 0, -1).astype(np.int32)
    assert bool((c.update(torch.as_tensor(end).cuda()) == 1).all())
    kept = np.where(row % 2 == 0, 0, n)
    assert used_pages(c).sum() == kept.sum()
    to = c.compact().cpu().numpy()
    M = int(kept.sum())
    assert used_pages(c)[:M].all() and not used_pages(c)[M:].any()
    moved = c.table.cpu().numpy()
    for j in range(3):
        at = kept > j
        assert np.array_equal(moved[at, j], to[first[at] + j])
    assert np.array_equal(c.refs.cpu().numpy(), (np.arange(N) < M).astype(np.int32))
    # all ask for 40 pages: the first rows get them, in order
    g = c.update(torch.full((R,), 40, dtype=torch.int32, device="cuda:0")).cpu().numpy()
    need = np.cumsum(40 - kept)
    fits = need <= N - M
    assert np.array_equal(g, fits.astype(np.int32))
    assert s.status() == _lib.LLMK_STATUS_PAGES_FULL
    assert np.array_equal(c.lengths.cpu().numpy(), np.where(fits, 40, kept))
    assert used_pages(c).sum() == M + need[fits][-1]
    # and all end
    assert bool((c.update(torch.zeros(R, dtype=torch.int32, device="cuda:0")) == 1).all())
    assert not used_pages(c).any() and not bool(c.refs.any())
    assert s.status() == 0
    del c
    s.close()
    torch.cuda.empty_cache()
