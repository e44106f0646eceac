"""The plain form that the GPU tests compare llmk_pages_* with, against what the
documentation promises, on the CPU."""
import numpy as np

from pages_util import Plain


def test_rows_grow_share_and_end():
    c = Plain(4, 8, 4, 12)
    g, bad, full = c.update([5, -1, -1, -1])
    assert list(c.held(0)) == [0, 1] and g.all() and not bad and not full
    # two children of row 0; all three then write into its half-filled page 1
    g, bad, full = c.update([6, 6, 7, -1], [-1, 0, 0, -1])
    assert g.all() and not bad and not full
    # rows 0 and 1 leave it, the last of its holders keeps it
    assert [list(c.held(r)) for r in range(3)] == [[0, 2], [0, 3], [0, 1]]
    assert list(c.refs[:4]) == [3, 1, 1, 1]
    assert c.contents[2] == 1 and c.contents[3] == 1
    c.check()
    # row 0 ends, page 2 is the lowest free one again
    c.update([0, 8, 9, -1])
    assert list(c.held(2)) == [0, 1, 2]
    c.check()


def test_a_prefix_is_forked_and_a_row_renamed():
    c = Plain(3, 8, 4, 8)
    c.update([13, -1, -1])
    g, bad, _ = c.update([0, 13, 6], [-1, 0, 0])  # row 0's pages pass to row 1, a prefix to row 2
    assert g.all() and not bad
    assert list(c.held(1)) == [0, 1, 2, 3] and list(c.held(2)) == [0, 1] and c.lengths[0] == 0
    c.check()


def test_too_few_pages_and_bad_requests():
    c = Plain(5, 4, 4, 5)
    g, bad, full = c.update([8, 12, 4, -1, 3])  # 2 + 3 fit, the rest do not
    assert list(g) == [1, 1, 0, 1, 0] and full and not bad
    g, bad, full = c.update([-1, -1, 17, -1, -1])  # above max_pages * page_tokens
    assert list(g) == [1, 1, 0, 1, 1] and bad and not full
    g, bad, full = c.update(None, [-1, 0, 9, 3, 2])  # not empty; no such row; itself; a child
    assert list(g) == [1, 0, 0, 0, 0] and bad
    c.check()


def test_a_row_that_waits_keeps_its_shared_page_from_being_written():
    c = Plain(3, 4, 4, 1)
    c.update([2, -1, -1])
    c.update(None, [-1, 0, 0])
    g, _, full = c.update([3, 3, 3])  # no page for a copy
    assert list(g) == [0, 0, 0] and full and list(c.lengths) == [2, 2, 2]
    c.update([0, 0, -1])
    g, _, full = c.update([-1, -1, 3])  # alone with it now
    assert g.all() and not full and list(c.held(2)) == [0]


def test_compaction():
    rng = np.random.default_rng(0)
    for _ in range(50):
        c = Plain(6, 10, 3, 40)
        for _ in range(6):
            par = np.where(c.lengths == 0, rng.integers(-1, 6, 6), -1)
            c.update(rng.integers(-1, 31, 6), par)
            c.check()
        what = [[int(c.contents[p]) for p in c.held(r)] for r in range(6)]
        c.compact()
        c.check()
        M = int((c.refs > 0).sum())
        assert (c.refs[:M] > 0).all() and (c.refs[M:] == 0).all()
        assert what == [[int(c.contents[p]) for p in c.held(r)] for r in range(6)]
