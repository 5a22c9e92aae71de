"""Pins the draft-tree oracle (oracle/drafts.py) with closed forms and
invariants; each test names the mistake it would catch.  No GPU."""

import numpy as np

from oracle import attention as A
from oracle import drafts as T


def test_visibility_of_a_small_tree_and_bad_parents():
    #      0          roots: 0 and 4 (its parent 7 is no earlier draft)
    #    1   2        an off-by-one would let 3 see 2, or 1 see itself only
    #    3
    sees, depths = T.tree_visibility([-1, 0, 0, 1, 7])
    want = np.array([[1, 0, 0, 0, 0], [1, 1, 0, 0, 0], [1, 0, 1, 0, 0], [1, 1, 0, 1, 0],
                     [0, 0, 0, 0, 1]], dtype=bool)
    assert np.array_equal(sees, want) and depths.tolist() == [0, 1, 1, 2, 0]
    sees, depths = T.tree_visibility([-1, 0, 1], count=2)
    assert not sees[2].any() and depths.tolist() == [0, 1, -1]


def test_mask_words_put_draft_64_into_the_second_word():
    sees = np.zeros((1, 70), dtype=bool)
    sees[0, [0, 63, 64, 69]] = True
    words = T.mask_words(sees).view(np.uint64)
    assert words.tolist() == [[1 | 1 << 63, 1 | 1 << 5]]


def test_tree_attention_is_decode_along_each_path():
    # a draft's result is the plain decode over its prefix and path: catches
    # a mask applied to the wrong rows, and a wrong head map
    rng = np.random.default_rng(0)
    prefix, parents = 5, [-1, 0, 0, 2]
    q = rng.standard_normal((4, 6, 8))
    k, v = rng.standard_normal((9, 2, 8)), rng.standard_normal((9, 2, 8))
    sees, _ = T.tree_visibility(parents)
    out, weight = T.tree_attention(q, k, v, sees, prefix, 8 ** -0.5)
    for i, path in enumerate(([0], [0, 1], [0, 2], [0, 2, 3])):
        rows = list(range(prefix)) + [prefix + j for j in path]
        want = A.attention_decode_twopass(q[i], k[rows], v[rows], 3, 8 ** -0.5)
        np.testing.assert_allclose(out[i], want, atol=1e-12)
    assert (weight >= np.abs(out) - 1e-12).all()


def test_tree_attention_keeps_unseen_rows_out_and_empty_rows_zero():
    # 0 times an infinity is a NaN: a product over all rows would spread it
    rng = np.random.default_rng(1)
    q, k, v = (rng.standard_normal(s) for s in ((2, 1, 4), (2, 1, 4), (2, 1, 4)))
    v[1], k[1] = np.inf, np.nan
    sees = np.array([[True, False], [False, False]])
    out, _ = T.tree_attention(q, k, v, sees, 0, 0.5)
    np.testing.assert_allclose(out[0, 0], v[0, 0], atol=1e-15)
    assert not out[1].any()


def test_resize_grows_shrinks_and_restores_the_stack():
    table = [[3, -1, -1], [5, 6, -1]]
    lengths, free, count = [2, 8], [9, 8, 7, -1, -1], 3
    count, rows, granted = T.resize(table, lengths, free, count, [5, 3], 4, 10)
    # sequence 1 gives page 6 back, sequence 0 takes it (the top of the stack)
    assert granted == [1, 1] and table == [[3, 6, -1], [5, -1, -1]] and count == 3
    assert rows == [(14, 2, 0), (15, 3, 0), (24, 4, 0)] and lengths == [5, 3]
    # cutting back what a call grew leaves the stack as it was
    before = list(free[:count])
    count, _, _ = T.resize(table, lengths, free, count, [12, 8], 4, 20)
    assert count == 1
    count, _, _ = T.resize(table, lengths, free, count, [5, 3], 4, 0)
    assert free[:count] == before and table == [[3, 6, -1], [5, -1, -1]]


def test_resize_refuses_in_order():
    # sequence 1 asks for more pages than are left and makes 2 wait; 3 needs
    # no page; 4 asks for more rows than a sequence can hold
    table = [[0, -1, -1], [1, -1, -1], [2, -1, -1], [3, -1, -1], [4, -1, -1]]
    lengths = [1, 4, 4, 1, 4]
    count, rows, granted = T.resize(table, lengths, [7, 6], 2, [5, 12, 5, 4, 13], 4, 100)
    assert granted == [1, 0, 0, 1, 0] and lengths == [5, 4, 4, 4, 4] and count == 1
    assert [r[2] for r in rows] == [0, 0, 0, 0, 3, 3, 3]
    # rows past `tokens` are refused, the ones before them stand
    lengths = [1, 1]
    _, rows, granted = T.resize([[0, -1], [1, -1]], lengths, [], 0, [3, 4], 4, 4)
    assert granted == [1, 0] and len(rows) == 2


def test_commit_moves_the_path_and_nothing_else():
    rows = np.arange(10)
    assert T.commit(rows, 3, [1, 2, 5], 3).tolist() == [0, 1, 2, 4, 5, 8, 6, 7, 8, 9]
    assert T.commit(rows, 3, [1, 2, 5], 1).tolist() == [0, 1, 2, 4, 4, 5, 6, 7, 8, 9]
    # a path ends where it stops rising
    assert T.commit(rows, 3, [2, 2, 5], 3).tolist() == [0, 1, 2, 5, 4, 5, 6, 7, 8, 9]
