"""Pins the oracle of the 4-bit pool, the rotated rows and the verified
drafts (oracle/q4.py) with closed forms and hand-written cases; each test
names the mistake it would catch.  No GPU."""

import numpy as np
import pytest

from oracle import attention as A
from oracle import q4 as Q
from oracle import rope as R


def test_codes_of_a_group_by_hand():
    # least 1, step 1: codes are the numbers less one; ties go to even (a
    # rounding up of halves would give 3 for 2.5 steps)
    x = np.ones((1, 1, 32))
    x[0, 0, :5] = [16.0, 3.5, 4.5, 2.0, 1.25]
    codes, step, least = Q.encode(x)
    assert step.tolist() == [[[1.0]]] and least.tolist() == [[[1.0]]]
    assert codes[0, 0, :6].tolist() == [15, 2, 4, 1, 0, 0]
    assert Q.decode(codes, step, least)[0, 0, :3].tolist() == [16.0, 3.0, 5.0]


def test_codes_stay_within_half_a_step():
    # a step or least value of the wrong group, or rounded the wrong way
    rng = np.random.default_rng(0)
    x = rng.standard_normal((7, 3, 96)) * np.exp(rng.normal(size=(7, 3, 96)))
    codes, step, least = Q.encode(x)
    off = np.abs(Q.decode(codes, step, least) - x).reshape(7, 3, 3, 32)
    # half a step, and what the float16 step and least value are off:
    # 15 codes by half an ulp of the step, half an ulp of the least value
    most = step * (0.5 + 15 * 2.0 ** -11) + np.abs(least) * 2.0 ** -11 + 2.0 ** -24
    assert (off <= most.astype(np.float64)[..., None] + 1e-6).all()


def test_groups_that_are_constant_or_not_finite():
    x = np.full((1, 1, 64), 0.125)
    x[0, 0, 40] = np.nan
    codes, step, least = Q.encode(x)
    assert not codes.any() and step[0, 0].tolist() == [0.0, 0.0]
    got = Q.decode(codes, step, least)[0, 0]
    assert (got[:32] == 0.125).all() and np.isnan(got[32:]).all()
    x[0, 0, 40], x[0, 0, 3] = -np.inf, 1e9
    codes, step, least = Q.encode(x)
    assert np.isnan(least[0, 0, 1]) and np.isfinite(step).all() and codes[0, 0, 3] == 15


def test_pool_puts_even_channels_low_and_steps_along_rows():
    pool = Q.empty_pool(3, 2, 32, 64)
    x = np.zeros((2, 2, 64))
    x[0, 1, 32:36] = [15.0, 1.0, 2.0, 3.0]
    x[1] = np.nan
    Q.put(pool, [32 + 5, 96], x)  # the second lies outside
    data, scales = pool
    assert data[1, 1, 5, 16:18].tolist() == [15 | 1 << 4, 2 | 3 << 4]
    assert scales[1, 1, 0, 1, 5] == 1.0 and np.count_nonzero(scales) == 1
    assert np.array_equal(Q.get(pool, [37, -1])[0], x[0]) and not Q.get(pool, [96]).any()


def test_gross_of_a_row_by_hand():
    # a sign of the least value that is kept would make them cancel
    pool = Q.empty_pool(1, 1, 32, 64)
    x = np.full((1, 1, 64), -3.0)
    x[0, 0, 0] = 12.0  # least -3, step 1: 3 + 15, the others 3
    Q.put(pool, [4], x)
    assert Q.gross(pool, [4])[0, 0, :2].tolist() == [18.0, 3.0]


@pytest.mark.parametrize("rotary", [8, 6])
def test_rotation_matches_the_llama_tables(rotary):
    # wrong pairs, sign or frequencies
    rng = np.random.default_rng(1)
    x, at = rng.standard_normal((4, 3, 8)), np.array([0, 1, 7, 90])
    cos, sin = R.rope_tables(128, rotary, 500.0)
    want = R.rope_norm_batch(x, at, cos, sin, rotary)
    assert np.abs(Q.rotate(x, at, rotary, "norm", 500.0) - want).max() < 2e-5
    # neox: the same with its halves side by side
    order = np.concatenate([np.arange(rotary).reshape(2, -1).T.reshape(-1), np.arange(rotary, 8)])
    neox = Q.rotate(x, at, rotary, "neox", 500.0)[..., order]
    assert np.allclose(neox, Q.rotate(x[..., order], at, rotary, "norm", 500.0))


def test_attention_of_the_last_token_is_decode():
    rng = np.random.default_rng(2)
    q, k, v = (rng.standard_normal(s) for s in ((2, 4, 8), (6, 2, 8), (6, 2, 8)))
    out, weight = Q.attend(q, k, v, 4, 6, 2, 8 ** -0.5)
    for i in range(2):
        want = A.attention_decode_twopass(q[i], k[:5 + i], v[:5 + i], 2, 8 ** -0.5)
        assert np.allclose(out[i], want, atol=1e-6)
    assert (weight >= np.abs(out)).all()
    assert not Q.attend(q, k, v, 4, 5, 2, 1.0)[0][1].any()  # its row lies past length
    assert not Q.attend(q, k, v, 4, 6, 1, 1.0)[0][1].any()  # it does not count


def test_verification_by_hand():
    p = np.array([[0.5, 0.3, 0.2, 0.0], [0.1, 0.2, 0.3, 0.4], [0.25] * 4])
    q = np.array([[0.2, 0.6, 0.2, 0.0], [0.1, 0.1, 0.4, 0.4], [0.25] * 4])
    # chain: u q(1) = 0.49 * 0.6 < 0.3 stands, 0.51 * 0.6 does not
    assert Q.verify([9, 1, 3], p, [0.0, 0.49, 0.9], draft=q) == ([0, 1, 2], [1, 3, 0])
    # refused: max(p - q, 0) = [0.3, 0, 0, 0] leaves token 0
    assert Q.verify([9, 1, 3], p, [0.99, 0.51, 0.9], draft=q) == ([0], [0])
    # behind an accepted draft 1 a refusal of 2: max(p - q, 0) = [0, 0.1, 0, 0]
    assert Q.verify([9, 1, 2], p, [0.0, 0.1, 0.8], draft=q) == ([0, 1], [1, 1])
    # brothers without a distribution: 1 refused (0.6 >= 0.3), 0 against 1 - 0.3
    assert Q.verify([9, 1, 0], p, [0.0, 0.6, 0.7], [-1, 0, 0]) == ([0, 2], [0, 0])
    # both refused: token 2 is left; the same token twice weighs nothing again
    assert Q.verify([9, 1, 0], p, [0.5, 0.6, 0.8], [-1, 0, 0]) == ([0], [2])
    assert Q.verify([9, 1, 1], p, [0.6, 0.6, 0.0], [-1, 0, 0]) == ([0], [0])
    # drawn brothers: r = [0.3, 0, 0, 0], Z = 0.3, then 0.9 * 0.2 * 0.3 < 0.3
    assert Q.verify([9, 1, 0], p, [0.5, 0.9, 0.9], [-1, 0, 0], q) == ([0, 2], [0, 2])
    # no drafts; nothing left; a leaf draws from p
    assert Q.verify([9, 1], p[:2], [0.5, 0.5], count=0) == ([], [])
    assert Q.verify([9], np.zeros((1, 4)), [0.5]) == ([0], [-1])
    assert Q.verify([9], p[:1], [0.79]) == ([0], [1])
    assert Q.verify([9, 7], p[:2], [0.99, 0.0], draft=q[:2]) == ([0], [0])


def test_verified_tokens_follow_the_target():
    # a wrong residual, or children tested against the wrong Z, shifts the
    # distribution of the first new token: three drawn brothers, 20000 trials;
    # 5 standard deviations of a share are at most 5 * 0.5 / sqrt(20000) = 0.018
    rng = np.random.default_rng(3)
    p = np.array([0.4, 0.1, 0.2, 0.3])
    q = np.array([0.1, 0.6, 0.2, 0.1])
    for draft in (q, None):
        seen = np.zeros(4)
        for _ in range(20000):
            kids = rng.choice(4, 3, p=q) if draft is not None else [1, 1, 3]
            rows = np.stack([p, p, p, p])
            _, new = Q.verify([0, *kids], rows, rng.random(4), [-1, 0, 0, 0],
                              None if draft is None else np.stack([q] * 4))
            seen[new[0]] += 1
        assert np.abs(seen / seen.sum() - p).max() < 0.018


def test_least_and_step_are_cut_where_float16_ends():
    """By hand: 3e38 is 65504 + 15 * 65504; 20000 .. 120000 has step 6668 (4
    apart there); -3e38 .. 3e38 becomes -65504 + 15 * 65504 at most."""
    x = np.zeros((3, 32))
    x[0], x[1, :16], x[1, 16:] = 3e38, 20000.0, 120000.0
    x[2, ::2], x[2, 1::2] = -3e38, 3e38
    got = Q.decode(*Q.encode(x))
    assert (got[0] == 16 * 65504).all()
    assert (got[1, :16] == 20000).all() and (got[1, 16:] == 20000 + 15 * 6668).all()
    assert (got[2, ::2] == -65504).all() and (got[2, 1::2] == 14 * 65504).all()
