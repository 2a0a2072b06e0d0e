"""The bounds that the attention tests hold results to, tried on results that are wrong: none of them may pass."""
import numpy as np
import pytest

import kv4_bounds as kb


def exact(k, v, q, scale, window=0, whole_q=True):
    n, rows = k.shape[0], q.shape[0]
    return kb.Exact(q, k, v, np.arange(n - rows, n), np.float64(np.float32(scale)), window, whole_q)


def test_rounding_in_one_step():
    x = np.array([5.078125 + 2.0**-30, 5.078125, 5.078125 - 2.0**-30, 1.0 + 2.0**-8, 1.0 + 3 * 2.0**-8, 3.4e38, 3.39e38, 2.0**-134, 3 * 2.0**-134, -0.0, np.inf, np.nan])
    want = [5.09375, 5.0625, 5.0625, 1.0, 1.015625, np.inf, kb.BF16_MAX, 0.0, 2.0**-132, -0.0, np.inf, np.nan]
    assert np.array_equal(kb.bf16_once(x), want, equal_nan=True)


@pytest.mark.parametrize("case", kb.LONG)
def test_a_long_result_that_lost_any_run_of_tokens_is_refused(case):
    k, v, at, qs, scale = kb.long_case(*case)
    n, rows = case[:2]
    exacts = [exact(k, v, q, scale) for q in qs]
    for e in exacts:
        assert e.over(e.y).max() <= 0 and e.over(np.zeros_like(e.y)).min() > 0
    assert len(at) == -(-n // 64)
    refused = set()                                                        # runs without which some row is refused
    for e in exacts:
        for h in range(e.heads):
            p, vv = e._weights(h, e.seen), e.held[1][:, h // e.group]
            for r in range(rows):
                for c in range(np.flatnonzero(e.q[r, h])[0], (n - rows) // 64, classes_of(case)):
                    gone = slice(64 * c, 64 * c + 64)
                    y = (e.y[r, h] - p[r, gone] @ vv[gone]) / (1 - p[r, gone].sum())
                    if np.any(np.abs(y - e.y[r, h]) > e.bound[r, h]):
                        refused.add(c)
    assert refused == set(range((n - rows) // 64))                         # (behind that, a run is not seen by every row)


def classes_of(case):
    cols = case[1] * case[3]
    return min(-(-16 // cols) * cols, case[4])


@pytest.mark.parametrize("case", kb.EDGES)
def test_a_mask_off_by_one_is_refused(case):
    n, rows, window = case[0], case[1], case[-1]
    k, v, q, scale = kb.edge_case(*case)
    e = exact(k, v, q, scale, window)
    assert e.over(e.y).max() <= 0
    tokens = np.arange(n - rows, n)
    if window != 1:
        assert np.all(e.over(e.masked(kb.visible(tokens - 1, n, window and window - 1))) > 0)              # the row's own token left out
    assert np.all(e.over(e.masked(kb.visible(tokens + 1, n, window and window + 1)))[:-1] > 0)             # the next one seen
    if window:
        cut = tokens >= window                                                                            # rows that have passed a token
        assert cut.any() and np.all(e.over(e.masked(kb.visible(tokens, n, window + 1)))[cut] > 0)
        if window != 1:
            assert np.all(e.over(e.masked(kb.visible(tokens, n, window - 1)))[tokens >= window - 1] > 0)


@pytest.mark.parametrize("case", kb.RANDOM)
def test_zeros_and_neighbours_are_refused(case):
    k, v, q, scale = kb.random_case(*case)
    e = exact(k, v, q, scale, whole_q=False)
    assert e.over(e.y).max() <= 0 and np.all(e.over(np.zeros_like(e.y)) > 0)
    assert np.all(e.over(np.roll(e.y, 1, -1)) > 0)                         # the right size in the wrong places
    if q.shape[0] > 1:
        assert np.all(e.over(np.roll(e.y, 1, 0)) > 0)
