"""The plain forms of the paged operators against what their definitions fix by themselves."""

import numpy as np
import pytest

from oracle import attention as oa
from oracle import paged as op
from oracle import rope as orope


@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (3, 2), (100, 5)])
def test_seen_counts(window, sinks):
    keep = op.seen(np.arange(-1, 9), 9, window, sinks)
    for r, pos in enumerate(range(-1, 9)):
        want = {j for j in range(9) if j <= pos and (not window or j > pos - window or j < sinks)}
        assert set(np.flatnonzero(keep[r])) == want


def test_attend_without_window_is_causal_attention():
    rng = np.random.default_rng(0)
    q, k, v = (rng.standard_normal((7, 8)).astype(np.float32) for _ in range(3))
    got, weight = op.attend(q, k, v, op.seen(np.arange(7), 7), 0.3)
    want = oa.attention_bhsd(q[None, None], k[None, None], v[None, None], causal=True, sm_scale=0.3, dtype="float32")
    np.testing.assert_allclose(got, want[0, 0], atol=1e-6)
    assert (weight >= np.abs(got) - 1e-12).all()
    empty, _ = op.attend(q[:1], k, v, np.zeros((1, 7), bool), 0.3)
    assert (empty == 0).all()


def test_rotate_pairs():
    rng = np.random.default_rng(1)
    x = rng.standard_normal((5, 12)).astype(np.float32)
    angle = rng.standard_normal((5, 4))
    c, s = np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)
    half = op.rotate(x, c, s, False)
    np.testing.assert_array_equal(half[:, :8], orope.rotate(x[:, :8], c, s))
    inter = op.rotate(x, c, s, True)
    order = np.r_[0:8:2, 1:8:2]
    np.testing.assert_array_equal(inter[:, order], op.rotate(x[:, np.r_[order, 8:12]], c, s, False)[:, :8])
    for y in (half, inter):
        np.testing.assert_array_equal(y[:, 8:], x[:, 8:])


def test_append_places_tokens_and_skips():
    rng = np.random.default_rng(2)
    kp = np.zeros((3, 1, 16, 4), np.float32)
    table = np.array([[2, 0], [1, 7]])
    k = rng.standard_normal((2, 3, 1, 4)).astype(np.float32)
    _, kn, vn = op.append(None, k, -k, kp, kp, table, [15, 14], new_lens=[2, 3])
    np.testing.assert_array_equal(kn[2, 0, 15], k[0, 0, 0])
    np.testing.assert_array_equal(kn[0, 0, 0], k[0, 1, 0])
    np.testing.assert_array_equal(vn[1, 0, 14:], -k[1, :2, 0])
    assert np.count_nonzero(kn.any(-1)) == 4  # the third token of sequence 1 has no page


def test_beam_select_small():
    x = np.log(np.array([[[0.5, 0.25, 0.25], [0.125, 0.125, 0.75]]]))
    s, p, t = op.beam_select(x, np.log([[0.5, 0.5]]), 4)
    np.testing.assert_allclose(np.exp(s[0]), [0.375, 0.25, 0.125, 0.125])
    assert p[0].tolist() == [1, 0, 0, 0] and t[0].tolist() == [2, 0, 1, 2]
    s, p, t = op.beam_select(x, np.array([[-np.inf, 0.0]]), 5)
    assert p[0].tolist() == [1, 1, 1, -1, -1] and t[0].tolist() == [2, 0, 1, -1, -1]
