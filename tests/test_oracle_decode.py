"""The oracle of rope and sample against small cases written out."""
import numpy as np

from oracle import decode as DC


def test_rope_by_hand():
    x = np.array([[[1.0, 2.0, 3.0, 4.0, 9.0]]])
    y, angle, pair = DC.rope(x, [1], [np.pi / 2, np.pi])
    assert np.allclose(y, [[[-3, -2, 1, -4, 9]]]) and np.allclose(angle, [np.pi]) and pair[0, 0].tolist() == [4, 6, 4, 6, 0]
    y, _, _ = DC.rope(x, [1], [np.pi / 2, np.pi], interleaved=True, magnitude=2.0)
    assert np.allclose(y, [[[-4, 2, -6, -8, 9]]])
    back, _, _ = DC.rope(DC.rope(x, [7], [0.3, 0.1])[0], [7], [0.3, 0.1], inverse=True)
    assert np.allclose(back, x)
    assert DC.positions([5, 3], [2, 1]).tolist() == [3, 4, 2]


def test_kept_by_hand():
    x = np.log([0.1, 0.4, 0.2, 0.2, 0.1])
    k = lambda *a: np.nonzero(DC.kept(x, *a)[0])[0].tolist()
    assert k(1.0) == [0, 1, 2, 3, 4] and k(1.0, 2) == [1, 2] and k(0.0) == [1] and k(1.0, 0, 0.39) == [1]
    assert k(1.0, 0, 0.7) == [1, 2, 3] and k(1.0, 2, 0.7) == [1, 2] and k(1.0, 0, 1.0, 0.3) == [1, 2, 3] and k(1.0, 0, 0.0) == [1]
    w, _ = DC.kept([np.nan, -np.inf, 0.0], 1.0)
    assert w.tolist() == [0, 0, 1] and not DC.kept([np.nan, -np.inf], 1.0)[0].any()
    w, _ = DC.kept(x, 1.0)
    assert [DC.tokens(w, u, 1e-12) for u in (0.0, 0.05, 0.3, 0.65, 0.95)] == [[0], [0], [1], [2], [4]]
    assert DC.tokens(w, 0.5, 1e-12) == [1, 2]
