"""The oracle of the 4-bit form: hand-made groups, the bound it promises, its bytes."""

import numpy as np

from oracle import q4


def _group(*head):
    x = np.zeros((1, 128), np.float32)
    x[0, :len(head)] = head
    return x


def test_hand_made_groups():
    c, s = q4.quantise(_group(8.0, -8.0, 3.5, 4.5, -7.6, 0.49, 0.5, 0.51))
    assert s[0, 0] == -1.0 and s[0, 1] == 0.0
    # x / -1: -8, 8 (limited to 7), -3.5 and -4.5 (ties to even), 7.6, and about zero
    assert c[0, :8].tolist() == [0, 15, 4, 4, 15, 8, 8, 7]
    assert (c[0, 8:] == 8).all()
    c, s = q4.quantise(_group(-8.0, 8.0))  # the first of equal magnitudes
    assert s[0, 0] == 1.0 and c[0, :2].tolist() == [0, 15]
    c, s = q4.quantise(_group(np.inf, 1.0))
    assert np.isnan(s[0, 0]) and (c[0] == 8).all() and s[0, 1] == 0
    c, s = q4.quantise(_group(1e30, -1e29))
    assert s[0, 0] == -65504 and c[0, :3].tolist() == [0, 15, 8]
    assert q4.quantise(_group(1e-9, 1e-10))[1][0, 0] == 0


def test_bound_and_bytes():
    rng = np.random.default_rng(1)
    x = (rng.standard_normal((200, 128)) * np.exp(rng.uniform(-3, 3, (200, 1)))).astype(np.float32)
    c, s = q4.quantise(x)
    err = np.abs(q4.values(c, s) - x)
    step = np.repeat(np.abs(s.astype(np.float64)), 32, -1)
    assert (err <= step * (0.5 + 2 ** -7) + 0 * err)[c != 15].all() and (err <= step * (1 + 2 ** -7)).all()
    rms = np.sqrt((err ** 2).sum() / (x.astype(np.float64) ** 2).sum())
    assert 0.05 < rms < 0.1
    b = q4.rows(c, s)
    assert b.shape == (200, 72)
    c2, s2 = q4.from_rows(b)
    assert np.array_equal(c, c2) and np.array_equal(s, s2)


def test_attention_of_one_key_is_its_value():
    rng = np.random.default_rng(2)
    q, k, v = (rng.standard_normal(sh) for sh in ((3, 4, 128), (5, 2, 128), (5, 2, 128)))
    out, bound = q4.attend(q, k, v, [0, 2, 4], [0, 2, 4], 0.1)
    assert np.allclose(out[1, 3], v[2, 1]) and (bound > 0).all()
    out, _ = q4.attend(q, k, v, [0] * 3, [4] * 3, 0.0)
    assert np.allclose(out[0, 0], v[:, 0].mean(0))
