"""The oracle of the window, the 8-bit cache and the page copies, pinned on the CPU."""

import numpy as np
import pytest
import torch

from oracle import serving as R
from oracle.attention import attention


def test_e4m3_is_torchs():
    codes = np.arange(256, dtype=np.uint8)
    t = torch.from_numpy(codes).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(R.e4m3_values(), t, equal_nan=True)
    rng = np.random.default_rng(0)
    x = np.concatenate([rng.uniform(-448, 448, 20000), rng.normal(0, 0.01, 20000), 2.0 ** rng.uniform(-14, 8.8, 20000),
                        (R.e4m3_values()[:126] + R.e4m3_values()[1:127]) / 2, [0.0, -0.0, np.inf, -np.inf, np.nan]])
    x = x.astype(np.float32)
    want = torch.from_numpy(x).to(torch.float8_e4m3fn)
    got = R.e4m3_codes(x)
    same = (torch.from_numpy(got) == want.view(torch.uint8)) | want.isnan()
    assert bool(same.all()) and np.array_equal(np.isnan(R.e4m3_decode(got)), want.isnan().numpy())


@pytest.mark.parametrize("top,exp", [(0.0, -100), (448.0, 0), (448.0 + 1e-9, 1), (224.0, -1), (1.75, -8), (1.76, -7),
                                     (1e-40, -100), (3.4e38, 120)])
def test_scale_for(top, exp):
    assert R.scale_for(top) == 2.0 ** exp


def test_window_is_a_loop_over_pairs():
    rng = np.random.default_rng(1)
    for L, S, left, right, sinks, causal in ((5, 9, 2, 0, 1, True), (9, 5, 1, 2, 2, False), (4, 4, -1, 1, 0, False),
                                             (6, 6, 3, -1, 2, False), (3, 7, 0, 0, 0, True)):
        q, k, v = (rng.normal(size=(1, n, 1, 4)) for n in (L, S, S))
        got = R.window(q, k, v, 0.5, left, right, sinks, causal).out
        for i in range(L):
            p, keys = i + S - L, []
            for j in range(S):
                after = j > p + (0 if causal else right) and (causal or right >= 0)
                before = left >= 0 and j < p - left and j >= sinks
                if not after and not before:
                    keys.append(j)
            if not keys:
                assert np.all(got[0, i] == 0)
                continue
            w = np.exp(0.5 * k[0, keys, 0] @ q[0, i, 0])
            assert np.allclose(got[0, i, 0], (w / w.sum()) @ v[0, keys, 0], atol=1e-12)


def test_open_window_is_plain_attention():
    rng = np.random.default_rng(2)
    q, k, v = (rng.normal(size=(2, n, 3, 8)) for n in (7, 11, 11))
    assert np.allclose(R.window(q, k, v, 0.3, -1, -1, 0, True).out, attention(q, k, v, 0.3, True), atol=1e-13)
    assert np.allclose(R.window(q, k, v, 0.3, 100, -1, 4, False).out, attention(q, k, v, 0.3), atol=1e-13)


def test_unseen_infinities_stay_out():
    v = np.ones((1, 6, 1, 4))
    v[0, 0] = np.nan
    k = v.copy()
    out = R.window(np.ones((1, 6, 1, 4)), k, v, 1.0, 2, 0, 0, True).out
    assert np.isnan(out[0, :3]).all() and np.array_equal(out[0, 3:], np.ones((3, 1, 4)))


def test_store_rule():
    """The statements of the rule, one by one, on one page of one head."""
    def cache():
        return R.Cache8(*(np.zeros((2, 1, 16, 4), np.uint8) for _ in range(2)), *(np.zeros((2, 1)) for _ in range(2)))

    def row(x):
        return np.full((1, 1, 4), x)

    c = cache()
    c.store(row(448.0), row(1.0), [0])
    assert c.scales[0][0, 0] == 1.0 and c.values(0)[0, 0, 0, 0] == 448.0 and c.scales[1][0, 0] == 2.0 ** -8
    c.store(row(900.0), row(1.0), [1])  # grows to 2^2 (448 * 2 < 900), the first code is rescaled
    assert c.scales[0][0, 0] == 4.0 and c.values(0)[0, 0, 0, 0] == 448.0 and c.values(0)[0, 0, 1, 0] == 896.0
    c.store(row(1.0), row(1.0), [2])    # does not shrink
    assert c.scales[0][0, 0] == 4.0
    c.store(row(1.0), row(1.0), [16])   # another page
    assert c.scales[0][0, 0] == 4.0 and c.scales[0][1, 0] == 2.0 ** -8
    c.store(row(1.0), row(1.0), [0])    # position 0: anew
    assert c.scales[0][0, 0] == 2.0 ** -8
    c.store(np.concatenate([row(2.0), row(3.0)]), np.concatenate([row(2.0), row(3.0)]), [5, 5])  # the last one stays
    assert c.values(0)[0, 0, 5, 0] == 3.0
    c.store(row(np.inf), row(np.nan), [6])
    assert np.isnan(c.values(0)[0, 0, 6]).all() and c.scales[0][0, 0] == 2.0 ** -7
    c.store(row(1e9), row(1.0), [-1])   # padding
    assert c.scales[0][0, 0] == 2.0 ** -7
    x = np.arange(2 * 16 * 4, dtype=np.uint8).reshape(2, 1, 16, 4)
    assert np.array_equal(R.k_rows(R.k_words(x)), x) and R.k_words(x)[0, 0].ravel()[16 * 0 + 4] == x[0, 0, 1, 0]


def test_copy_pages():
    x = np.arange(5)
    assert list(R.copy_pages(x, [(0, 3), (1, 4), (-1, 2), (2, -1)])) == [0, 1, 2, 0, 1]
