"""The MXFP4 oracle against the format's definition, by brute force."""

import numpy as np
import pytest

from oracle import quant as oq


def test_e2m1_nearest_ties_to_even_and_saturates():
    # every quarter step of the positive range, and each side of it
    for q in np.arange(0, 7, 0.125):
        for v in (q, np.nextafter(q, 9), np.nextafter(q, -9)):
            a = min(abs(v), 6.0)
            d = [abs(a - x) for x in oq.E2M1_VALUES]
            best = [i for i, x in enumerate(d) if x == min(d)]
            want = best[0] if len(best) == 1 else next(i for i in best if i % 2 == 0)
            assert oq.e2m1_encode(v) & 7 == want, v
    assert oq.e2m1_encode(1e30) == 7 and oq.e2m1_encode(-1e30) == 15
    assert oq.e2m1_encode(-0.0) == 8 and oq.e2m1_encode(-0.1) == 8


def test_block_rule():
    x = np.zeros((3, 64))
    x[0, 0], x[0, 33] = 6.0, 2.0 ** -130
    x[1, 5] = np.nan
    x[1, 40] = 7.9  # saturates: X = 0, 7.9 -> 6
    x[2, 32] = -np.inf
    codes, scales = oq.mxfp4_quantize(x)
    assert scales.tolist() == [[127, 0], [255, 127], [0, 255]]
    assert codes[0, 0] == 7 and codes[0, 33] == 0 and codes[1, 40] == 7
    v = oq.mxfp4_dequantize(codes, scales)
    assert v[0, 0] == 6.0 and v[1, 40] == 6.0
    assert np.isnan(v[1, :32]).all() and np.isnan(v[2, 32:]).all() and not np.isnan(v[2, :32]).any()


def test_representable_values_survive():
    rng = np.random.default_rng(0)
    codes = rng.integers(0, 16, (4, 96)).astype(np.uint8)
    codes[:, ::32] = 7  # a 6 in every block fixes its exponent
    scales = rng.integers(3, 250, (4, 3)).astype(np.uint8)
    c, s = oq.mxfp4_quantize(oq.mxfp4_dequantize(codes, scales))
    np.testing.assert_array_equal(s, scales)
    np.testing.assert_array_equal(c, codes)


@pytest.mark.parametrize("n,k", [(1, 32), (5, 96), (8, 256)])
def test_stored_form(n, k):
    rng = np.random.default_rng(n)
    codes, scales = rng.integers(0, 16, (n, k)), rng.integers(0, 256, (n, k // 32))
    b, w = oq.mxfp4_pack(codes, scales)
    assert b.shape == (n, k // 2) and w.shape == (-(-k // 128), -(-n // 4) * 4)
    for i in range(n):
        for j in range(k):
            assert (b[i, j // 2] >> (4 * (j % 2))) & 15 == codes[i, j]
        for j in range(k // 32):
            assert (int(w[j // 4, i]) >> (8 * (j % 4))) & 255 == scales[i, j]
