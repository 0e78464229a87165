"""The e4m3 rule of rows that are not ordinary, from its definition (the GPU calls are held to
the same function bit for bit in ``test_gpu_e4m3_rows.py``)."""
import numpy as np
import pytest

import oracle as O


def _rows():
    """[12, 40] float32 rows by what their largest value is."""
    a = np.random.default_rng(1).standard_normal((12, 40)).astype(np.float32)
    a[1, 0] = np.nan
    a[2, 39] = -np.nan
    a[3, 7] = np.inf
    a[4, 8] = -np.inf
    a[5, [0, 1, 2]] = np.inf, -np.inf, np.nan
    a[6] = 0.0
    for row, most in ((7, 2.0**-119), (8, 1e-36), (9, 2.0**-126), (10, 3e-39)):
        a[row] = a[row] / np.abs(a[row]).max() * np.float32(most)
    a[11, 1:] = 0.0
    a[11, 0] = 2.0**-133
    return a


BAD = [1, 2, 3, 4, 5]


def test_rows_that_are_not_finite_read_back_as_nan():
    q, s = O.quantize_rows_e4m3(_rows())
    back = O.e4m3_decode(q) * s[:, None]
    assert np.array_equal(np.isnan(back).all(1), np.isin(np.arange(12), BAD))
    assert not np.isnan(np.delete(back, BAD, axis=0)).any()


@pytest.mark.parametrize("row", [0, 6, 7, 8, 9, 10, 11])
def test_small_rows_keep_their_values(row):
    """Half a step of the code, the factor's, the product's and the scale's roundings, where the
    scale is subnormal half of float32's smallest step times the code."""
    a = _rows()
    q, s = O.quantize_rows_e4m3(a)
    v = a[row].astype(np.float64)
    back = O.e4m3_decode(q[row]).astype(np.float64) * np.float64(s[row])
    bound = np.maximum(np.abs(v) * 2.0**-4, 2.0**-10 * np.float64(s[row])) * (1 + 2.0**-20)
    bound += np.abs(v) * 4 * 2.0**-24 + 448 * 2.0**-150
    assert (np.abs(back - v) <= bound).all()


def test_columns_are_rows_of_the_transpose():
    a = _rows()
    q, s = O.quantize_cols_e4m3(a.T)
    qr, sr = O.quantize_rows_e4m3(a)
    assert np.array_equal(q, qr.T) and np.array_equal(s, sr, equal_nan=True)


def test_blocks_that_are_not_finite_read_back_as_nan():
    a = _rows()[:, :32].repeat(2, axis=1)
    a[1, 32:] = 1.0                     # NaN in the first block only
    q, e = O.quantize_blocks_e4m3(a)
    bad = ~np.isfinite(a.reshape(12, 2, 32)).all(2)
    assert np.array_equal(e == 255, bad) and bad[1].tolist() == [True, False]
    back = O.dequantize_blocks_e4m3(q, e).reshape(12, 2, 32)
    assert np.isnan(back[bad]).all() and np.isfinite(back[~bad]).all()
