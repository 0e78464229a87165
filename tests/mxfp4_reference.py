"""MXFP4 in NumPy and float64, for the tests: 32 values of a row share a power-of-two
scale (an E8M0 byte, biased by 127), each is an e2m1 code.  Rounding is a search
among the eight sizes, not the arithmetic that the kernels use."""
import numpy as np

SIZES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
BORDERS = (SIZES[1:] + SIZES[:-1]) / 2          # halfway between neighbours
# a value on a border goes to the even code of the two
BORDER_UP = (np.arange(7) % 2 == 1)             # border i lies between codes i and i + 1


def exponents(amax):
    """Biased exponents of block maxima: the smallest scale at which the largest value
    rounds to 6 or less, that is, is below 7 units (7 is a tie, with 8 the even code)."""
    amax = np.asarray(amax, dtype=np.float64)
    e = np.zeros(amax.shape, dtype=np.int64)
    fine = np.isfinite(amax) & (amax > 0)
    a = np.where(fine, amax, 1.0)
    guess = np.floor(np.log2(a)).astype(np.int64) - 4
    for _ in range(6):
        guess = np.where(a >= 7.0 * np.ldexp(1.0, guess), guess + 1, guess)
    e = np.where(fine, np.maximum(guess + 127, 0), 0)
    return np.where(np.isfinite(amax), e, 255)


def codes(v, e):
    """e2m1 codes of values [..., 32] at biased exponents [...]."""
    v = np.asarray(v, dtype=np.float64)
    nan = (e == 255)[..., None]
    m = np.where(nan, 0.0, v) / np.ldexp(1.0, np.where(e == 255, 127, e) - 127)[..., None]
    a = np.abs(m)
    c = np.zeros(a.shape, dtype=np.int64)
    for border, up in zip(BORDERS, BORDER_UP):
        c += (a >= border) if up else (a > border)
    return np.where(nan, 0, c | (np.signbit(m).astype(np.int64) << 3))


def quantise(v):
    """(packed codes [R, C/2], exponents [R, C/32]) of rows."""
    v = np.asarray(v, dtype=np.float64)
    b = v.reshape(v.shape[0], -1, 32)
    with np.errstate(invalid="ignore"):
        e = exponents(np.where(np.isnan(b).any(-1), np.nan, np.abs(b).max(-1)))
    c = codes(b, e).reshape(v.shape)
    return (c[:, 0::2] | (c[:, 1::2] << 4)).astype(np.uint8), e.astype(np.uint8)


def values(q, e):
    """float64 values of packed codes [R, C/2] and exponents [R, C/32]."""
    c = np.stack((q & 15, q >> 4), -1).reshape(q.shape[0], -1).astype(np.int64)
    v = np.where(c >= 8, -1.0, 1.0) * SIZES[c & 7]
    e = e.astype(np.int64)
    s = np.where(e == 255, np.nan, np.ldexp(1.0, np.where(e == 255, 0, e) - 127))
    return (v.reshape(q.shape[0], -1, 32) * s[..., None]).reshape(q.shape[0], -1)


def operand_rows(packed, exps):
    """Rows of a packed operand [rows/32, K/64, 64, 16], [K/128, rows, 4], value by value
    from the layout's definition: (codes [rows, K/2], exponents [rows, K/32])."""
    rows, k = packed.shape[0] * 32, packed.shape[1] * 64
    q = np.empty((rows, k // 2), dtype=np.uint8)
    e = np.empty((rows, k // 32), dtype=np.uint8)
    for p in range(rows):
        for b in range(k // 32):
            q[p, b * 16:(b + 1) * 16] = packed[p // 32, b // 2, (b % 2) * 32 + p % 32]
            e[p, b] = exps[b // 4, p, b % 4]
    return q, e


def packed_operand(q, e):
    """The other way."""
    rows, k = q.shape[0], q.shape[1] * 2
    packed = np.empty((rows // 32, k // 64, 64, 16), dtype=np.uint8)
    exps = np.empty((k // 128, rows, 4), dtype=np.uint8)
    for p in range(rows):
        for b in range(k // 32):
            packed[p // 32, b // 2, (b % 2) * 32 + p % 32] = q[p, b * 16:(b + 1) * 16]
            exps[b // 4, p, b % 4] = e[p, b]
    return packed, exps


def gate_up_column(p, d_ff):
    """(0 gate / 1 up, column) of packed gate/up row p."""
    return (p // 32) % 2, (p // 64) * 32 + p % 32


def half_step(m):
    """Half the distance between the neighbours of |m| units (and 6 to 7: half of 2)."""
    return np.where(m < 2, 0.25, np.where(m < 4, 0.5, 1.0))


def swiglu_with_bound(g, u, dg, du):
    """h = silu(g) u in float64 and how far a float32 computation from sums off by dg and
    du may be from it: |silu'| <= 1.1, and 2^-19 relative for the exponential (its
    argument's rounding grows with |g| <= 88), reciprocal and products."""
    with np.errstate(over="ignore"):
        s = g / (1.0 + np.exp(-g))
    h = s * u
    return h, 1.1 * dg * (np.abs(u) + du) + np.abs(s) * du + np.abs(h) * 2.0**-19 + 1e-37


def check_quantised(q, e, h, bound, what=""):
    """Codes and exponents of rows whose exact values are h, each known to `bound`: the
    exponent is one that a value within the bound has, every code the nearest or, within
    the bound, across a border."""
    b, d = h.reshape(h.shape[0], -1, 32), bound.reshape(h.shape[0], -1, 32)
    amax, dmax = np.abs(b).max(-1), d.max(-1)
    lo, hi = exponents(np.maximum(amax - dmax, 0)), exponents(amax + dmax)
    assert ((e >= lo) & (e <= hi)).all(), f"{what}: exponents"
    scale = np.ldexp(1.0, e.astype(np.int64) - 127)[..., None]
    got = values(q, e).reshape(b.shape)
    # the half step where the value may lie, the bound's upper end included
    allowed = half_step((np.abs(b) + d) / scale) * scale + d
    off = np.abs(got - b) - allowed
    assert (off <= 0).all(), f"{what}: {int((off > 0).sum())} codes beyond half a step, by {off.max()}"


def product_bound(a, b, k):
    """How far a float32 sum over k exact products may be from the exact one, however it
    is ordered and whether it rounds or cuts: k steps of 2^-23 of the sum of sizes."""
    return k * 2.0**-23 * (np.abs(a) @ np.abs(b).T)
