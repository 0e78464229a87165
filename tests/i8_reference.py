"""int8 rows, operands and products restated in NumPy, for the tests."""
import numpy as np


def bf16(v):
    """float32 values rounded to bf16 (ties to even), in float32; NaN stays NaN."""
    v = np.ascontiguousarray(v, dtype=np.float32)
    u = v.view(np.uint32).astype(np.uint64)
    r = ((((u + 0x7FFF + ((u >> 16) & 1)) >> 16) << 16) & 0xFFFFFFFF).astype(np.uint32).view(np.float32)
    return np.where(np.isnan(v), v, r)


def quantise(v):
    """(codes int8, scales float32) of float32 rows: the rule in single float32 operations."""
    v = np.ascontiguousarray(v, dtype=np.float32)
    with np.errstate(all="ignore"):
        amax = np.abs(v).max(-1)                      # (NaN where there is one)
        up = np.where(amax < np.float32(2.0**-64), np.float32(2.0**64), np.float32(1.0))
        zero = amax == 0
        scale = np.where(zero, np.float32(1.0), amax / np.float32(127.0)).astype(np.float32)
        inv = np.where(zero, np.float32(0.0), np.float32(127.0) / (amax * up)).astype(np.float32)
        q = np.rint(v * up[..., None] * inv[..., None])
    return np.where(np.isfinite(amax)[..., None], q, 0.0).astype(np.int8), scale


def operand(codes):
    """int8 codes [rows, K] of an expert as a packed operand keeps them."""
    rows, k = codes.shape
    return codes.reshape(rows // 32, 32, k // 32, 2, 16).transpose(0, 2, 3, 1, 4).reshape(rows // 32, k // 32, 64, 16)


def gate_up_rows(gate, up):
    """[F, K] gate and up rows in the packed order: 32 of one, 32 of the other."""
    f, k = gate.shape
    return np.stack((gate.reshape(-1, 32, k), up.reshape(-1, 32, k)), 1).reshape(2 * f, k)


def product(rows_q, rows_scale, w_q, w_scale):
    """float32 [R, n] of int8 rows times an expert's int8 rows: the exact sums rounded once,
    times the column's scale, times the row's, each product rounded to float32."""
    sums = rows_q.astype(np.float64) @ w_q.astype(np.float64).T      # below 2^53: exact
    with np.errstate(all="ignore"):
        y = sums.astype(np.float32) * w_scale.astype(np.float32)[None, :]
        return (y * rows_scale.astype(np.float32)[:, None]).astype(np.float32)


def swiglu_with_bound(g, u):
    """silu(g) u of float32 sums in float64, and how far the float32 one may be off: (1.25 |g| +
    8) 2^-24 of itself, and |g u| 2^-126 where the reciprocal is subnormal."""
    g, u = g.astype(np.float64), u.astype(np.float64)
    with np.errstate(over="ignore"):
        h = g / (1.0 + np.exp(-g)) * u
    return h, np.abs(h) * (1.25 * np.abs(g) + 8) * 2.0**-24 + np.abs(g * u) * 2.0**-126
