"""A KV cache in 4 or 8 bits, in float64: the codes of a row, its record, attention over the values.

Pinned by: the tables of the two element formats written out value by value, rounding by search for the
nearest table entry, torch's own e4m3 conversion (tests/test_oracle_kv_quant.py).  No counterpart in the
reference, whose cache has the model's type: parity unpinned.
"""
import numpy as np

BLOCK = 8
FP4 = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
# e4m3: 4 exponent bits with bias 7, 3 mantissa bits, no infinities; code 127 is NaN
FP8 = np.array([(c % 8) / 8 * 2.0 ** -6 if c < 8 else (1 + c % 8 / 8) * 2.0 ** (c // 8 - 7) for c in range(127)])
MAX = {"bf16": 255 * 2.0 ** 120, "f16": 65504.0, "f32": float(np.finfo(np.float32).max)}


def exponent_range(bits, dtype):
    largest = 15 if dtype == "f16" else 127
    lo = {"f16": {4: -23, 8: -15}}.get(dtype, {4: -100, 8: -100})[bits]
    return lo, largest - {4: 2, 8: 8}[bits]


def block_exponent(amax, bits, dtype):
    """Smallest e with amax <= top * 2^e, inside the range of the type."""
    lo, hi = exponent_range(bits, dtype)
    top = {4: 7.0, 8: 464.0}[bits]
    e = lo
    while e < hi and amax > top * 2.0 ** e:
        e += 1
    return e


def encode(x, bits, dtype):
    """x (..., D) float64 -> codes (..., D) uint8 (with sign), scale bytes (..., D / 8) uint8."""
    x = np.asarray(x, dtype=np.float64)
    table = FP4 if bits == 4 else FP8
    blocks = x.reshape(-1, BLOCK)
    codes = np.zeros(blocks.shape, dtype=np.uint8)
    scales = np.zeros(len(blocks), dtype=np.uint8)
    # exponents by table over all blocks at once (block_exponent is the definition, one block at a time)
    lo, hi = exponent_range(bits, dtype)
    bad = ~(np.abs(blocks) <= MAX[dtype]).all(axis=1)
    amax = np.where(bad, 0.0, np.abs(np.where(bad[:, None], 0.0, blocks)).max(axis=1))
    limits = {4: 7.0, 8: 464.0}[bits] * 2.0 ** np.arange(lo, hi + 1, dtype=np.float64)
    e = lo + np.minimum(np.searchsorted(limits, amax, side="left"), hi - lo)
    y = np.abs(np.where(bad[:, None], 0.0, blocks)) / 2.0 ** e[:, None].astype(np.float64)
    below = np.clip(np.searchsorted(table, y, side="right") - 1, 0, len(table) - 2)
    down, up = y - table[below], table[below + 1] - y
    codes = np.where((down > up) | ((down == up) & (below % 2 == 1)), below + 1, below).astype(np.uint8)
    sign = np.signbit(np.where(bad[:, None], 0.0, blocks))
    codes |= np.where(sign, 8 if bits == 4 else 128, 0).astype(np.uint8)
    scales = np.where(bad, 255, e + 127).astype(np.uint8)
    return codes.reshape(x.shape), scales.reshape(*x.shape[:-1], -1)


def decode(codes, scales, bits):
    table = FP4 if bits == 4 else FP8
    sign_bit = 8 if bits == 4 else 128
    mag = table[codes & (sign_bit - 1)]
    x = np.where(codes & sign_bit, -mag, mag).reshape(*scales.shape, BLOCK)
    s = np.where(scales == 255, np.nan, 2.0 ** (scales.astype(np.float64) - 127))
    return (x * s[..., None]).reshape(codes.shape)


def held(x, bits, dtype):
    return decode(*encode(x, bits, dtype), bits)


def row_bytes(bits, dim):
    return -(-(dim * bits // 8 + dim // BLOCK) // 16) * 16


def record(x, bits, dtype):
    """(..., D) -> (..., row_bytes) uint8 with zeros in the padding."""
    codes, scales = encode(x, bits, dtype)
    dim = codes.shape[-1]
    out = np.zeros((*codes.shape[:-1], row_bytes(bits, dim)), dtype=np.uint8)
    packed = codes if bits == 8 else codes[..., 0::2] | (codes[..., 1::2] << 4)
    out[..., : packed.shape[-1]] = packed
    out[..., packed.shape[-1] : packed.shape[-1] + scales.shape[-1]] = scales
    return out


def rotate(x, cos, sin):
    """x (..., D) float64, cos and sin (..., D): x * cos + rotate_half(x) * sin."""
    half = x.shape[-1] // 2
    turned = np.concatenate((-x[..., half:], x[..., :half]), axis=-1)
    return x * cos + turned * sin


def attention(q, k, v, mask, scale):
    """q (B, H, n, D), k, v (B, Hkv, kv, D) float64 (NaN allowed), mask (B, n, kv) bool.
    Returns out (B, n, H, D) and the mean |v| under the same weights (NaN left out of it).  Masked keys take no
    part, whatever they hold; a query without keys gives zeros."""
    B, H, n, D = q.shape
    group = H // k.shape[1]
    out = np.zeros((B, n, H, D))
    size = np.zeros((B, n, H, D))
    for b in range(B):
        for h in range(H):
            kk, vv = k[b, h // group], v[b, h // group]
            for i in range(n):
                on = mask[b, i]
                if not on.any():
                    continue
                with np.errstate(invalid="ignore"):
                    s = kk[on] @ q[b, h, i] * scale
                    p = np.exp(s - s.max())
                    p /= p.sum()
                    out[b, i, h] = p @ vv[on]
                    size[b, i, h] = np.nan_to_num(p) @ np.abs(np.nan_to_num(vv[on]))
    return out, size
