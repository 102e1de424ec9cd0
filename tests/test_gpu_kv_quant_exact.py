"""Keys whose rotated value lies next to the border of two codes, or of two block scales, by less than the model's type
or fp32 resolves beside it: the record is that of the exact sum wherever fp64 holds it."""
from fractions import Fraction

import numpy as np
import pytest
import torch

from oracle import kv_quant_oracle as K
from test_gpu_kv_quant import NAME, _new, _np

pytestmark = pytest.mark.gpu


def _held(block, bits, dtype):
    """What the cache holds for eight exact numbers: the format's definition in rational arithmetic."""
    table = [Fraction(float(t)) for t in (K.FP4 if bits == 4 else K.FP8)]
    lo, hi = K.exponent_range(bits, dtype)
    top, amax = (7 if bits == 4 else 464), max(abs(x) for x in block)
    e = lo
    while e < hi and amax > top * Fraction(2) ** e:
        e += 1
    out = []
    for x in block:
        y = abs(x) / Fraction(2) ** e
        best = min(abs(y - t) for t in table)
        near = [i for i, t in enumerate(table) if abs(y - t) == best]
        code = next((i for i in near if i % 2 == 0), near[0])  # (the nearest, ties to the even code)
        out.append(float(table[code] * Fraction(2) ** e * (-1 if x < 0 else 1)))
    return out


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("apart", [10, 20, 30, 40, 50])
def test_records_of_sums_next_to_a_border(apart, dtype, bits):
    from recurrent_drafting_amd import kv_cache

    dim = 32
    # every border as it is, and 2^-apart of it to either side, in either half of a row
    if bits == 4:
        borders = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0]
    else:
        borders = [1.0625, 1.1875, 1.3125, 1.9375, 3.625, 464.0, 29.0, 2.0 ** -10]
    rows = []
    for sign in (1, -1):
        for side in (0, 1, -1):
            for b in borders:
                x = np.zeros(dim)
                x[0], x[16] = sign * b, side * 2.0 ** -apart * b  # o1 = x1 - x2
                x[9], x[25] = side * 2.0 ** -apart * b, sign * b  # o2 = x2 + x1
                x[1] = x[24] = 4.0 if bits == 4 else 256.0        # (their partners are zero; they set the scale)
                if b in (7.0, 464.0):
                    x[1] = x[24] = 0.0
                rows.append(x)
    x = torch.tensor(np.stack(rows)).to(dtype)
    assert np.array_equal(_np(x), np.stack(rows))
    n = len(rows)
    cache = _new(n, 1, 1, dim, dtype, bits)
    k = x.view(n, 1, dim).cuda()
    ones = torch.ones(1, dim, dtype=dtype, device="cuda")
    _, keys, _ = kv_cache.rope_append(k.clone(), k, k.clone(), ones, ones, torch.zeros(n, 1, dtype=torch.long, device="cuda"),
                                      cache.sliced[0])
    got = _np(keys.read())[:, 0, 0]
    for r, row in enumerate(rows):
        exact = [Fraction(float(t)) for t in row]
        turned = [exact[d] - exact[d + 16] for d in range(16)] + [exact[d] + exact[d - 16] for d in range(16, 32)]
        want = [t for blk in range(0, dim, 8) for t in _held(turned[blk : blk + 8], bits, NAME[dtype])]
        assert np.array_equal(np.abs(got[r]), np.abs(want)) and np.array_equal(np.sign(got[r]), np.sign(want)), (r, row)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rotations_without_a_number(dtype, bits):
    """Infinities and NaN in either half, and sums beyond the type's largest: NaN blocks, the others as they are."""
    from recurrent_drafting_amd import kv_cache

    dim, big = 32, float(torch.finfo(dtype).max)
    rows = torch.zeros(6, dim)
    rows[:] = 0.5
    for r, (a, b) in enumerate([(np.inf, 1.0), (1.0, -np.inf), (np.nan, 1.0), (np.inf, np.inf), (-big, big), (big, -big)]):
        rows[r, 3], rows[r, 19] = a, b
    x = rows.to(dtype)
    cache = _new(6, 1, 1, dim, dtype, bits)
    k = x.view(6, 1, dim).cuda()
    ones = torch.ones(1, dim, dtype=dtype, device="cuda")
    _, keys, _ = kv_cache.rope_append(k.clone(), k, k.clone(), ones, ones, torch.zeros(6, 1, dtype=torch.long, device="cuda"),
                                      cache.sliced[0])
    got = _np(keys.read())[:, 0, 0]
    with np.errstate(invalid="ignore"):
        want = K.held(K.rotate(_np(x), np.ones(dim), np.ones(dim)), bits, NAME[dtype])
    assert np.array_equal(got, want, equal_nan=True) and np.isnan(got[:, :8]).all()
