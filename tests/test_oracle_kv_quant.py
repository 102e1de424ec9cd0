"""The oracle of the 4- and 8-bit cache: its tables, its rounding, its block exponents."""
import numpy as np
import pytest
import torch

from oracle import kv_quant_oracle as K


def test_tables():
    assert K.FP8[-1] == 448.0 and K.FP8[1] == 2.0 ** -9 and (np.diff(K.FP8) > 0).all()
    torch_table = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(K.FP8, torch_table)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("bits,top,largest", [(4, 7.0, 6.0), (8, 464.0, 448.0)])
def test_block_exponents(bits, top, largest, dtype):
    lo, hi = K.exponent_range(bits, dtype)
    assert largest * 2.0 ** hi <= K.MAX[dtype] < largest * 2.0 ** (hi + 1) * (8 / 6 if bits == 4 else 8 / 7)
    for amax in [0.0, 2.0 ** lo, top * 2.0 ** lo, top * 2.0 ** lo * (1 + 1e-9), 1.0, 1.75, 1.76, 6.0, 7.0, 7.5, 8.0,
                 464.0, 464.5, K.MAX[dtype]]:
        if amax > K.MAX[dtype]:
            continue
        e = K.block_exponent(amax, bits, dtype)
        assert lo <= e <= hi
        assert amax <= top * 2.0 ** e or e == hi
        assert e == lo or amax > top * 2.0 ** (e - 1)
        x = np.zeros(8)
        x[3] = -amax
        assert int(K.encode(x, bits, dtype)[1][0]) == e + 127


@pytest.mark.parametrize("bits", [4, 8])
def test_rounding_is_to_the_nearest_with_ties_to_even(bits):
    rng = np.random.default_rng(0)
    table = K.FP4 if bits == 4 else K.FP8
    mid = (table[1:] + table[:-1]) / 2
    for e in (0, -5, 9):
        for i, m in enumerate(mid):
            x = np.array([table[-1], m, -m, np.nextafter(m, 0), np.nextafter(m, 1e9), table[i], 0.0, -table[i + 1]]) * 2.0 ** e
            y = K.held(x, bits, "f32") / 2.0 ** e
            even = table[i] if i % 2 == 0 else table[i + 1]
            assert y.tolist() == [table[-1], even, -even, table[i], table[i + 1], table[i], 0.0, -table[i + 1]]
    x = rng.standard_normal((50, 64))
    codes, scales = K.encode(x, bits, "bf16")
    y = K.decode(codes, scales, bits)
    unit = np.repeat(2.0 ** (scales.astype(float) - 127), 8, axis=1)
    grid = np.concatenate((-table[::-1], table))
    best = np.abs(x[..., None] / unit[..., None] - grid).min(axis=-1)
    assert np.allclose(np.abs(x - y) / unit, best, atol=0, rtol=1e-12)
    if bits == 8:  # torch rounds the same way once the block's power of two is taken out
        t = torch.tensor(x / unit).to(torch.float32).to(torch.float8_e4m3fn).double().numpy()
        assert np.array_equal(t * unit, y)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("bits", [4, 8])
def test_values_are_exact_in_the_type_and_bad_blocks_are_nan(bits, dtype):
    torch_type = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}[dtype]
    rng = np.random.default_rng(1)
    x = rng.standard_normal((400, 32)) * 10.0 ** rng.uniform(-9, 4.5, (400, 1))
    y = K.held(np.clip(x, -K.MAX[dtype], K.MAX[dtype]), bits, dtype)
    assert np.array_equal(torch.tensor(y).to(torch_type).double().numpy(), y)
    for bad in (np.nan, np.inf, -np.inf, K.MAX[dtype] * 1.01):
        x = np.ones(32)
        x[9] = bad
        y = K.held(x, bits, dtype)
        assert np.isnan(y[8:16]).all() and (np.delete(y, slice(8, 16)) == 1).all()
    assert (K.held(np.full(32, K.MAX[dtype]), bits, dtype) <= K.MAX[dtype]).all()


def test_record():
    assert [K.row_bytes(4, 128), K.row_bytes(8, 128), K.row_bytes(4, 64), K.row_bytes(8, 64), K.row_bytes(4, 32)] == [80, 144, 48, 80, 32]
    x = np.array([0.5, -1.0, 6.0, 0, 0, 0, 0, 0] + [2.0] * 24)
    r = K.record(x, 4, "bf16")
    assert r[0] == 1 | (0xA << 4) and r[1] == 7 and r[16:20].tolist() == [127, 126, 126, 126] and not r[20:].any()


def test_attention_leaves_masked_keys_out():
    rng = np.random.default_rng(2)
    q, k, v = rng.standard_normal((1, 2, 3, 8)), rng.standard_normal((1, 1, 5, 8)), rng.standard_normal((1, 1, 5, 8))
    mask = np.ones((1, 3, 5), bool)
    mask[0, 1, 2] = False
    mask[0, 2] = False
    want, _ = K.attention(q, k, v, mask, 0.3)
    t = torch.nn.functional.scaled_dot_product_attention(
        torch.tensor(q), torch.tensor(k).expand(1, 2, 5, 8), torch.tensor(v).expand(1, 2, 5, 8),
        attn_mask=torch.tensor(mask)[:, None], scale=0.3).transpose(1, 2).numpy()
    assert np.allclose(want[0, :2], t[0, :2])
    v[0, 0, 2] = np.nan
    k[0, 0, 2] = np.inf
    got, _ = K.attention(q, k, v, mask, 0.3)
    assert np.array_equal(got[0, 1], want[0, 1]) and np.isnan(got[0, 0]).all() and not got[0, 2].any()
