"""The 4- and 8-bit KV cache on the GPU against the float64 oracle: rows appended (with the rotation and
without), read back, moved, and attended over.

Records and values are compared bit for bit.  Tolerance of the attention, per output element o = sum p v
with weights p (sum 1) and A = sum p |v|, u = eps / 2 of the model's type:
  u |o|                     the output's rounding
  u (A + |o|)               every weight rounded once, for the second product and for the sum it is divided by:
                            sum p d (v - o) with |d| <= u
  2 d A                     scores off by d move numerator and denominator by a factor e^d each;
                            d = D 2^-23 scale max_k sum |q k| (fp32 sums of exact products) + |s| 2^-22
                            (the score in log2 units, rounded twice) + 2^-21 (the exponential)
  n 2^-25 max |v|           fp16 weights below 2^-14 of the row's largest are rounded to multiples of 2^-24;
                            the largest is at least 1 (the running maximum is one of the scores), so the sum is too
  n 2^-125 max |v|          weights below fp32's smallest normal number 2^-126 are zero (relative to a sum that
                            is at least 1/2: the running maximum is a score as fp32 rounds it)
  (n + D) 2^-24 A           fp32 accumulation
The generic kernel keeps fp32 weights: the same bound covers it.
"""
import math
import os
import sys

import numpy as np
import pytest
import torch
from transformers.models.llama.configuration_llama import LlamaConfig

from oracle import kv_quant_oracle as K

sys.path.insert(0, os.path.join(os.path.dirname(__file__), "golden"))
import tiny_models as tm  # noqa: E402

pytestmark = pytest.mark.gpu

NAME = {torch.bfloat16: "bf16", torch.float16: "f16", torch.float32: "f32"}
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _cuda():
    return torch.device("cuda")


def _new(batch, max_len, heads, dim, dtype, bits, layers=1):
    from recurrent_drafting_amd import kv_cache

    return kv_cache.Cache(batch, max_len, layers, heads, dim, dtype, _cuda(), bits=bits)


def _tables(dim, positions, dtype):
    angle = np.outer(np.arange(positions), 1.0 / 10000.0 ** (np.arange(0, dim, 2) / dim))
    angle = np.concatenate((angle, angle), axis=1)
    return torch.tensor(np.cos(angle)).to(dtype), torch.tensor(np.sin(angle)).to(dtype)


def _np(t):
    return t.detach().cpu().double().numpy()


# ---- writing and reading ------------------------------------------------------------------------------

@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("batch,n,heads,kv_heads,dim,prev", [
    (1, 1, 2, 1, 32, 0), (2, 5, 4, 4, 64, 3), (1, 3, 3, 3, 96, 1), (2, 17, 8, 2, 128, 40), (1, 2, 2, 2, 256, 7),
    (3, 40, 12, 12, 64, 11)])
def test_rotation_and_append(batch, n, heads, kv_heads, dim, prev, dtype, bits):
    from recurrent_drafting_amd import kv_cache

    g = torch.Generator().manual_seed(dim + n)
    qkv = torch.randn(batch, n, (heads + 2 * kv_heads) * dim, generator=g).to(dtype)
    qkv[..., 3] *= 50
    position_ids = torch.randint(0, prev + n, (batch, n), generator=g)
    cos, sin = _tables(dim, prev + n, dtype)
    cache = _new(batch, prev + n + 2, kv_heads, dim, dtype, bits, layers=3)
    before = torch.randint(0, 250, cache._cache.shape, dtype=torch.uint8, generator=g)
    cache._cache.copy_(before)
    layer = 1
    for view in cache.sliced[layer]:
        view.length = prev
    d = qkv.cuda()
    q, k, v = d[..., : heads * dim], d[..., heads * dim : (heads + kv_heads) * dim], d[..., (heads + kv_heads) * dim :]
    got_q, keys, values = kv_cache.rope_append(q, k, v, cos.cuda(), sin.cuda(), position_ids.cuda(), cache.sliced[layer])
    assert torch.equal(d.cpu(), qkv)  # the projection's output is left as it was
    assert got_q.shape == (batch, heads, n, dim) and keys.shape == values.shape == (batch, kv_heads, prev + n, dim)
    assert cache.sliced[layer][0].length == cache.sliced[layer][1].length == prev + n

    x = _np(qkv).reshape(batch, n, heads + 2 * kv_heads, dim).transpose(0, 2, 1, 3)
    c, s = _np(cos)[position_ids.numpy()][:, None], _np(sin)[position_ids.numpy()][:, None]
    want_q = K.rotate(x[:, :heads], c, s)
    # two products and a sum in fp32, then the rounding to the type
    slack = (np.abs(x[:, :heads] * c) + np.abs(K.rotate(np.abs(x[:, :heads]), 0 * c, np.abs(s)))) * 2.0 ** -22
    u = torch.finfo(dtype).eps / 2
    tiny = 2.0 ** -24 if dtype == torch.float16 else 0.0
    assert (np.abs(_np(got_q) - want_q) <= u * np.abs(want_q) + slack + tiny).all()
    want = before.numpy().copy()
    code_and_scale = dim * bits // 8 + dim // 8  # the padding behind them is not written
    want[layer, 0, :, :, prev : prev + n, :code_and_scale] = K.record(
        K.rotate(x[:, heads : heads + kv_heads], c, s), bits, NAME[dtype])[..., :code_and_scale]
    want[layer, 1, :, :, prev : prev + n, :code_and_scale] = K.record(x[:, heads + kv_heads :], bits, NAME[dtype])[..., :code_and_scale]
    assert np.array_equal(cache._cache.cpu().numpy(), want)


def _special_rows(dim, dtype, rng):
    """Rows that hold what the format has borders for."""
    big = float(torch.finfo(dtype).max)
    rows = [np.zeros(dim), -np.zeros(dim), np.full(dim, big), np.full(dim, -big), np.full(dim, float(torch.finfo(dtype).tiny)),
            np.tile([7.0, 5.0, 2.5, 0.25, -0.75, 1.25, -3.5, 1.75], dim // 8), np.tile([464.0, 432.0, 0.001, 7.5, 8.5, -17, 1, 0], dim // 8),
            np.tile([1.0, np.nan, 2, 3, 4, 5, 6, 7], dim // 8), np.concatenate(([np.inf], np.ones(dim - 1))),
            np.concatenate((np.ones(dim - 1), [-np.inf])), rng.standard_normal(dim) * 1e-30, rng.standard_normal(dim) * 3e4,
            rng.integers(-64, 64, dim) / 8.0]
    return torch.tensor(np.stack(rows)).to(dtype)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [32, 64, 128, 160])
def test_append_and_read_back(dim, dtype, bits):
    rng = np.random.default_rng(dim)
    special = _special_rows(dim, dtype, rng)
    n, batch, heads = len(special), 2, 3
    x = torch.tensor(rng.standard_normal((batch, heads, n, dim))).to(dtype)
    x[1, 2] = special
    cache = _new(batch, n + 5, heads, dim, dtype, bits)
    key, value = cache.sliced[0]
    value.append(x[:, :, :2].cuda())
    value.append(x[:, :, 2:].transpose(1, 2).contiguous().cuda().transpose(1, 2))  # other strides
    assert value.length == n and key.length == 0 and not cache._cache[0, 0].any()
    got = value.slice(0)
    assert got.dtype == dtype and got.shape == (batch, heads, n, dim)
    want = K.held(_np(x), bits, NAME[dtype])
    assert np.array_equal(_np(got), want, equal_nan=True)
    rec = cache._cache[0, 1].cpu().numpy()
    assert np.array_equal(rec[:, :, :n], K.record(_np(x), bits, NAME[dtype])) and not rec[:, :, n:].any()
    assert np.array_equal(_np(value.slice(3)), want[:, :, 3:], equal_nan=True)
    assert value.slice(n).shape == (batch, heads, 0, dim)
    more = torch.tensor(rng.standard_normal((batch, heads, 1, dim))).to(dtype)
    assert np.array_equal(_np(value.cat(more.cuda())),
                          np.concatenate((want, K.held(_np(more), bits, NAME[dtype])), axis=2), equal_nan=True)
    value.append(torch.empty(batch, heads, 0, dim, dtype=dtype, device="cuda"))
    assert value.length == n + 1
    # a view whose last dimension is strided, and another float type, as an assignment would take them
    key.append(torch.tensor(rng.standard_normal((batch, heads, dim, 2))).cuda().transpose(2, 3))
    assert key.length == 2


def test_keys_next_to_a_border_are_rounded_from_the_exact_rotation():
    """A key component of 1.25 (the border of the codes 1 and 1.5) plus a rotation of less than fp32's last
    bit: the code is decided by the exact sum."""
    from recurrent_drafting_amd import kv_cache

    dim, dtype = 32, torch.bfloat16
    x = torch.zeros(4, dim, dtype=dtype)
    x[:, 0], x[:, 1] = 1.25, 4.0  # block scale 1
    x[0, 16], x[1, 16] = 2.0 ** -30, -(2.0 ** -30)  # partner of component 0
    cos, sin = torch.ones(1, dim, dtype=dtype), torch.ones(1, dim, dtype=dtype)
    x[2, 16] = 0.0
    x[3, 0], x[3, 16] = 1.75, 2.0 ** -40
    cache = _new(4, 1, 1, dim, dtype, 4)
    k = x.view(4, 1, dim).cuda()
    # component 1 alone turns too: its partner 17 is zero
    _, keys, _ = kv_cache.rope_append(k.clone(), k, k.clone(), cos.cuda(), sin.cuda(),
                                      torch.zeros(4, 1, dtype=torch.long, device="cuda"), cache.sliced[0])
    want = K.held(K.rotate(_np(x), np.ones(dim), np.ones(dim)), 4, "bf16")
    got = _np(keys.read())[:, 0, 0]
    assert np.array_equal(got, want)
    assert got[:, 0].tolist() == [1.0, 1.5, 1.0, 1.5]


# ---- attention ----------------------------------------------------------------------------------------

def _bound(q, k, v, mask, scale, dtype, out, size):
    u = torch.finfo(dtype).eps / 2
    D = q.shape[-1]
    group = q.shape[1] // k.shape[1]
    kk = np.repeat(np.abs(np.nan_to_num(k)), group, axis=1)
    dots = np.einsum("bhnd,bhkd->bnhk", np.abs(q), kk).max(axis=3) * scale
    d = (D * 2.0 ** -23 * dots + dots * 2.0 ** -22 + 2.0 ** -21)[..., None]
    n = mask.sum(axis=2)[:, :, None, None]
    vmax = np.abs(np.nan_to_num(v)).max()
    tiny = n * vmax * 2.0 ** -125
    if dtype == torch.float16:
        tiny = tiny + n * 2.0 ** -25 * vmax + 2.0 ** -25
    return 2 * u * np.abs(out) + (u + 2 * d + (n + D) * 2.0 ** -24) * size + tiny


def _tree_mask(rng, batch, n, prev, pads):
    mask = np.zeros((batch, n, prev + n), bool)
    for b in range(batch):
        mask[b, :, pads[b] : prev] = True
        up = np.eye(n, dtype=bool)
        for t in range(1, n):
            up[t] |= up[rng.integers(0, t)]
        mask[b, :, prev:] = up
    return mask


def _filled(rng, batch, kv_heads, kv, dim, dtype, bits, gain=1.0, max_len=None):
    k = torch.tensor(rng.standard_normal((batch, kv_heads, kv, dim)) * gain * np.exp(0.5 * rng.standard_normal(dim))).to(dtype)
    v = torch.tensor(rng.standard_normal((batch, kv_heads, kv, dim))).to(dtype)
    cache = _new(batch, max_len or kv + 3, kv_heads, dim, dtype, bits)
    cache.sliced[0][0].append(k.cuda())
    cache.sliced[0][1].append(v.cuda())
    return cache, K.held(_np(k), bits, NAME[dtype]), K.held(_np(v), bits, NAME[dtype])


def _check(q, cache, k, v, mask, dtype, scale=None, force_generic=False, fix=False):
    from recurrent_drafting_amd import attention

    prepared = attention.prepare(torch.tensor(mask).cuda(), fix_empty_rows=fix, n_heads=q.shape[1])
    out = attention.masked_attention(q.cuda(), cache.sliced[0][0].rows(), cache.sliced[0][1].rows(), prepared, scale=scale,
                                     force_generic=force_generic)
    B, H, n, D = q.shape
    scale = scale or 1.0 / math.sqrt(D)
    if fix:
        mask = mask | ~mask.any(axis=2, keepdims=True)
    want, size = K.attention(_np(q), k, v, mask, scale)
    got = _np(out).reshape(B, n, H, D)
    nan = np.isnan(want)
    assert np.array_equal(np.isnan(got), nan)
    bound = _bound(_np(q), k, v, mask, scale, dtype, want, size)
    off = np.abs(np.where(nan, 0, got - want)) - np.where(nan, 0, bound)
    assert (off <= 0).all(), f"worst {off.max()} beyond its bound at {np.unravel_index(off.argmax(), off.shape)}"
    return out


SHAPES = [  # batch, heads, kv_heads, n_q, prev
    (1, 1, 1, 1, 0), (1, 4, 4, 1, 1), (2, 8, 2, 1, 31), (1, 8, 8, 1, 33), (2, 6, 1, 3, 64), (1, 16, 1, 1, 700), (3, 4, 2, 7, 45),
    (1, 2, 2, 16, 100), (1, 2, 2, 17, 100), (2, 7, 7, 33, 257), (1, 10, 2, 23, 500), (1, 2, 1, 129, 63), (2, 3, 3, 64, 1100)]


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("batch,heads,kv_heads,n,prev", SHAPES)
def test_attention_over_a_tree(batch, heads, kv_heads, n, prev, dim, dtype, bits):
    rng = np.random.default_rng(heads * 1000 + n + prev)
    cache, k, v = _filled(rng, batch, kv_heads, prev + n, dim, dtype, bits)
    q = torch.tensor(2 * rng.standard_normal((batch, heads, n, dim))).to(dtype)
    pads = [0] + [int(p) for p in rng.integers(0, prev // 2 + 1, batch - 1)]
    _check(q, cache, k, v, _tree_mask(rng, batch, n, prev, pads), dtype)


@pytest.mark.parametrize("dtype,dim,bits", [(torch.float32, 128, 4), (torch.float32, 64, 8), (torch.bfloat16, 96, 4),
                                            (torch.float16, 256, 8), (torch.bfloat16, 32, 8), (torch.float32, 160, 4)])
def test_attention_of_the_generic_kernel(dtype, dim, bits):
    rng = np.random.default_rng(dim)
    cache, k, v = _filled(rng, 2, 2, 301, dim, dtype, bits)
    q = torch.tensor(rng.standard_normal((2, 6, 5, dim))).to(dtype)
    mask = _tree_mask(rng, 2, 5, 296, [0, 37])
    mask[1, 2] = False
    _check(q, cache, k, v, mask, dtype)


def test_generic_and_mfma_kernels_on_one_shape():
    rng = np.random.default_rng(5)
    cache, k, v = _filled(rng, 2, 2, 200, 128, torch.bfloat16, 4)
    q = torch.tensor(rng.standard_normal((2, 8, 6, 128))).bfloat16()
    mask = _tree_mask(rng, 2, 6, 194, [0, 90])
    _check(q, cache, k, v, mask, torch.bfloat16)
    _check(q, cache, k, v, mask, torch.bfloat16, force_generic=True)


@pytest.mark.parametrize("bits", [4, 8])
def test_prompt_with_left_padding_and_empty_rows(bits):
    """A causal prompt: the padded queries attend to nothing (zeros) or, rewritten, to everything."""
    rng = np.random.default_rng(7)
    n = 150
    cache, k, v = _filled(rng, 2, 2, n, 128, torch.bfloat16, bits)
    q = torch.tensor(rng.standard_normal((2, 4, n, 128))).bfloat16()
    mask = np.broadcast_to(np.tril(np.ones((n, n), bool)), (2, n, n)).copy()
    mask[1, :, :70] = False
    out = _check(q, cache, k, v, mask, torch.bfloat16)
    assert not out[1, :70].any()
    _check(q, cache, k, v, mask, torch.bfloat16, fix=True)


@pytest.mark.parametrize("dtype,bits,dim", [(torch.bfloat16, 4, 128), (torch.float16, 8, 64)])
@pytest.mark.parametrize("scale", [1e-3, 1.0, 30.0])
def test_large_and_small_scores(dtype, bits, dim, scale):
    """Scores from nearly equal to far beyond what one exponential holds: the running maximum moves often."""
    rng = np.random.default_rng(11)
    cache, k, v = _filled(rng, 1, 2, 900, dim, dtype, bits)
    q = torch.tensor(rng.standard_normal((1, 4, 3, dim)) + 0.3).to(dtype)
    _check(q, cache, k, v, np.ones((1, 3, 900), bool), dtype, scale=scale)


def test_documents_and_scattered_masks():
    rng = np.random.default_rng(13)
    cache, k, v = _filled(rng, 2, 2, 400, 64, torch.bfloat16, 4)
    q = torch.tensor(rng.standard_normal((2, 4, 40, 64))).bfloat16()
    mask = rng.random((2, 40, 400)) < 0.1
    mask[0, :, 100:300] = False       # a hole longer than a unit
    mask[1, 7] = False
    mask[1, 9] = False
    mask[1, 9, 399] = True            # one key, the last
    _check(q, cache, k, v, mask, torch.bfloat16)


@pytest.mark.parametrize("force_generic", [False, True])
@pytest.mark.parametrize("dtype,bits,dim", [(torch.bfloat16, 4, 128), (torch.float16, 8, 64), (torch.bfloat16, 8, 128), (torch.float16, 4, 64)])
def test_nan_stays_with_the_rows_that_attend_to_it(dtype, bits, dim, force_generic):
    """NaN blocks in K and V: keys that nobody attends to, keys that some rows attend to, keys outside the
    spans, and cache rows filled with 0xFF around everything."""
    rng = np.random.default_rng(17)
    kv, n = 150, 6
    x = rng.standard_normal((2, 1, 2, kv, dim))
    x[1, 0, 0, 20, 9] = np.nan     # V: nobody
    x[0, 0, 1, 21, 3] = np.inf     # K: nobody
    x[1, 0, 0, 90, 17] = np.inf    # V: rows 0 and 3, one block of 8 dims
    x[1, 0, 1, 91, dim - 1] = np.nan
    x[0, 0, 1, 140, 5] = np.nan    # K: row 4
    mask = np.ones((1, n, kv), bool)
    mask[0, :, :10] = mask[0, :, 20:22] = mask[0, :, 148:] = False
    mask[0, [1, 2, 4, 5], 90] = False
    mask[0, [0, 1, 3, 4, 5], 91] = False
    mask[0, [0, 1, 2, 3, 5], 140] = False
    k, v = (torch.tensor(t).to(dtype) for t in x)
    cache = _new(1, kv + 40, 2, dim, dtype, bits)
    cache._cache.fill_(0xFF)
    cache.sliced[0][0].append(k.cuda())
    cache.sliced[0][1].append(v.cuda())
    cache._cache[:, :, :, :, :10] = 0xFF
    q = torch.tensor(rng.standard_normal((1, 4, n, dim))).to(dtype)
    out = _check(q, cache, K.held(_np(k), bits, NAME[dtype]), K.held(_np(v), bits, NAME[dtype]), mask, dtype, force_generic=force_generic)
    bad = torch.isnan(out[0].view(n, 4, dim)).any(dim=2).cpu()
    assert bad.tolist() == [[True, True, False, False], [False] * 4, [False, False, True, True], [True, True, False, False],
                            [False, False, True, True], [False] * 4]


def test_strides_of_queries():
    """q as heads of a token-major projection, as a contiguous (B, H, n, D) tensor, and as a slice that only
    the generic kernel can read (rows off the 16-byte grid)."""
    rng = np.random.default_rng(19)
    cache, k, v = _filled(rng, 2, 2, 90, 128, torch.bfloat16, 4)
    base = torch.tensor(rng.standard_normal((2, 4, 3, 128))).bfloat16()
    mask = _tree_mask(rng, 2, 3, 87, [0, 5])
    a = _check(base, cache, k, v, mask, torch.bfloat16)
    b = _check(base.transpose(1, 2).contiguous().transpose(1, 2), cache, k, v, mask, torch.bfloat16)
    assert torch.equal(a, b)
    from recurrent_drafting_amd import attention

    wide = torch.zeros(2, 4, 3, 131, dtype=torch.bfloat16, device="cuda")
    wide[..., 1:129] = base.cuda()
    prepared = attention.prepare(torch.tensor(mask).cuda(), n_heads=4)
    c = attention.masked_attention(wide[..., 1:129], cache.sliced[0][0].rows(), cache.sliced[0][1].rows(), prepared)
    assert (a.float() - c.float()).abs().max() <= 2 ** -6


def test_long_slabs_pass_32_bit_offsets():
    """Rows of the last batch row and head lie more than 4 GiB behind the cache's first."""
    from recurrent_drafting_amd import attention, kv_cache

    batch, heads, max_len, dim = 8, 16, 270000, 128
    cache = _new(batch, max_len, heads, dim, torch.bfloat16, 8)
    assert cache._cache[0, 0].numel() > 2 ** 32
    prev = max_len - 40
    g = torch.Generator().manual_seed(3)
    cache.set_length(prev)
    k, v, q = (torch.randn(batch, 40, heads * dim, generator=g).bfloat16() for _ in range(3))
    cos, sin = torch.ones(1, dim).bfloat16(), torch.zeros(1, dim).bfloat16()
    q_heads, keys, values = kv_cache.rope_append(q.cuda(), k.cuda(), v.cuda(), cos.cuda(), sin.cuda(),
                                                 torch.zeros(batch, 40, dtype=torch.long, device="cuda"), cache.sliced[0])
    mask = torch.zeros(batch, 1, max_len, dtype=torch.bool)
    mask[:, :, prev:] = True
    prepared = attention.prepare(mask.cuda(), n_heads=heads)
    out = attention.masked_attention(q_heads[:, :, :1], keys, values, prepared)
    hk = K.held(_np(k).reshape(batch, 40, heads, dim).transpose(0, 2, 1, 3), 8, "bf16")
    hv = K.held(_np(v).reshape(batch, 40, heads, dim).transpose(0, 2, 1, 3), 8, "bf16")
    assert np.array_equal(_np(cache.sliced[0][0].slice(prev)), hk) and np.array_equal(_np(cache.sliced[0][1].slice(prev)), hv)
    qq = _np(q).reshape(batch, 40, heads, dim).transpose(0, 2, 1, 3)[:, :, :1]
    ones = np.ones((batch, 1, 40), bool)
    want, size = K.attention(qq, hk, hv, ones, dim ** -0.5)
    bound = _bound(qq, hk, hv, ones, dim ** -0.5, torch.bfloat16, want, size)
    assert (np.abs(_np(out).reshape(batch, 1, heads, dim) - want) <= bound).all()


def test_one_long_row_is_cut_into_pieces():
    rng = np.random.default_rng(23)
    for dtype, bits, dim, group in [(torch.bfloat16, 4, 128, 4), (torch.float16, 8, 64, 1)]:
        kv = 20011
        cache, k, v = _filled(rng, 1, 2, kv, dim, dtype, bits)
        q = torch.tensor(2 * rng.standard_normal((1, 2 * group, 2, dim))).to(dtype)
        mask = np.ones((1, 2, kv), bool)
        mask[0, 0, :777] = False
        mask[0, 1, 12000:] = False
        _check(q, cache, k, v, mask, dtype)

# ---- launches large enough for the layouts with many rows ---------------------------------------------

def _repeated(q, k, v, batch, copies, dtype, bits):
    """The two sequences and two kv heads of q, k and v over `batch` rows and 2 * copies kv heads, in a cache
    whose other rows are filled with 0xFF."""
    rep = lambda x: x[torch.arange(batch) % 2].repeat(1, copies, 1, 1).cuda()
    cache = _new(batch, k.shape[2] + 3, 2 * copies, k.shape[3], dtype, bits)
    cache._cache.fill_(0xFF)
    for view, x in zip(cache.sliced[0], (k, v)):
        view.append(rep(x))
    return rep(q), cache


LARGE = [  # batch, kv heads, group, n_q, prev, mask
    (8, 24, 1, 230, 300, "tree"), (13, 16, 2, 121, 133, "tree"), (10, 8, 4, 225, 0, "causal"), (8, 32, 1, 115, 150, "tree"),
    (16, 20, 1, 250, 20, "causal"), (9, 64, 1, 255, 260, "scattered"),
    (8, 32, 1, 250, 260, "tree"), (12, 16, 2, 225, 0, "causal")]


@pytest.mark.parametrize("dtype,bits,dim", [(torch.bfloat16, 4, 128), (torch.float16, 8, 64), (torch.bfloat16, 8, 128), (torch.float16, 4, 64)])
@pytest.mark.parametrize("batch,kv_heads,group,n,prev,kind", LARGE)
@pytest.mark.parametrize("poisoned", [False, True])
def test_large_launches(batch, kv_heads, group, n, prev, kind, dtype, bits, dim, poisoned):
    """Two sequences and two kv heads against the oracle, and every copy of them over the batch and the heads
    with the same bits.  Poisoned: NaN blocks that some rows attend to and that nobody attends to."""
    from recurrent_drafting_amd import attention

    rng = np.random.default_rng(1000 * n + batch)
    kv = prev + n
    x = rng.standard_normal((2, 2, 2, kv, dim))
    pads = [0, kv // 5]
    if kind == "tree":
        mask = _tree_mask(rng, 2, n, prev, pads)
    else:
        mask = np.broadcast_to(np.tril(np.ones((n, kv), bool), prev), (2, n, kv)).copy()
        mask[1, :, : pads[1]] = False  # (of a prompt's second sequence the first rows attend to nothing)
        if kind == "scattered":
            mask &= rng.random(mask.shape) < 0.2
    if poisoned:
        x[1, 0, 0, 40, 9], x[1, 1, 1, kv - 2, dim - 1], x[0, 1, 0, kv // 2, 5] = np.nan, np.inf, np.nan
        mask[0, :, 40] = False                        # V: nobody
        mask[1, : n - 3, kv - 2] = False              # V: some of the last rows
        mask[1, n // 2 :, kv // 2] = False            # K: some of the first rows
    k, v = (torch.tensor(t).to(dtype) for t in x)
    q = torch.tensor(2 * rng.standard_normal((2, 2 * group, n, dim))).to(dtype)
    big_q, cache = _repeated(q, k, v, batch, kv_heads // 2, dtype, bits)
    prepared = attention.prepare(torch.tensor(mask[np.arange(batch) % 2]).cuda(), fix_empty_rows=False, n_heads=kv_heads * group)
    out = attention.masked_attention(big_q, cache.sliced[0][0].rows(), cache.sliced[0][1].rows(), prepared)
    out = out.view(batch, n, kv_heads // 2, 2 * group, dim)
    same = out[torch.arange(batch) % 2, :, :1].expand_as(out)
    assert torch.equal(out.nan_to_num(123.0), same.nan_to_num(123.0))
    hk, hv = K.held(_np(k), bits, NAME[dtype]), K.held(_np(v), bits, NAME[dtype])
    want, size = K.attention(_np(q), hk, hv, mask, dim ** -0.5)
    got = _np(out[:2, :, 0]).reshape(2, n, 2 * group, dim)
    nan = np.isnan(want)
    assert np.array_equal(np.isnan(got), nan) and nan.any() == poisoned
    bound = _bound(_np(q), hk, hv, mask, dim ** -0.5, dtype, want, size)
    assert (np.abs(np.where(nan, 0, got - want)) <= np.where(nan, 0, bound)).all()


@pytest.mark.parametrize("dtype,bits,dim", [(torch.bfloat16, 4, 128), (torch.float16, 8, 64)])
def test_large_packed_and_shifted_launches(dtype, bits, dim):
    """Packed rows of different counts with cache rows in place: the same bits as every sequence by itself at
    its full length and unshifted, and rows behind the last one as they were."""
    from recurrent_drafting_amd import attention, kv_cache
    from recurrent_drafting_amd.packed_rows import PackedRows

    rng = np.random.default_rng(53)
    batch, heads, n, prev = 8, 32, 240, 250
    counts = [240, 1, 33, 128, 129, 240, 31, 200]
    rows = PackedRows.from_counts(torch.tensor(counts, dtype=torch.int32).cuda(), sum(counts), n)
    k, v = (torch.tensor(rng.standard_normal((batch, heads, prev + n, dim))).to(dtype) for _ in range(2))
    q = torch.tensor(rng.standard_normal((batch, heads, n, dim))).to(dtype).cuda()
    pads = [0, 100, 40, 0, 64, 7, 200, 33]
    mask = torch.tensor(_tree_mask(rng, batch, n, prev, pads)).cuda()
    plain = _new(batch, prev + n, heads, dim, dtype, bits)
    for view, x in zip(plain.sliced[0], (k, v)):
        view.append(x.cuda())
    want = attention.masked_attention(q, plain.sliced[0][0].rows(), plain.sliced[0][1].rows(),
                                      attention.prepare(mask, n_heads=heads)).view(batch, n, heads, dim)
    # cache row = column - shift
    shift = torch.tensor([0, 100, 37, -1, 64, 7, 31, -2], dtype=torch.int32)
    moved = _new(batch, prev + n + 2, heads, dim, dtype, bits)
    moved._cache.fill_(0xFF)
    for b in range(batch):
        s = int(shift[b])
        lo = max(s, 0)
        moved._cache[0, :, b, :, lo - s : prev + n - s] = plain._cache[0, :, b, :, lo:]
    moved.set_length(prev + n)
    moved.rows_in_place = True
    moved.shift.copy_(shift)
    prepared = attention.prepare(mask, n_heads=heads, kv_shift=moved.shift)
    packed = torch.cat([q[b, :, :c] for b, c in enumerate(counts)], dim=1).transpose(0, 1)
    packed = torch.cat((packed, packed.new_full((rows.rows - sum(counts), heads, dim), float("nan"))))
    key, value = (kv_cache.QuantizedRows(moved, 0, side, 0, prev + n) for side in (0, 1))
    got = attention.masked_attention(packed, key, value, prepared, rows=rows).view(rows.rows, heads, dim)
    at = 0
    for b, c in enumerate(counts):
        assert torch.equal(got[at : at + c], want[b, :c]), b
        at += c


# ---- packed rows, rows in place, moves ------------------------------------------------------------------

@pytest.mark.parametrize("dtype,bits,dim", [(torch.bfloat16, 4, 128), (torch.float16, 8, 64), (torch.float32, 4, 32)])
def test_packed_rows_and_shifted_rows(dtype, bits, dim):
    """The decode loop's two layouts together: only the slots that exist, cache rows kept in place.  The
    same records, rotated queries and outputs as the padded call on an unshifted cache; rows behind the
    last token stay as they were."""
    from recurrent_drafting_amd import attention, kv_cache
    from recurrent_drafting_amd.packed_rows import PackedRows

    rng = np.random.default_rng(29)
    batch, heads, kv_heads, n, prev = 3, 4, 2, 11, 60
    counts = torch.tensor([11, 1, 6], dtype=torch.int32)
    rows = PackedRows.from_counts(counts.cuda(), int(counts.sum()), n)
    x = torch.tensor(rng.standard_normal((batch, n, (heads + 2 * kv_heads) * dim))).to(dtype)
    old = torch.tensor(rng.standard_normal((2, batch, kv_heads, prev, dim))).to(dtype)
    cos, sin = _tables(dim, prev + n, dtype)
    position_ids = torch.tensor(rng.integers(0, prev + n, (batch, n)))
    shift = torch.tensor([0, 4, -3], dtype=torch.int32)
    pads = [0, 7, 2]
    mask = _tree_mask(rng, batch, n, prev, pads)
    split = lambda t: (t[..., : heads * dim], t[..., heads * dim : (heads + kv_heads) * dim], t[..., (heads + kv_heads) * dim :])

    plain = _new(batch, prev + n, kv_heads, dim, dtype, bits)
    for side in (0, 1):
        plain.sliced[0][side].append(old[side].cuda())
    q0, k0, v0 = kv_cache.rope_append(*split(x.cuda()), cos.cuda(), sin.cuda(), position_ids.cuda(), plain.sliced[0])
    want = attention.masked_attention(q0, k0, v0, attention.prepare(torch.tensor(mask).cuda(), n_heads=heads))

    cache = _new(batch, prev + n + 4, kv_heads, dim, dtype, bits)
    cache._cache.fill_(0xFF)
    for b in range(batch):  # column c in cache row c - shift
        s = int(shift[b])
        lo = max(0, s)
        cache._cache[0, :, b, :, lo - s : prev - s] = plain._cache[0, :, b, :, lo:prev]
    cache.set_length(prev)
    cache.rows_in_place = True
    cache.shift.copy_(shift)
    cache._shifted = True
    packed = rows.take(x.cuda())
    before = cache._cache.clone()
    q1, k1, v1 = kv_cache.rope_append(*split(packed), cos.cuda(), sin.cuda(), position_ids.cuda(), cache.sliced[0], rows)
    prepared = attention.prepare(torch.tensor(mask).cuda(), n_heads=heads, kv_shift=cache.shift)
    got = attention.masked_attention(q1, k1, v1, prepared, rows=rows)
    r = 0
    for b in range(batch):
        s, c = int(shift[b]), int(counts[b])
        new = cache._cache[0, :, b, :, prev - s : prev - s + c]
        used = dim * bits // 8 + dim // 8  # (the padding of a record is never written)
        assert torch.equal(new[..., :used], plain._cache[0, :, b, :, prev : prev + c, :used])
        changed = (cache._cache[0, :, b] != before[0, :, b]).any(dim=3).any(dim=0).any(dim=0).nonzero().flatten().tolist()
        assert set(changed) <= set(range(prev - s, prev - s + c))
        assert torch.equal(q1[r : r + c], q0[b, :, :c].transpose(0, 1))
        assert torch.equal(got[r : r + c], want[b, :c])
        r += c
    # the rows back in their columns, read in the model's type
    cache.rows_in_place = False
    for side in (0, 1):
        a, e = cache.sliced[0][side].slice(0), plain.sliced[0][side].slice(0)
        for b in range(batch):
            c = prev + int(counts[b])
            assert torch.equal(a[b, :, pads[b] : c], e[b, :, pads[b] : c])


@pytest.mark.parametrize("bits", [4, 8])
def test_unpack_and_realign_move_records(bits):
    """Cache.unpack and the re-alignment on records: the same rows as on the values."""
    rng = np.random.default_rng(31)
    batch, heads, dim, prev, width, length, n = 2, 2, 128, 9, 3, 4, 7
    cache, k, v = _filled(rng, batch, heads, prev + n, dim, torch.bfloat16, bits, max_len=prev + width * length + 2)
    index = torch.tensor(rng.integers(0, n, (batch, width, length)))
    cache.unpack(prev, index.cuda())
    for side, x in enumerate((k, v)):
        got = _np(cache.sliced[0][side].slice(0))
        assert np.array_equal(got[:, :, :prev], x[:, :, :prev])
        for b in range(batch):
            assert np.array_equal(got[b, :, prev:], x[b][:, prev + index[b].flatten().numpy()])


# ---- together ------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype,dim,bits", [(torch.bfloat16, 128, 4), (torch.float16, 64, 8), (torch.bfloat16, 128, 8), (torch.float32, 32, 4)])
def test_prompt_tree_and_tokens_of_one_sequence(dtype, dim, bits):
    """A layer's calls over a generation: a prompt, a packed tree, single tokens; each attends over all rows
    written so far.  Every output against the oracle on the oracle's own cache."""
    from recurrent_drafting_amd import attention

    rng = np.random.default_rng(37)
    batch, heads, kv_heads = 2, 4, 2
    steps = [(70, "causal"), (13, "tree"), (1, "tree"), (1, "tree"), (45, "tree")]
    total = sum(n for n, _ in steps)
    cache = _new(batch, total, kv_heads, dim, dtype, bits, layers=2)
    cos, sin = _tables(dim, total, dtype)
    held = [np.zeros((batch, kv_heads, 0, dim))] * 2
    prev, pads = 0, [0, 12]
    for n, kind in steps:
        x = torch.tensor(rng.standard_normal((batch, n, (heads + 2 * kv_heads) * dim))).to(dtype)
        position_ids = torch.tensor(np.maximum(prev + np.arange(n) - np.array(pads)[:, None], 0))
        if kind == "causal":
            mask = np.broadcast_to(np.tril(np.ones((n, n), bool)), (batch, n, n)).copy()
            mask[1, :, : pads[1]] = False
        else:
            mask = _tree_mask(rng, batch, n, prev, pads)
        d = x.cuda()
        prepared = attention.prepare(torch.tensor(mask).cuda(), fix_empty_rows=True, n_heads=heads)
        out = attention.rope_attention(d[..., : heads * dim], d[..., heads * dim : (heads + kv_heads) * dim],
                                       d[..., (heads + kv_heads) * dim :], cos.cuda(), sin.cuda(), position_ids.cuda(),
                                       cache.sliced[1], prepared)
        y = _np(x).reshape(batch, n, -1, dim).transpose(0, 2, 1, 3)
        c, s = _np(cos)[position_ids.numpy()][:, None], _np(sin)[position_ids.numpy()][:, None]
        held = [np.concatenate((held[0], K.held(K.rotate(y[:, heads : heads + kv_heads], c, s), bits, NAME[dtype])), axis=2),
                np.concatenate((held[1], K.held(y[:, heads + kv_heads :], bits, NAME[dtype])), axis=2)]
        q = K.rotate(y[:, :heads], c, s)
        q_held = torch.tensor(q).to(torch.float32).to(dtype)  # (the rotated queries are rounded to the type)
        full = mask | ~mask.any(axis=2, keepdims=True)
        want, size = K.attention(_np(q_held), *held, full, dim ** -0.5)
        bound = _bound(_np(q_held), *held, full, dim ** -0.5, dtype, want, size)
        # a query component that fp32 rounds to the other neighbour moves a score by u |q k| scale at most
        u = torch.finfo(dtype).eps / 2
        kk = np.repeat(np.abs(held[0]), heads // kv_heads, axis=1)
        flip = 2 * u * dim ** -0.5 * np.abs(_np(q_held)).max() * kk.max()
        assert (np.abs(_np(out).reshape(batch, n, heads, dim) - want) <= bound + 2 * flip * size).all()
        prev += n
    assert not cache._cache[0].any()
    for side in (0, 1):
        assert np.array_equal(_np(cache.sliced[1][side].slice(0)), held[side])


def test_side_stream_graphs_and_shared_masks():
    """One prepared mask used on two streams and in two captured graphs whose replays alternate with eager
    work: every replay gives the eager result."""
    from recurrent_drafting_amd import attention, kv_cache

    rng = np.random.default_rng(41)
    kv = 6000  # long enough that the keys are cut into pieces (a workspace per call)
    cache, _, _ = _filled(rng, 1, 2, kv, 128, torch.bfloat16, 4)
    key, value = cache.sliced[0]
    prepared = attention.prepare(torch.ones(1, 2, kv, dtype=torch.bool, device="cuda"), n_heads=8)
    qs = [torch.randn(1, 8, 2, 128, device="cuda").bfloat16() for _ in range(4)]
    want = [attention.masked_attention(q, key.rows(), value.rows(), prepared).clone() for q in qs]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = attention.masked_attention(qs[0], key.rows(), value.rows(), prepared)
    side.synchronize()
    assert torch.equal(got, want[0])

    graphs, ins, outs = [], [], []
    x = torch.randn(1, 2, 12 * 128, device="cuda").bfloat16()
    cos, sin = _tables(128, 8, torch.bfloat16)
    cos, sin, pos = cos.cuda(), sin.cuda(), torch.zeros(1, 2, dtype=torch.long, device="cuda")
    for i in (0, 1):
        q = qs[i].clone()
        graph = torch.cuda.CUDAGraph()
        small = _new(1, 2, 2, 128, torch.bfloat16, 4)
        with torch.cuda.graph(graph):
            out = attention.masked_attention(q, key.rows(), value.rows(), prepared)
            kv_cache.rope_append(x[..., :1024], x[..., 1024:1280], x[..., 1280:], cos, sin, pos, small.sliced[0])
            back = small.sliced[0][1].slice(0)
        graphs.append(graph), ins.append(q), outs.append((out, back))
    v_held = torch.tensor(K.held(_np(x[..., 1280:]).reshape(1, 2, 2, 128).transpose(0, 2, 1, 3), 4, "bf16")).bfloat16()
    for turn in range(3):
        for i in (0, 1):
            j = (i + turn) % 4
            ins[i].copy_(qs[j])
            outs[i][0].zero_()
            graphs[i].replay()
            eager = attention.masked_attention(qs[j], key.rows(), value.rows(), prepared)
            torch.cuda.synchronize()
            assert torch.equal(outs[i][0], want[j]) and torch.equal(eager, want[j])
            assert torch.equal(outs[i][1].cpu(), v_held)
    # both at once on two streams
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for i in (0, 1):
        ins[i].copy_(qs[2 + i])
    torch.cuda.synchronize()
    for _ in range(5):
        for i in (0, 1):
            with torch.cuda.stream(streams[i]):
                graphs[i].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0][0], want[2]) and torch.equal(outs[1][0], want[3])


def test_a_captured_forward_follows_its_mask():
    """The mask is prepared inside the capture: its span table is written once for the layers of the capture,
    again by every replay, and is not what an eager call on the same stream reads afterwards."""
    from recurrent_drafting_amd import attention

    rng = np.random.default_rng(59)
    kv, n = 300, 20
    cache = _new(2, kv, 2, 64, torch.float16, 8, layers=3)
    for views in cache.sliced:
        for view in views:
            view.append(torch.tensor(rng.standard_normal((2, 2, kv, 64))).half().cuda())
    q = torch.randn(2, 4, n, 64, device="cuda").half()
    masks = [torch.tensor(_tree_mask(rng, 2, n, kv - n, pads)).cuda() for pads in ([0, 90], [200, 0], [33, 250])]

    def forward(mask):
        prepared = attention.prepare(mask, n_heads=4)
        return prepared, [attention.masked_attention(q, k.rows(), v.rows(), prepared) for k, v in cache.sliced]

    want = [[o.clone() for o in forward(m)[1]] for m in masks]
    static, stream = masks[0].clone(), torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        prepared, outs = forward(static)
    assert len(prepared.spans) == 1 and all(isinstance(key, tuple) for key in prepared.spans)
    for turn in (1, 2, 0, 1):
        static.copy_(masks[turn])
        graph.replay()
        eager = forward(masks[2])[1]
        torch.cuda.synchronize()
        for i in range(3):
            assert torch.equal(outs[i], want[turn][i]) and torch.equal(eager[i], want[2][i])
    with torch.cuda.stream(stream):
        again = attention.masked_attention(q, cache.sliced[1][0].rows(), cache.sliced[1][1].rows(), prepared)
    stream.synchronize()
    assert torch.equal(again, want[1][1]) and len(prepared.spans) == 2


def test_same_call_twice_gives_the_same_bits():
    from recurrent_drafting_amd import attention

    rng = np.random.default_rng(43)
    cache, _, _ = _filled(rng, 2, 2, 5000, 128, torch.float16, 8)
    q = torch.randn(2, 8, 3, 128, device="cuda").half()
    prepared = attention.prepare(torch.ones(2, 3, 5000, dtype=torch.bool, device="cuda"), n_heads=8)
    first = attention.masked_attention(q, cache.sliced[0][0].rows(), cache.sliced[0][1].rows(), prepared)
    for _ in range(3):
        assert torch.equal(first, attention.masked_attention(q, cache.sliced[0][0].rows(), cache.sliced[0][1].rows(), prepared))


def test_refusals_with_tensors():
    from recurrent_drafting_amd import attention, kv_cache

    rng = np.random.default_rng(47)
    cache, _, _ = _filled(rng, 1, 2, 20, 64, torch.bfloat16, 4)
    other, _, _ = _filled(rng, 1, 2, 20, 64, torch.bfloat16, 8)
    key, value = cache.sliced[0]
    prepared = attention.prepare(torch.ones(1, 1, 20, dtype=torch.bool, device="cuda"), n_heads=4)
    q = torch.zeros(1, 4, 1, 64, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(AssertionError):
        attention.masked_attention(q, key.rows(), other.sliced[0][1].rows(), prepared)
    with pytest.raises(AssertionError):
        attention.masked_attention(q, key.rows(), value.slice(0), prepared)
    with pytest.raises(AssertionError):
        attention.masked_attention(q.half(), key.rows(), value.rows(), prepared)
    with pytest.raises(AssertionError):
        attention.masked_attention(q, key.rows(1), value.rows(1), prepared)
    shifted = attention.prepare(torch.ones(1, 1, 19, dtype=torch.bool, device="cuda"), n_heads=4,
                                kv_shift=torch.zeros(1, dtype=torch.int32, device="cuda"))
    with pytest.raises(AssertionError, match="first row"):  # a shift could point in front of the slice
        attention.masked_attention(q, key.rows(1), value.rows(1), shifted)
    with pytest.raises(RuntimeError, match="scale"):
        attention.masked_attention(q, key.rows(), value.rows(), prepared, scale=-0.5)
    x = torch.zeros(1, 1, 4 * 64, dtype=torch.bfloat16, device="cuda")
    cos, sin = torch.ones(1, 64, dtype=torch.bfloat16, device="cuda"), torch.zeros(1, 64, dtype=torch.bfloat16, device="cuda")
    pos = torch.zeros(1, 1, dtype=torch.long, device="cuda")
    with pytest.raises(RuntimeError, match="GPU|cuda"):
        kv_cache.rope_append(x, x[..., :128], x[..., :128].cpu(), cos, sin, pos, cache.sliced[0])
    with pytest.raises(AssertionError):  # another type than the cache was made for
        kv_cache.rope_append(x.half(), x[..., :128].half(), x[..., :128].half(), cos.half(), sin.half(), pos, cache.sliced[0])
    assert key.length == 20


@pytest.mark.parametrize("bits", [4, 8])
def test_generate_with_the_cache_in_few_bits(bits, monkeypatch):
    """`RecurrentDrafting.kv_bits`: rows kept in place and rows moved every step decode the same tokens (the
    records move as they are), and the cache is the one asked for."""
    import recurrent_drafting_amd as rd

    llama_sd, drafter_sd = tm.markov(3)  # a model whose drafts are accepted: rows shift both ways
    ids = tm.prompt(3, 9, tm.LLAMA["vocab_size"], 3, [0, 4, 1])
    streams, set_length = [], rd.kv_cache.Cache.set_length
    for in_place in (True, False):
        llm = rd.modeling_llama.LlamaForCausalLM(LlamaConfig(**tm.LLAMA))
        drafter = rd.modeling_drafter.Drafter(rd.configuration_drafter.DrafterConfig(**tm.DRAFTER))
        llm.load_state_dict(llama_sd, strict=False)
        drafter.load_state_dict(drafter_sd)
        model = rd.RecurrentDrafting(llm.float().cuda().eval(), drafter.float().cuda().eval())
        model.kv_bits, model.kv_rows_in_place = bits, in_place
        made = []
        monkeypatch.setattr(rd.kv_cache.Cache, "set_length",
                            lambda self, length: (made.append(self), set_length(self, length)))
        streams.append([t.cpu().tolist() for t in model.generate(
            rd.stats.Ledger(), ids.cuda(), 40, rd.BeamShape(6, 4), rd.SamplingArgs(1.0, True), rd.SpecialTokens(0, None))])
        assert made and {c.bits for c in made} == {bits} and made[0]._cache.dtype == torch.uint8
    assert streams[0] == streams[1] and len(streams[0]) > 3
