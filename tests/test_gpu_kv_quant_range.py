"""Weights of the attention over a cache in 4 or 8 bits at both ends of fp16's range.

The kernel holds fp16 weights 2^7 times as large as bf16's: the running maximum's is 2^7, the largest 2^15.  The bound is
that of test_gpu_kv_quant.py with its fp16 term tightened by this factor: weights below 2^-14 are rounded to multiples
of 2^-24, off by 2^-25 at most, which is 2^-32 / S of a sum that is 2^7 S at least, S the sum relative to its largest weight;
numerator and denominator are both off by it, n 2^-32 (max |v| + |o|) / S <= n 2^-31 max |v| / S.
"""
import numpy as np
import pytest
import torch

from oracle import kv_quant_oracle as K
from test_gpu_kv_quant import NAME, _new, _np, _repeated

pytestmark = pytest.mark.gpu


def _bound(q, k, v, mask, scale, dtype, out, size):
    u = torch.finfo(dtype).eps / 2
    D = q.shape[-1]
    kk = np.repeat(np.abs(k), q.shape[1] // k.shape[1], axis=1)
    dots = np.einsum("bhnd,bhkd->bnhk", np.abs(q), kk).max(axis=3) * scale
    d = (D * 2.0 ** -23 * dots + dots * 2.0 ** -22 + 2.0 ** -21)[..., None]
    n = mask.sum(axis=2)[:, :, None, None]
    scores = np.einsum("bhnd,bhkd->bnhk", q, np.repeat(k, q.shape[1] // k.shape[1], axis=1)) * scale
    scores = np.where(mask[:, :, None], scores, -np.inf)
    total = np.exp(scores - scores.max(axis=3, keepdims=True)).sum(axis=3)[..., None]
    lost = n * np.abs(v).max() / total * (2.0 ** -31 if dtype == torch.float16 else 2.0 ** -125)
    return 2 * u * np.abs(out) + (u + 2 * d + (n + D) * 2.0 ** -24) * size + lost + 2.0 ** -25


def _rows(keys, heads, dim, dtype, values):
    """k and v (1, heads, kv, dim): dim 0 of the keys, all dims of the values."""
    kv = len(keys)
    k = torch.zeros(1, heads, kv, dim)
    k[..., 0] = torch.tensor(keys)
    v = torch.tensor(values).float().view(1, 1, kv, 1).expand(1, heads, kv, dim)
    return k.to(dtype), v.to(dtype)


def _launch(gain, k, v, heads, n, copies, dtype, bits):
    """Queries of `gain` in dim 0, the cache that holds k and v (or `copies` / 2 copies of them for 8 rows)."""
    dim, kv = k.shape[3], k.shape[2]
    q = torch.zeros(1, heads, n, dim, dtype=dtype)
    q[..., 0] = gain
    if copies > 1:
        return _repeated(q.expand(2, -1, -1, -1), k.expand(2, -1, -1, -1), v.expand(2, -1, -1, -1), 8, copies // 2, dtype, bits)
    cache = _new(1, kv + 1, k.shape[1], dim, dtype, bits)
    for view, x in zip(cache.sliced[0], (k, v)):
        view.append(x.cuda())
    return q, cache


def _compare(q, k, v, cache, mask, bits, dtype):
    """Scores are q . k: the scale is 1."""
    from recurrent_drafting_amd import attention

    prepared = attention.prepare(torch.tensor(mask).cuda(), fix_empty_rows=False, n_heads=q.shape[1])
    out = attention.masked_attention(q.cuda(), cache.sliced[0][0].rows(), cache.sliced[0][1].rows(), prepared, scale=1.0)
    out = _np(out).reshape(q.shape[0], q.shape[2], q.shape[1], q.shape[3])[:1]
    heads = k.shape[1] * (q.shape[1] // cache.sliced[0][0].shape[1])
    hk, hv = K.held(_np(k), bits, NAME[dtype]), K.held(_np(v), bits, NAME[dtype])
    some = _np(q[:1, :heads])
    want, size = K.attention(some, hk, hv, mask[:1], 1.0)
    bound = _bound(some, hk, hv, mask[:1], 1.0, dtype, want, size)
    off = np.abs(out[:, :, :heads] - want)
    assert (off <= bound).all(), f"off by {off.max()}, bound {bound[off > bound].min()}"
    return want, bound


# queries and keys: one row, two row blocks of a wave, a tile of eight waves (over copies of a sequence)
LAYOUTS = [(1, 900, 1), (1, 40001, 1), (40, 900, 1), (250, 510, 32)]


@pytest.mark.parametrize("n,kv,copies", LAYOUTS)
@pytest.mark.parametrize("dtype,bits,dim", [(torch.float16, 4, 128), (torch.float16, 8, 64), (torch.float16, 8, 128), (torch.float16, 4, 64), (torch.bfloat16, 8, 128)])
def test_one_large_weight_and_a_long_flat_tail(n, kv, copies, dtype, bits, dim):
    """Keys of value 0 (one for every wave where keys are not cut) with nearly all of the weight, every other with 2^-27.4 or 2^-30.8 of it and the value 6144:
    the result is the tail's share."""
    keys = np.where(np.arange(kv) % 3 == 0, -2.0, 0.0)
    large = 7 + 32 * np.arange(8 if kv == 900 else 1)
    keys[large] = 16.0
    values = np.full(kv, 6144.0)
    values[large] = 0.0
    k, v = _rows(keys, 2, dim, dtype, values)
    q, cache = _launch(1.1875, k, v, 4 if n == 1 else 2, n, copies, dtype, bits)
    want, bound = _compare(q, k, v, cache, np.ones((q.shape[0], n, kv), bool), bits, dtype)
    assert (np.abs(want) > 4 * bound).all()  # (a lost tail would be seen)


@pytest.mark.parametrize("n,kv,copies", LAYOUTS)
@pytest.mark.parametrize("dtype,bits,dim", [(torch.float16, 4, 128), (torch.float16, 8, 64)])
def test_scores_that_rise_just_below_the_limit_of_the_running_maximum(n, kv, copies, dtype, bits, dim):
    """The first keys set the maximum, later ones lie 2^7.93 and 2^5.95 above it, with values up to the type's largest."""
    keys = np.where(np.arange(kv) < kv // 8, 0.0, 4.0 - np.arange(kv) % 2)
    values = np.where(np.arange(kv) % 5 == 0, -40000.0, 65504.0)
    k, v = _rows(keys, 2, dim, dtype, values)
    q, cache = _launch(1.375, k, v, 2, n, copies, dtype, bits)
    _compare(q, k, v, cache, np.ones((q.shape[0], n, kv), bool), bits, dtype)
