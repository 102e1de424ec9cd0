"""Attention over a cache in 4 or 8 bits with scores so large that fp32 rounds a score by more than a weight has room
for: the weights depend on the differences of scores alone.

The products q . k are exact in fp32 here (multiples of one power of two within 24 bits of it).  Tolerance: the
output's rounding u |o|, the weights' (u, fp16 below 2^-21 of the largest 2^-32 of it) and the accumulation's as in
test_gpu_kv_quant.py; a difference of scores of at most 2^5 in log2 units is off by 2^5 2^-22 (the scale in log2 units and
the product, rounded once each), the exponential by 2^-21: 2 d = 2 ln 2 2^-17 + 2^-20 <= 2^-16.
"""
import numpy as np
import pytest
import torch

from oracle import kv_quant_oracle as K
from test_gpu_kv_quant import NAME, _new, _np, _repeated

pytestmark = pytest.mark.gpu

# queries, keys, copies of the sequence and its kv heads: one row, a long one cut into pieces, two row blocks, eight waves
LAYOUTS = [(1, 200, 1), (1, 20000, 1), (40, 300, 1), (250, 510, 32)]


def _run(q, k, v, n, copies, dtype, bits):
    """(outputs (n, D) of the first head, the values the cache holds)"""
    from recurrent_drafting_amd import attention

    kv, dim = k.shape
    q = q.to(dtype).view(1, 1, 1, dim).expand(1, 2, n, dim).contiguous()
    k, v = (x.to(dtype).view(1, 1, kv, dim).expand(1, 2, kv, dim).contiguous() for x in (k, v))
    assert torch.equal(torch.tensor(K.held(_np(k), bits, NAME[dtype])), k.double())
    if copies > 1:
        big, cache = _repeated(q.expand(2, -1, -1, -1), k.expand(2, -1, -1, -1), v.expand(2, -1, -1, -1), 8, copies // 2, dtype, bits)
    else:
        big, cache = q.cuda(), _new(1, kv + 1, 2, dim, dtype, bits)
        for view, x in zip(cache.sliced[0], (k, v)):
            view.append(x.cuda())
    prepared = attention.prepare(torch.ones(big.shape[0], n, kv, dtype=torch.bool, device="cuda"), n_heads=big.shape[1])
    out = attention.masked_attention(big, cache.sliced[0][0].rows(), cache.sliced[0][1].rows(), prepared)
    return _np(out).reshape(big.shape[0], n, big.shape[1], dim)[0, :, 0], K.held(_np(v[0, 0]), bits, NAME[dtype])


def _check(out, values, weights, dtype):
    p = weights / weights.sum()
    want, size = p @ values, p @ np.abs(values)
    u, kv = torch.finfo(dtype).eps / 2, len(values)
    lost = kv * 2.0 ** -31 * np.abs(values).max() / weights.sum() if dtype == torch.float16 else 0.0
    bound = 2 * u * np.abs(want) + (u + 2.0 ** -16 + (kv + out.shape[1]) * 2.0 ** -24) * size + lost + 2.0 ** -25
    off = np.abs(out - want) - bound
    assert np.isfinite(out).all() and (off <= 0).all(), f"beyond the bound by {off.max()}"


CASES = [(torch.bfloat16, 4, 128), (torch.float16, 8, 64), (torch.bfloat16, 8, 64), (torch.float16, 4, 128)]


@pytest.mark.parametrize("n,kv,copies", LAYOUTS)
@pytest.mark.parametrize("dtype,bits,dim", CASES)
@pytest.mark.parametrize("sign", [1, -1])
def test_equal_scores_of_any_size(n, kv, copies, dtype, bits, dim, sign):
    """Every key the same: the mean of the values."""
    g = torch.Generator().manual_seed(kv)
    v = torch.randn(kv, dim, generator=g)
    for power in (0, 8, 11, 13, 15) + ((30, 55) if dtype == torch.bfloat16 else ()):
        q = torch.full((dim,), sign * 1.25 * 2.0 ** power)
        k = torch.full((kv, dim), 1.5 * 2.0 ** power)
        out, values = _run(q, k, v, n, copies, dtype, bits)
        _check(out, values, np.ones(kv), dtype)


@pytest.mark.parametrize("n,kv,copies", LAYOUTS)
@pytest.mark.parametrize("dtype,bits,dim", CASES)
def test_neighbouring_scores_far_from_zero(n, kv, copies, dtype, bits, dim):
    """Scores of about 2^23 to 2^25 that differ by a few units; every 32 keys hold all of them."""
    g = torch.Generator().manual_seed(kv)
    v = torch.randn(kv, dim, generator=g)
    step = torch.arange(kv) % 3
    for sign in (1, -1):
        for power in (10, 11):
            q = torch.full((dim,), 1024.0)
            k = torch.full((kv, dim), sign * 2.0 ** power)
            k[:, 8:16] = 0.0                       # a block with a scale of its own
            k[:, 9] = step * 2.0 ** (power - 15)
            out, values = _run(q, k, v, n, copies, dtype, bits)
            apart = (step - 2).double().numpy() * 1024.0 * 2.0 ** (power - 15) * dim ** -0.5
            _check(out, values, np.exp(apart), dtype)


@pytest.mark.parametrize("n,kv,copies", LAYOUTS)
@pytest.mark.parametrize("dtype,bits,dim", CASES)
@pytest.mark.parametrize("rising", [True, False])
def test_scores_far_apart(n, kv, copies, dtype, bits, dim, rising):
    """The keys of the largest score take all of the weight, whether they come first or last."""
    g = torch.Generator().manual_seed(kv)
    v = torch.randn(kv, dim, generator=g)
    order = torch.arange(kv) * 5 // kv             # 0 .. 4
    if not rising:
        order = 4 - order
    for power in (4, 11):
        q = torch.full((dim,), 1.25 * 2.0 ** power)
        k = ((order - 2) * 2.0 ** power).view(kv, 1).expand(kv, dim)
        out, values = _run(q, k.contiguous(), v, n, copies, dtype, bits)
        _check(out, values, (order == 4).double().numpy(), dtype)
