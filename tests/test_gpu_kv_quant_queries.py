"""Queries of the attention over a cache in 4 or 8 bits in layouts other than whole aligned rows: the same bits as
with aligned ones."""
import numpy as np
import pytest
import torch

from test_gpu_kv_quant import _filled, _tree_mask

pytestmark = pytest.mark.gpu


def _off_grid(q, how):
    """The values of q at another place in memory, `how` off the 16-byte grid."""
    if how == "address":  # contiguous, one element behind an aligned address
        flat = torch.empty(q.numel() + 8, dtype=q.dtype, device=q.device)
        out = flat[1 : 1 + q.numel()].view(q.shape)
    elif how == "rows":  # a slice of a wider projection: rows 8 k + 3 elements apart
        out = torch.empty(*q.shape[:-1], q.shape[-1] + 11, dtype=q.dtype, device=q.device)[..., 8:-3]
    else:  # the last dimension strided
        out = torch.empty(*q.shape, 2, dtype=q.dtype, device=q.device)[..., 0]
    out.copy_(q)
    assert torch.equal(out, q)
    return out


@pytest.mark.parametrize("how", ["address", "rows", "strided"])
@pytest.mark.parametrize("dtype,bits,dim", [(torch.bfloat16, 4, 128), (torch.float16, 8, 64)])
@pytest.mark.parametrize("batch,n", [(1, 1), (2, 3), (2, 130)])
def test_queries_off_the_grid(batch, n, dtype, bits, dim, how):
    from recurrent_drafting_amd import attention
    from recurrent_drafting_amd.packed_rows import PackedRows

    rng = np.random.default_rng(n)
    prev, heads = 90, 4
    cache, _, _ = _filled(rng, batch, 2, prev + n, dim, dtype, bits)
    keys, values = (view.rows() for view in cache.sliced[0])
    q = torch.tensor(rng.standard_normal((batch, heads, n, dim))).to(dtype).cuda()
    mask = torch.tensor(_tree_mask(rng, batch, n, prev, [0, 5][:batch])).cuda()
    prepared = attention.prepare(mask, n_heads=heads)
    want = attention.masked_attention(q, keys, values, prepared)
    off = _off_grid(q, how)
    kept = off.clone()
    assert torch.equal(attention.masked_attention(off, keys, values, prepared), want)
    assert torch.equal(off, kept)
    # packed rows: the slots that exist, and stand-in rows behind them
    counts = [n] + [max(1, n // 2)] * (batch - 1)
    rows = PackedRows.from_counts(torch.tensor(counts, dtype=torch.int32).cuda(), sum(counts), n)
    packed = torch.zeros(rows.rows, heads, dim, dtype=dtype, device="cuda")
    packed[: sum(counts)] = torch.cat([q[b, :, :c].transpose(0, 1) for b, c in enumerate(counts)])
    got = attention.masked_attention(_off_grid(packed, how), keys, values, prepared, rows=rows)
    at = 0
    for b, c in enumerate(counts):
        assert torch.equal(got[at : at + c], want[b, :c])
        at += c


def test_a_type_that_runs_on_the_generic_kernel():
    from recurrent_drafting_amd import attention

    rng = np.random.default_rng(3)
    cache, _, _ = _filled(rng, 1, 2, 60, 128, torch.float32, 4)
    keys, values = (view.rows() for view in cache.sliced[0])
    q = torch.tensor(rng.standard_normal((1, 4, 3, 128))).float().cuda()
    prepared = attention.prepare(torch.ones(1, 3, 60, dtype=torch.bool, device="cuda"), n_heads=4)
    want = attention.masked_attention(q, keys, values, prepared)
    for how in ("address", "rows", "strided"):
        assert torch.equal(attention.masked_attention(_off_grid(q, how), keys, values, prepared), want)
