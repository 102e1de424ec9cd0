"""Edges of the 4- and 8-bit cache's calls that the host answers."""
import math

import pytest
import torch

from test_kv_quant_limits import EINVAL, F32, _attend, _lib


@pytest.mark.parametrize("bits", [None, 4, 8])
def test_a_slice_behind_the_last_row_is_empty(bits):
    """As of a cache in the model's type."""
    from recurrent_drafting_amd import kv_cache

    cache = kv_cache.Cache(2, 6, 1, 3, 64, torch.bfloat16, torch.device("cpu"), bits=bits)
    key, _ = cache.sliced[0]
    key.length = 2
    for prev in (2, 3, 6, 9):
        got = key.slice(prev)
        assert got.shape == (2, 3, 0, 64) and got.dtype == torch.bfloat16
        assert key.rows(prev).shape == (2, 3, 0, 64)
    if bits is not None:
        assert key.rows(9).read().shape == (2, 3, 0, 64) and key.rows(9).records.shape[2] == 0

@pytest.mark.parametrize("dtype,dim", [(0, 128), (F32, 128), (1, 96)])
def test_a_scale_that_overflows_in_log2_units_is_refused(dtype, dim):
    lib = _lib()
    largest = 3.4028234663852886e38
    record = {128: 80, 96: 64}[dim]
    for scale in (largest, 2.4e38, largest * math.log(2) * 1.00001):
        assert _attend(lib, scale=scale, dtype=dtype, dim=dim, cs=(record * 512, record * 256, record)) == EINVAL
        assert b"scale" in lib.rd_last_error()
