"""What the entry points of the 4- and 8-bit cache refuse, answered on the host: null data pointers
wherever a size is wrong, so that nothing can be launched, and the Python surface's own checks."""
import ctypes as C

import pytest
import torch

EINVAL, ELIMIT, EWORKSPACE = -1, -2, -3
BF16, F16, F32 = 0, 1, 2
FAKE = 0x1000  # an aligned address that no refused call ever reads


def _lib():
    from recurrent_drafting_amd import _hip

    return _hip.lib()


def _s(*v):
    return (C.c_int64 * len(v))(*v)


def test_row_bytes():
    lib = _lib()
    for bits, dim, want in [(4, 128, 80), (8, 128, 144), (4, 64, 48), (8, 64, 80), (4, 32, 32), (4, 256, 160), (8, 256, 288),
                            (4, 96, 64), (3, 128, 0), (16, 128, 0), (4, 0, 0), (4, 48, 0), (4, 288, 0), (8, -32, 0)]:
        assert lib.rd_kv_quant_row_bytes(bits, dim) == want


def test_nothing_is_captured_on_the_null_stream():
    assert _lib().rd_stream_capture_id(None) == 0


def _append(lib, batch=2, n_new=3, heads=4, kv_heads=2, dim=64, bits=4, row0=0, max_len=8, dtype=BF16, table=16,
            q=FAKE, strides=(256 * 3, 256), cache=(48 * 8 * 2, 48 * 8, 48), k_cache=FAKE):
    return lib.rd_rope_append_quant(q, _s(*strides), FAKE, _s(*strides), FAKE, _s(*strides), dtype, batch, n_new, heads,
                                    kv_heads, dim, FAKE, FAKE, table, FAKE, n_new, FAKE, _s(*strides), k_cache, FAKE,
                                    _s(*cache), bits, row0, max_len, None, None, None)


@pytest.mark.parametrize("change,code,word", [
    (dict(batch=0), EINVAL, b"bad sizes"), (dict(n_new=0), EINVAL, b"bad sizes"), (dict(batch=65536), ELIMIT, b"65535"),
    (dict(dtype=3), EINVAL, b"dtype"), (dict(bits=5), EINVAL, b"bits"), (dict(dim=48), ELIMIT, b"multiple of 32"),
    (dict(dim=288), ELIMIT, b"at most 256"), (dict(q=None), EINVAL, b"null"), (dict(table=0), EINVAL, b"table"),
    (dict(row0=6), EINVAL, b"do not fit"), (dict(row0=-1), EINVAL, b"do not fit"), (dict(n_new=9), EINVAL, b"do not fit"),
    (dict(q=FAKE + 2), EINVAL, b"aligned"), (dict(k_cache=FAKE + 8), EINVAL, b"aligned"),
    (dict(strides=(772, 256)), EINVAL, b"strides"), (dict(cache=(48 * 16, 48 * 8, 32)), EINVAL, b"strides"),
    (dict(cache=(48 * 16 + 8, 48 * 8, 48)), EINVAL, b"strides"), (dict(row0=2 ** 62), EINVAL, b"do not fit"),
])
def test_append_refusals(change, code, word):
    lib = _lib()
    assert _append(lib, **change) == code and word in lib.rd_last_error()


def _rows(lib, which, batch=2, heads=2, n=4, dim=64, bits=8, dtype=F16, x=FAKE, xs=(512, 256, 64), cache=FAKE,
          cs=(80 * 16, 80 * 8, 80), row0=0, max_len=8):
    if which == "write":
        return lib.rd_kv_quantize(x, _s(*xs), dtype, batch, heads, n, dim, bits, cache, _s(*cs), row0, max_len, None)
    return lib.rd_kv_dequantize(cache, _s(*cs), bits, dtype, batch, heads, row0, n, dim, max_len, x, _s(*xs), None)


@pytest.mark.parametrize("which", ["write", "read"])
@pytest.mark.parametrize("change,code,word", [
    (dict(batch=0), EINVAL, b"bad sizes"), (dict(n=0), EINVAL, b"bad sizes"), (dict(heads=65536), ELIMIT, b"65535"),
    (dict(dtype=7), EINVAL, b"dtype"), (dict(bits=2), EINVAL, b"bits"), (dict(dim=40), ELIMIT, b"multiple of 32"),
    (dict(x=None), EINVAL, b"null"), (dict(cache=None), EINVAL, b"null"), (dict(n=9), EINVAL, b"do not fit"),
    (dict(row0=5), EINVAL, b"do not fit"), (dict(cache=FAKE + 4), EINVAL, b"aligned"), (dict(cs=(1280, 640, 64)), EINVAL, b"strides"),
])
def test_row_refusals(which, change, code, word):
    lib = _lib()
    assert _rows(lib, which, **change) == code and word in lib.rd_last_error()


def test_reading_wants_aligned_rows():
    lib = _lib()
    assert _rows(lib, "read", x=FAKE + 2) == EINVAL and b"16-byte" in lib.rd_last_error()
    assert _rows(lib, "read", xs=(512, 256, 68)) == EINVAL and b"16-byte" in lib.rd_last_error()


def _attend(lib, batch=2, heads=8, kv_heads=2, n_q=3, kv=100, dim=128, bits=4, dtype=BF16, scale=0.1, q=FAKE, spans=FAKE,
            cache=FAKE, cs=(80 * 512, 80 * 256, 80), max_len=256, ws=None, ws_bytes=0, qs=(8192, 128, 1024)):
    return lib.rd_verify_attention_quant(q, _s(*qs), cache, FAKE, _s(*cs), bits, max_len, FAKE, _s(*qs), dtype, batch, heads,
                                         kv_heads, n_q, kv, dim, scale, FAKE, FAKE, spans, ws, ws_bytes, 0, None, None)


@pytest.mark.parametrize("change,code,word", [
    (dict(batch=0), EINVAL, b"bad sizes"), (dict(kv=0), EINVAL, b"bad sizes"), (dict(kv_heads=3), EINVAL, b"multiple"),
    (dict(dtype=9), EINVAL, b"dtype"), (dict(bits=6), EINVAL, b"bits"), (dict(dim=80), ELIMIT, b"multiple of 32"),
    (dict(batch=65536), ELIMIT, b"65535"), (dict(kv=2 ** 23 + 1), ELIMIT, b"2^23"), (dict(n_q=2 ** 29), ELIMIT, b"query rows"),
    (dict(q=None), EINVAL, b"null"), (dict(spans=None), EINVAL, b"null"), (dict(max_len=0), EINVAL, b"empty"),
    (dict(spans=FAKE + 4), EINVAL, b"aligned"),
    (dict(scale=0.0), EINVAL, b"scale"), (dict(scale=-1.0), EINVAL, b"scale"), (dict(scale=float("nan")), EINVAL, b"scale"),
    (dict(scale=float("inf")), EINVAL, b"scale"), (dict(cache=FAKE + 8), EINVAL, b"aligned"),
    (dict(cs=(80 * 512, 80 * 256, 96)), EINVAL, b"strides"), (dict(cs=(80 * 512 + 4, 80 * 256, 80)), EINVAL, b"strides"),
    (dict(batch=1, kv=8192), EWORKSPACE, b"workspace"), (dict(batch=1, kv=8192, ws=FAKE, ws_bytes=16), EWORKSPACE, b"workspace"),
    (dict(batch=1, kv=8192, ws=FAKE + 16, ws_bytes=2 ** 40), EINVAL, b"256B"),
])
def test_attention_refusals(change, code, word):
    lib = _lib()
    assert _attend(lib, **change) == code and word in lib.rd_last_error()


def test_spans_and_workspace_sizes():
    lib = _lib()
    assert lib.rd_attn_spans_ints(3, 1) == 12 and lib.rd_attn_spans_ints(2, 17) == 16 and lib.rd_attn_spans_ints(0, 1) == 0
    assert lib.rd_attn_spans(None, 1, 1, 1, None, None) == EINVAL and lib.rd_attn_spans(FAKE, 0, 1, 1, FAKE, None) == EINVAL
    assert lib.rd_attn_spans(FAKE, 65536, 1, 1, FAKE, None) == ELIMIT
    need = lib.rd_verify_attention_quant_workspace_bytes
    assert need(BF16, 1, 32, 8, 1, 64, 128) == 0                        # a short cache is not cut
    assert need(F32, 1, 32, 8, 1, 65536, 128) == 0 == need(BF16, 1, 32, 8, 1, 65536, 96)  # the generic kernel cuts nothing
    long = need(F16, 1, 32, 8, 1, 65536, 128)
    assert long > 0 and long % 256 == 0 and need(F16, 1, 30, 8, 1, 65536, 128) == 0


def test_python_surface():
    from recurrent_drafting_amd import kv_cache

    for bits, dim in [(3, 128), (16, 128), (4, 48), (8, 512), (0, 64)]:
        with pytest.raises(ValueError, match="bits"):
            kv_cache.Cache(1, 4, 1, 2, dim, torch.bfloat16, torch.device("cpu"), bits=bits)
    with pytest.raises(TypeError, match="dtype"):
        kv_cache.Cache(1, 4, 1, 2, 64, torch.float64, torch.device("cpu"), bits=4)
    cache = kv_cache.Cache(2, 6, 3, 2, 64, torch.bfloat16, torch.device("cpu"), bits=4)
    key, _ = cache.sliced[1]
    assert cache._cache.shape == (3, 2, 2, 2, 6, 48) and cache._cache.dtype == torch.uint8
    assert key.shape == (2, 2, 0, 64) and key.bits == 4 and cache._geometry() == (3, 2, 2, 6, 48)
    with pytest.raises(RuntimeError, match="GPU"):  # no CPU path
        key.append(torch.zeros(2, 2, 1, 64, dtype=torch.bfloat16))
    with pytest.raises(AssertionError):
        key.append(torch.zeros(2, 2, 7, 64, dtype=torch.bfloat16))
    assert key.length == 0
    plain = kv_cache.Cache(2, 6, 1, 2, 64, torch.bfloat16, torch.device("cpu"))
    key, _ = plain.sliced[0]
    x = torch.randn(2, 2, 3, 64).bfloat16()
    assert torch.equal(key.cat(x), x) and torch.equal(key.slice(1), x[:, :, 1:]) and key.bits is None
    assert torch.equal(key.rows(), x)
