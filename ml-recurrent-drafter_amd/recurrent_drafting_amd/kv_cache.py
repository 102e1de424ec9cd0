"""Pre-allocated KV cache with the reference's View/Cache objects (recurrent_drafting/kv_cache.py).

One dense tensor (n_layers, 2, batch, n_heads, max_length, head_dim) lives in HBM for the whole
generation; `View.cat` appends in place and hands back a strided view, `Cache.unpack` and
`Cache.compact` move rows with the HIP kernels rd_kv_unpack / rd_kv_compact (in place, no clone).

Rows in place: the reference re-right-aligns the whole live cache after every step
(recurrent_drafting.py:200-209).  With `Cache.rows_in_place = True` (the decode loop of
`RecurrentDrafting` sets it) the cache rows never move: a per-row `Cache.shift` says that token
column c of row b lives in cache row c - shift[b]; the re-alignment adds the change of the left
padding to it, and `rope_append` and the attention subtract it.  `Cache.materialize()` moves the rows
once to the reference's layout; `View.cat`, `View.slice` and `Cache.unpack` call it first.

Rows in 4 or 8 bits: `Cache(..., bits=4)` holds every row as a record of small scaled floats (blocks
of 8 values with a common power of two; include/redrafter_hip.h has the format), 80 or 144 bytes at
head_dim 128 where bf16 takes 256.  Rows are rounded as they are written (`rope_append`, `View.append`,
`View.cat`) and read back in the model's type by `View.slice` and `View.cat`; `rope_append` and
`View.rows` hand out `QuantizedRows`, which `attention.masked_attention` reads as they are.  Moving rows
(unpack, compact, materialize, rows in place) moves the records.
"""

from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch

from . import _hip
from .packed_rows import PackedRows


class QuantizedRows:
    """Key or value rows [prev, length) of one layer of a cache held in 4 or 8 bits."""

    __slots__ = ("_owner", "_layer", "_kv", "_prev", "_length")

    def __init__(self, owner: "Cache", layer: int, kv: int, prev: int, length: int):
        # (prev behind the last row: no rows, as of a tensor's slice)
        self._owner, self._layer, self._kv, self._length = owner, layer, kv, length
        self._prev = prev if prev < length else length

    @property
    def bits(self) -> int:
        return self._owner.bits

    @property
    def head_dim(self) -> int:
        return self._owner.head_dim

    @property
    def dtype(self) -> torch.dtype:
        """The type the rows were rounded from and are read back in."""
        return self._owner.dtype

    @property
    def shape(self) -> Tuple[int, int, int, int]:
        owner = self._owner
        batch, n_heads, _ = owner.slab_shape
        return (batch, n_heads, self._length - self._prev, owner.head_dim)

    @property
    def records(self) -> torch.Tensor:
        """(batch, n_heads, length - prev, record bytes) uint8, a view of the cache."""
        return self._owner._cache[self._layer, self._kv, :, :, self._prev : self._length, :]

    def data_ptr(self) -> int:
        """Address of the first record."""
        owner = self._owner
        layer, kv, row = owner.slab_strides
        return owner._cache.data_ptr() + self._layer * layer + self._kv * kv + self._prev * row

    def read(self) -> torch.Tensor:
        """The values, (batch, n_heads, length - prev, head_dim) in `dtype`: exact, every value the records
        can hold is a number of that type."""
        return _read(self._owner, self._layer, self._kv, self._prev, self._length)


def _read(owner: "Cache", layer: int, kv: int, prev: int, length: int) -> torch.Tensor:
    """Rows [prev, length) of a layer's keys or values out of a cache in 4 or 8 bits (rd_kv_dequantize)."""
    cache, head_dim, n_rows = owner._cache, owner.head_dim, max(length - prev, 0)
    batch, n_heads, max_length = owner.slab_shape
    out = cache.new_empty((batch, n_heads, n_rows, head_dim), dtype=owner.dtype)
    if n_rows == 0 or batch == 0:
        return out
    _hip.on_current_device(cache)
    per_layer, per_side, _ = owner.slab_strides
    row = n_rows * head_dim
    _hip.check(
        _hip.lib().rd_kv_dequantize(
            cache.data_ptr() + layer * per_layer + kv * per_side, owner.byte_strides, owner.bits, owner.dtype_code,
            batch, n_heads, prev, n_rows, head_dim, max_length, out.data_ptr(),
            _hip.I64x3(n_heads * row, row, head_dim), _hip.stream(),
        )
    )
    return out


class View:
    """Key or value rows of one layer: cache[layer, kv, :, :, 0:length, :] (kv_cache.py:10-35)."""

    def __init__(self, cache: torch.Tensor, layer: int, kv: int, owner: Optional["Cache"] = None):
        self._cache = cache
        self._layer = layer
        self._kv = kv  # 0 = key, 1 = value
        self._owner = owner
        self.length = 0

    @property
    def shape(self) -> Tuple[int, int, int, int]:
        _, _, batch_size, n_heads, _, head_dim = self._cache.shape
        return (batch_size, n_heads, self.length, head_dim if self.bits is None else self._owner.head_dim)

    @property
    def bits(self) -> Optional[int]:
        """4 or 8 for a cache that holds its rows in so many bits, None for one in the model's type."""
        return None if self._owner is None else self._owner.bits

    def append(self, new_kv: torch.Tensor) -> None:
        """Appends (batch, n_heads, n_new, head_dim) rows in place (rounded to the cache's bits)."""
        batch_size, n_heads, _, head_dim = self.shape
        max_length = self._cache.shape[4]
        n_new = new_kv.shape[2]
        assert new_kv.shape == (batch_size, n_heads, n_new, head_dim)
        assert self.length + n_new <= max_length
        if self._owner is not None:
            self._owner.materialize()
        slab = self._cache[self._layer, self._kv]
        if self.bits is None:
            slab[:, :, self.length : self.length + n_new, :] = new_kv
        elif new_kv.numel():
            x = new_kv.to(self._owner.dtype)  # (what an assignment to a cache in the model's type does)
            if x.stride(3) != 1:
                x = x.contiguous()
            _hip.on_current_device(x, slab)
            _hip.check(
                _hip.lib().rd_kv_quantize(
                    x.data_ptr(), _hip.I64x3(*x.stride()[:3]), self._owner.dtype_code,
                    batch_size, n_heads, n_new, head_dim, self.bits, slab.data_ptr(),
                    self._owner.byte_strides, self.length, max_length, _hip.stream(),
                )
            )
        self.length += n_new

    def cat(self, new_kv: torch.Tensor) -> torch.Tensor:
        """Appends (batch, n_heads, n_new, head_dim) rows in place and returns rows [0, length) (of a
        cache in 4 or 8 bits: their values, read back)."""
        self.append(new_kv)
        return self.slice(0)

    def rows(self, prev: int = 0):
        """Rows [prev, length) as the attention reads them: a view of the cache in the model's type, or
        the `QuantizedRows` of one in 4 or 8 bits.  With cache rows in place these are cache rows, not
        token columns (a PreparedMask built with the cache's shifts goes with them)."""
        if self.bits is not None:
            return QuantizedRows(self._owner, self._layer, self._kv, prev, self.length)
        return self._cache[self._layer, self._kv, :, :, prev : self.length, :]

    def slice(self, prev: int) -> torch.Tensor:
        """Rows [prev, length) (of a cache in 4 or 8 bits: their values, read back)."""
        owner = self._owner
        if owner is not None:
            owner.materialize()
            if owner.bits is not None:
                return _read(owner, self._layer, self._kv, prev, self.length)
        return self.rows(prev)


def rope_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
                position_ids: torch.Tensor, past_key_value: Tuple[View, View],
                rows: Optional[PackedRows] = None):
    """Rotates q and k by their positions and appends the rotated k and v to the cache, one kernel.

    q (B, n, heads*D) and k, v (B, n, kv_heads*D) as the projections produce them (token rows may be
    strided, e.g. slices of one fused projection); cos/sin (positions, D) tables in q's dtype;
    position_ids (B, n) int64.  q is rotated in place.  Returns (q as (B, heads, n, D) view, keys,
    values) with keys/values the (B, kv_heads, length, D) views `View.cat` would return
    (modeling_llama.py:148-159, apply_rotary_pos_emb :87-110).

    With `rows`, q, k and v are (total, heads*D) / (total, kv_heads*D): only the slots that exist.
    The cache still grows by n rows per batch row (the slots that do not exist keep what the
    cache held), and q comes back as a (total, heads, D) view.

    A cache in 4 or 8 bits takes the records of the keys as fp64 rotates them and of the values, and keys and
    values come back as its `QuantizedRows`.  q is then rotated into a tensor of its own (rounded once; the
    projection's output is left as it was), of which the result is a view; rows behind the last token of
    a packed batch are not written."""
    key_view, value_view = past_key_value
    if key_view.bits is not None:
        return _rope_append_quantized(q, k, v, cos, sin, position_ids, key_view, value_view, rows)
    cache = key_view._cache
    batch, n_kv_heads, _, head_dim = key_view.shape
    max_length = cache.shape[4]
    if rows is None:
        n_new = q.shape[1]
        lead = (batch, n_new)
        strides = lambda t: _hip.I64x2(t.stride(0), t.stride(1))
    else:
        assert rows.batch == batch
        n_new = rows.n
        lead = (rows.rows,)
        strides = lambda t: _hip.I64x2(0, t.stride(0))
    n_heads = q.shape[-1] // head_dim
    assert q.shape == (*lead, n_heads * head_dim) and q.stride(-1) == 1
    assert k.shape == (*lead, n_kv_heads * head_dim) and k.stride(-1) == 1
    assert v.shape == k.shape and v.stride(-1) == 1
    assert q.dtype == k.dtype == v.dtype == cache.dtype == cos.dtype == sin.dtype
    assert cos.shape == sin.shape and cos.shape[1] == head_dim and cos.is_contiguous() and sin.is_contiguous()
    assert position_ids.shape == (batch, n_new) and position_ids.dtype == torch.long and position_ids.stride(1) == 1
    assert key_view.length == value_view.length and key_view.length + n_new <= max_length
    assert value_view._cache is cache and key_view._layer == value_view._layer
    owner = key_view._owner
    shift = owner.shift if owner is not None and owner.rows_in_place else None
    k_slab = cache[key_view._layer, 0]
    v_slab = cache[key_view._layer, 1]
    _hip.check(
        _hip.lib().rd_rope_append(
            _hip.ptr(q), strides(q), _hip.ptr(k), strides(k), _hip.ptr(v), strides(v),
            _hip.dtype_code(q.dtype), batch, n_new, n_heads,
            n_kv_heads, head_dim, _hip.ptr(cos), _hip.ptr(sin), cos.shape[0], _hip.ptr(position_ids),
            position_ids.stride(0), _hip.ptr(q), strides(q), _hip.ptr(k_slab), _hip.ptr(v_slab),
            (ctypes.c_int64 * 3)(k_slab.stride(0), k_slab.stride(1), k_slab.stride(2)), key_view.length,
            max_length, _hip.ptr(rows.row_start) if rows is not None else None, _hip.ptr(shift), _hip.stream(),
        )
    )
    key_view.length += n_new
    value_view.length += n_new
    if rows is None:
        q_heads = q.unflatten(2, (n_heads, head_dim)).transpose(1, 2)
    else:
        q_heads = q.unflatten(1, (n_heads, head_dim))
    return q_heads, k_slab[:, :, : key_view.length, :], v_slab[:, :, : value_view.length, :]


def _rope_append_quantized(q, k, v, cos, sin, position_ids, key_view: View, value_view: View,
                           rows: Optional[PackedRows]):
    """rope_append into a cache in 4 or 8 bits (rd_rope_append_quant).  For a single token the kernel takes less
    time than this function, so every tensor is asked once for what is needed of it."""
    cache, owner, layer, length = key_view._cache, key_view._owner, key_view._layer, key_view.length
    batch, n_kv_heads, max_length = owner.slab_shape
    head_dim = owner.head_dim
    q_shape, k_shape, q_stride, k_stride, v_stride = q.shape, k.shape, q.stride(), k.stride(), v.stride()
    width, kv_width = q_shape[-1], n_kv_heads * head_dim
    n_heads = width // head_dim
    n_new = q_shape[1] if rows is None else rows.n
    if rows is None:
        assert q_shape == (batch, n_new, n_heads * head_dim) and k_shape == (batch, n_new, kv_width)
        q_strides, k_strides, v_strides = _hip.I64x2(*q_stride[:2]), _hip.I64x2(*k_stride[:2]), _hip.I64x2(*v_stride[:2])
    else:
        assert rows.batch == batch
        assert q_shape == (rows.rows, n_heads * head_dim) and k_shape == (rows.rows, kv_width)
        q_strides, k_strides, v_strides = _hip.I64x2(0, q_stride[0]), _hip.I64x2(0, k_stride[0]), _hip.I64x2(0, v_stride[0])
    assert v.shape == k_shape and q_stride[-1] == k_stride[-1] == v_stride[-1] == 1
    dtype = q.dtype
    assert dtype == k.dtype == v.dtype == owner.dtype == cos.dtype == sin.dtype
    table = cos.shape
    assert table == sin.shape and table[1] == head_dim and cos.is_contiguous() and sin.is_contiguous()
    positions = position_ids.stride()
    assert position_ids.shape == (batch, n_new) and position_ids.dtype == torch.long and positions[1] == 1
    assert length == value_view.length and length + n_new <= max_length
    assert value_view._cache is cache and layer == value_view._layer
    _hip.on_current_device(q, k, v, cos, sin, position_ids, cache)
    # the result: (batch, heads, n, head_dim), a view of (batch, n, heads, head_dim)
    if rows is None:
        q_out = q.new_empty_strided((batch, n_heads, n_new, head_dim), (n_new * width, head_dim, width, 1))
        out_strides = _hip.I64x2(n_new * width, width)
    else:
        q_out = q.new_empty((rows.rows, n_heads, head_dim))
        out_strides = _hip.I64x2(0, width)
    keys = QuantizedRows(owner, layer, 0, 0, length + n_new)
    values = QuantizedRows(owner, layer, 1, 0, length + n_new)
    first = keys.data_ptr()
    _hip.check(
        _hip.lib().rd_rope_append_quant(
            q.data_ptr(), q_strides, k.data_ptr(), k_strides, v.data_ptr(), v_strides, owner.dtype_code, batch, n_new,
            n_heads, n_kv_heads, head_dim, cos.data_ptr(), sin.data_ptr(), table[0], position_ids.data_ptr(),
            positions[0], q_out.data_ptr(), out_strides, first, first + owner.slab_strides[1], owner.byte_strides,
            owner.bits, length, max_length, None if rows is None else _hip.ptr(rows.row_start),
            _hip.ptr(owner.shift) if owner._rows_in_place else None, _hip.stream(),
        )
    )
    key_view.length = value_view.length = length + n_new
    return q_out, keys, values


class Cache:
    def __init__(
        self,
        batch_size: int,
        max_length: int,
        n_layers: int,
        n_heads: int,
        head_dim: int,
        dtype: torch.dtype,
        device: torch.device,
        bits: Optional[int] = None,
    ) -> None:
        """bits: None for rows in `dtype` (the reference's cache); 4 or 8 for rows rounded from `dtype`
        to so many bits as they are written (head_dim a multiple of 32, at most 256)."""
        self.bits, self.dtype, self.head_dim = bits, dtype, head_dim
        row, element = head_dim, dtype
        if bits is not None:
            self.dtype_code = _hip.dtype_code(dtype)
            row, element = _hip.lib().rd_kv_quant_row_bytes(int(bits), head_dim), torch.uint8
            if bits not in (4, 8) or row == 0:
                raise ValueError(f"a cache in {bits} bits with head_dim {head_dim}: bits must be 4 or 8, head_dim a "
                                 "multiple of 32 and at most 256")
            self.bits = int(bits)
        # (the attention reads only the cache rows of keys that somebody attends to, so nothing is
        # asked of the memory around a row's live rows; zeros as upstream, kv_cache.py:49-53)
        self._storage = torch.zeros([n_layers, 2, batch_size, n_heads, max_length, row], dtype=element, device=device)
        self._cache = self._storage
        self.byte_strides = None  # of {batch, head, row} in a layer's keys or values, for the C ABI
        if bits is not None:
            layer, kv, batch, head, row, _ = self._cache.stride()
            self.byte_strides = _hip.I64x3(batch, head, row)
            self.slab_shape = (batch_size, n_heads, max_length)
            self.slab_strides = (layer, kv, row)  # bytes from layer to layer, from keys to values, from row to row
        self.sliced = tuple(
            (View(self._cache, layer, 0, self), View(self._cache, layer, 1, self)) for layer in range(n_layers)
        )
        # token column c of batch row b lives in cache row c - shift[b] (all zero: the reference's layout)
        self.shift = torch.zeros(batch_size, dtype=torch.int32, device=device)
        self._rows_in_place = False
        self._shifted = False  # host-side: a re-alignment may have left non-zero shifts

    @property
    def rows_in_place(self) -> bool:
        """True: re-alignments leave the cache rows where they are and update `shift` instead."""
        return self._rows_in_place

    @rows_in_place.setter
    def rows_in_place(self, value: bool) -> None:
        if not value:
            self.materialize()  # nobody would follow the shifts any more
        self._rows_in_place = bool(value)

    # -- geometry handed to the C ABI ---------------------------------------------------------
    def _geometry(self):
        n_layers, _, batch, n_heads, max_len, row = self._cache.shape  # (row: head_dim elements, or a record's bytes)
        return n_layers, batch, n_heads, max_len, row * self._cache.element_size()

    def materialize(self) -> None:
        """Moves the rows to the layout in which column and cache row agree (no-op unless a
        re-alignment with rows in place has happened since the last call)."""
        if not self._shifted:
            return
        n_layers, batch, n_heads, max_len, row_bytes = self._geometry()
        lib = _hip.lib()
        plan = torch.empty(lib.rd_kv_materialize_plan_ints(batch), dtype=torch.int32, device=self._cache.device)
        _hip.check(
            lib.rd_kv_materialize(
                _hip.ptr(self._cache), n_layers, batch, n_heads, max_len, row_bytes,
                self.sliced[0][0].length, _hip.ptr(self.shift), _hip.ptr(plan), _hip.stream(),
            )
        )
        self._shifted = False

    def set_length(self, length: int) -> None:
        for key, value in self.sliced:
            key.length = value.length = length

    def unpack(self, prompt_length: int, tree_attn_index: torch.Tensor) -> None:
        """Every candidate position (beam, k) gets its own cache row behind the prompt:
        row prompt_length + beam*L + k takes the packed row prompt_length + tree_attn_index[b,beam,k]
        (kv_cache.py:58-98)."""
        batch, width, length = tree_attn_index.shape
        n_layers, cb, n_heads, max_len, row_bytes = self._geometry()
        assert cb == batch
        self.materialize()
        n_out = width * length
        n_src = self.sliced[0][0].length - prompt_length
        assert n_src > 0, "no packed rows behind the prompt"
        assert prompt_length + n_out <= max_len
        index = tree_attn_index.contiguous()
        assert index.dtype == torch.long
        _hip.check(
            _hip.lib().rd_kv_unpack(
                _hip.ptr(self._cache), n_layers, batch, n_heads, max_len, row_bytes, prompt_length,
                _hip.ptr(index), n_out, n_src, _hip.stream(),
            )
        )
        self.set_length(prompt_length + n_out)

    def compact(self, prev: int, beam_length: int, plan: torch.Tensor, new_length: int) -> None:
        """Follows a plan written by rd_realign_plan: accepted rows kept, rows re-right-aligned."""
        n_layers, batch, n_heads, max_len, row_bytes = self._geometry()
        assert plan.dtype == torch.int32
        _hip.check(
            _hip.lib().rd_kv_compact(
                _hip.ptr(self._cache), n_layers, batch, n_heads, max_len, row_bytes, prev,
                beam_length, _hip.ptr(plan), _hip.stream(),
            )
        )
        self.set_length(new_length)
