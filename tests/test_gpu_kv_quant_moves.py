"""Records of a cache in 4 or 8 bits moved by the decode loop (re-alignment with rows in place and with moved rows,
rd_kv_append, rd_kv_compact, rd_kv_materialize), the loop itself on the matrix kernel, and rows that no call may
write."""
import ctypes as C
import os
import sys

import numpy as np
import pytest
import torch

sys.path.insert(0, os.path.join(os.path.dirname(__file__), "golden"))
import tiny_models as tm  # noqa: E402

pytestmark = pytest.mark.gpu


def _new(batch, max_len, heads, dim, dtype, bits, layers=1):
    from recurrent_drafting_amd import kv_cache

    return kv_cache.Cache(batch, max_len, layers, heads, dim, dtype, torch.device("cuda"), bits=bits)


# ---- moves ----------------------------------------------------------------------------------------------

@pytest.mark.parametrize("width,length", [(5, 4), (2, 30)])  # (30 rows of 144 bytes are more than rd_kv_append takes)
@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("bits,dim", [(4, 128), (8, 128), (4, 64), (8, 64), (4, 32)])
def test_realignment_moves_records(bits, dim, in_place, packed, width, length):
    """Three re-alignments with ragged accepted counts and ragged left padding; every live record of every layer,
    side and head against rows moved on the host.  packed: accepted rows out of the packed slots."""
    from recurrent_drafting_amd import acceptance

    rng = np.random.default_rng(dim + bits + length)
    batch, heads, layers, prev, n_slots = 4, 3, 2, 23, 9
    pads = [int(p) for p in rng.integers(0, 9, batch)]
    pads[1] = 0
    ids = rng.integers(1, 50, (batch, prev))
    for b in range(batch):
        ids[b, : pads[b]] = 0
    cache = _new(batch, prev + 3 * length + width * length + 20, heads, dim, torch.bfloat16, bits, layers)
    cache._cache.copy_(torch.tensor(rng.integers(0, 256, tuple(cache._cache.shape), dtype=np.uint8)))
    start = cache._cache.cpu().numpy()
    live = [start[:, :, b, :, pads[b] : prev] for b in range(batch)]  # (layers, 2, heads, tokens, record)
    cache.rows_in_place = in_place
    ids, shifted = torch.tensor(ids).cuda(), 0
    for _ in range(3):
        prev = ids.shape[1]
        beams = torch.tensor(rng.integers(1, 50, (batch, width, length))).cuda()
        accepted, seq = rng.integers(0, length, batch), rng.integers(0, width, batch)
        slots = rng.integers(0, n_slots, (batch, width, length))
        n_new_rows = n_slots if packed else width * length
        fresh = rng.integers(0, 256, (layers, 2, batch, heads, n_new_rows, start.shape[5]), dtype=np.uint8)
        shift = cache.shift.cpu().tolist()
        for b in range(batch):  # what a verification step appends, where the cache keeps column prev + t
            cache._cache[:, :, b, :, prev - shift[b] : prev - shift[b] + n_new_rows] = torch.tensor(fresh[:, :, b]).cuda()
        cache.set_length(prev + n_new_rows)
        old = (ids != 0).sum(1).tolist()
        ids = acceptance.realign(ids, torch.tensor(accepted).cuda(), torch.tensor(seq).cuda(), beams, cache, 0,
                                 unpacker=torch.tensor(slots).cuda() if packed else None)
        grown = [new - o for new, o in zip((ids != 0).sum(1).tolist(), old)]
        assert len(set(grown)) > 1
        for b in range(batch):
            rows = [int(slots[b, seq[b], j]) if packed else int(seq[b]) * length + j for j in range(grown[b])]
            live[b] = np.concatenate((live[b], fresh[:, :, b][:, :, :, rows]), axis=3)
        shifted += int(cache.shift.abs().sum())
    assert (shifted > 0) == in_place
    for view in cache.sliced[1]:  # (a row that is read is home first)
        view.slice(0)
    assert not cache._shifted and not cache.shift.any()
    end, total = cache._cache.cpu().numpy(), ids.shape[1]
    assert cache.sliced[0][0].length == total == max(x.shape[3] for x in live)
    for b in range(batch):
        assert np.array_equal(end[:, :, b, :, total - live[b].shape[3] : total], live[b]), b


# ---- the decode loop on the matrix kernel ----------------------------------------------------------------

@pytest.mark.parametrize("sampling", [False, True])
@pytest.mark.parametrize("dtype,bits,heads,kv_heads", [
    (torch.bfloat16, 4, 4, 4), (torch.bfloat16, 8, 4, 2), (torch.float16, 4, 8, 2), (torch.float16, 8, 8, 8)])
def test_generate_on_the_matrix_kernel(dtype, bits, heads, kv_heads, sampling):
    """Heads of 128 and 64 in bf16 and fp16: rows kept in place and rows moved every
    step give the same tokens, and no attention runs on the generic kernel."""
    import recurrent_drafting_amd as rd
    from recurrent_drafting_amd import _hip
    from transformers.models.llama.configuration_llama import LlamaConfig

    cfg = dict(tm.LLAMA, vocab_size=4000, hidden_size=512, intermediate_size=1024, num_attention_heads=heads,
               num_key_value_heads=kv_heads)
    dcfg = dict(tm.DRAFTER, vocab_size=4000, hidden_size=512, exit_dim=1024)
    # (the drafter mostly agrees with the LLM, whose attention counts for little)
    llama_sd, drafter_sd = tm.markov(41, llama_cfg=cfg, drafter_cfg=dcfg, mix=0.05)
    ids = tm.prompt(4, 60, cfg["vocab_size"], 5, [0, 31, 3, 50])
    streams, accepted = [], []
    for in_place in (True, False):
        llm = rd.modeling_llama.LlamaForCausalLM(LlamaConfig(**cfg))
        drafter = rd.modeling_drafter.Drafter(rd.configuration_drafter.DrafterConfig(**dcfg))
        llm.load_state_dict(llama_sd, strict=False)
        drafter.load_state_dict(drafter_sd)
        model = rd.RecurrentDrafting(llm.to(dtype).cuda().eval(), drafter.to(dtype).cuda().eval())
        model.kv_bits, model.kv_rows_in_place = bits, in_place
        torch.manual_seed(11)
        ledger = rd.stats.Ledger()
        _hip.timing_enable(True)
        try:
            streams.append([t.cpu().tolist() for t in model.generate(
                ledger, ids.cuda(), 60 + 48, rd.BeamShape(12, 5), rd.SamplingArgs(1.0, not sampling), rd.SpecialTokens(0, None))])
            torch.cuda.synchronize()
            ran = set(_hip.timing_collect())
        finally:
            _hip.timing_enable(False)
        assert {"attn_quant_kernel", "rope_append_quant_kernel", "attn_spans_kernel"} <= ran
        assert not ran & {"attn_quant_generic_kernel", "rope_append_kernel"}, ran
        accepted.append(max(ledger.records[0]["avg_num_accepted"]))
    assert streams[0] == streams[1] and len(streams[0]) > 3 and accepted[0] == accepted[1]
    assert accepted[0] > 0.2, "nothing was accepted: the rows never shifted"


# ---- rows that are not written ---------------------------------------------------------------------------

SENTINEL = 777.0


@pytest.mark.parametrize("batch,heads,kv_heads,n,prev,counts", [
    (2, 4, 2, 3, 60, [3, 1]),                                      # a wave's 16 rows
    (3, 4, 2, 40, 60, [40, 1, 17]),                                # two row blocks
    (1, 4, 4, 2, 5000, [1]),                                       # keys in pieces, joined by the merge
    (8, 32, 32, 250, 260, [250, 1, 33, 128, 129, 250, 31, 200])])  # eight waves side by side
@pytest.mark.parametrize("dtype,bits,dim", [(torch.bfloat16, 4, 128), (torch.float16, 8, 64), (torch.float32, 4, 32)])
def test_rows_behind_the_last_one_are_left_as_they_were(batch, heads, kv_heads, n, prev, counts, dtype, bits, dim):
    """A packed batch over the C ABI: rows of the output, and of the rotated queries, behind the last slot that exists,
    and the cache rows of slots that do not exist."""
    from recurrent_drafting_amd import _hip, attention
    from recurrent_drafting_amd.packed_rows import PackedRows

    if dtype == torch.float32 and n == 250:
        n, counts = 20, [20, 1, 3, 12, 19, 20, 11, 2]              # (the generic kernel has one layout)
    g = torch.Generator(device="cuda").manual_seed(n)
    total = sum(counts)
    rows = PackedRows.from_counts(torch.tensor(counts, dtype=torch.int32).cuda(), total, n)
    spare = rows.rows - total + 5
    cache = _new(batch, prev + n, kv_heads, dim, dtype, bits)
    for view in cache.sliced[0]:
        view.append(torch.randn(batch, kv_heads, prev, dim, generator=g, device="cuda").to(dtype))
    before = cache._cache.clone()
    lib, stream = _hip.lib(), _hip.stream()
    qkv = torch.randn(total + spare, (heads + 2 * kv_heads) * dim, generator=g, device="cuda").to(dtype)
    q, k, v = qkv.split([heads * dim, kv_heads * dim, kv_heads * dim], dim=1)
    cos, sin = torch.ones(1, dim, dtype=dtype, device="cuda"), torch.zeros(1, dim, dtype=dtype, device="cuda")
    positions = torch.zeros(batch, n, dtype=torch.long, device="cuda")
    turned = torch.full((total + spare, heads * dim), SENTINEL, dtype=dtype, device="cuda")
    two, three = C.c_int64 * 2, C.c_int64 * 3
    slab = cache._cache[0, 0].data_ptr(), cache._cache[0, 1].data_ptr()
    wide = two(0, qkv.stride(0))
    _hip.check(lib.rd_rope_append_quant(
        q.data_ptr(), wide, k.data_ptr(), wide, v.data_ptr(), wide, _hip.dtype_code(dtype), batch, n, heads, kv_heads, dim,
        cos.data_ptr(), sin.data_ptr(), 1, positions.data_ptr(), n, turned.data_ptr(), two(0, heads * dim), *slab,
        cache.byte_strides, bits, prev, prev + n, _hip.ptr(rows.row_start), None, stream))
    assert torch.equal(turned[:total], q[:total]) and (turned[total:] == SENTINEL).all()
    for b, c in enumerate(counts):
        assert torch.equal(cache._cache[0, :, b, :, :prev], before[0, :, b, :, :prev])
        assert (cache._cache[0, :, b, :, prev : prev + c] != before[0, :, b, :, prev : prev + c]).any()
        assert torch.equal(cache._cache[0, :, b, :, prev + c :], before[0, :, b, :, prev + c :])
    mask = torch.ones(batch, n, prev + n, dtype=torch.bool, device="cuda").tril(prev)
    prepared = attention.prepare(mask, n_heads=heads)
    spans = torch.empty(lib.rd_attn_spans_ints(batch, n), dtype=torch.int32, device="cuda")
    _hip.check(lib.rd_attn_spans(prepared.bits.data_ptr(), batch, n, prev + n, spans.data_ptr(), stream))
    need = lib.rd_verify_attention_quant_workspace_bytes(_hip.dtype_code(dtype), batch, heads, kv_heads, n, prev + n, dim)
    assert (need > 0) == (prev == 5000 and dtype != torch.float32)
    workspace = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
    out = torch.full((total + spare, heads * dim), SENTINEL, dtype=dtype, device="cuda")
    strides = three(0, dim, heads * dim)
    _hip.check(lib.rd_verify_attention_quant(
        turned.data_ptr(), strides, *slab, cache.byte_strides, bits, prev + n, out.data_ptr(), strides, _hip.dtype_code(dtype),
        batch, heads, kv_heads, n, prev + n, dim, dim ** -0.5, prepared.bits.data_ptr(), prepared.plan.data_ptr(),
        spans.data_ptr(), workspace.data_ptr(), need, 0, _hip.ptr(rows.row_start), stream))
    assert torch.isfinite(out[:total].float()).all() and not (out[:total] == SENTINEL).any()
    assert (out[total:] == SENTINEL).all()
