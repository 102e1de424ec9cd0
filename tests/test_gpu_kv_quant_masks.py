"""Attention over a cache in 4 or 8 bits follows the mask bits that it finds: bits that a replay has written, bits
of a static buffer, bits written between two eager calls.  Every result has the bits of a call with a mask
prepared for it alone."""
import contextlib

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

KV, N, HEADS, KV_HEADS = 420, 35, 4, 2


def _setting(dtype=torch.bfloat16, bits=4, dim=128):
    """(layers of keys and values, queries, three masks: their spans, their fully attended runs and their trees
    differ)"""
    from recurrent_drafting_amd import kv_cache

    g = torch.Generator().manual_seed(dim + bits)
    cache = kv_cache.Cache(2, KV, 2, KV_HEADS, dim, dtype, torch.device("cuda"), bits=bits)
    for views in cache.sliced:
        for view in views:
            view.append(torch.randn(2, KV_HEADS, KV, dim, generator=g).to(dtype).cuda())
    q = torch.randn(2, HEADS, N, dim, generator=g).to(dtype).cuda()
    rng = np.random.default_rng(61)
    masks = []
    for pads, hole in [([0, 300], (0, 0)), ([200, 0], (96, 160)), ([64, 130], (320, 384))]:
        mask = np.zeros((2, N, KV), bool)
        for b in range(2):
            mask[b, :, pads[b] : KV - N] = True
            mask[b, :, hole[0] : hole[1]] = False
            up = np.eye(N, dtype=bool)
            for t in range(1, N):
                up[t] |= up[rng.integers(0, t)]
            mask[b, :, KV - N :] = up
        masks.append(torch.tensor(mask).cuda())
    return cache.sliced, q, masks


def _forward(layers, q, prepared):
    from recurrent_drafting_amd import attention

    return [attention.masked_attention(q, k.rows(), v.rows(), prepared) for k, v in layers]


def _wanted(layers, q, masks):
    from recurrent_drafting_amd import attention

    want = [[o.clone() for o in _forward(layers, q, attention.prepare(m, n_heads=HEADS))] for m in masks]
    assert not torch.equal(want[0][0], want[1][0]) and not torch.equal(want[1][0], want[2][0])
    return want


def _same(got, want):
    return all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("mode", [contextlib.nullcontext, torch.inference_mode])
@pytest.mark.parametrize("dtype,bits,dim", [(torch.bfloat16, 4, 128), (torch.float16, 8, 64), (torch.float32, 4, 32)])
def test_eager_calls_with_the_mask_of_a_replayed_graph(dtype, bits, dim, mode):
    """prepare and attention captured; after every replay with a new mask, eager calls with the same PreparedMask on
    two streams, and another capture on one that has seen eager calls."""
    from recurrent_drafting_amd import attention

    with mode():
        layers, q, masks = _setting(dtype, bits, dim)
        want = _wanted(layers, q, masks)
        static, stream = masks[0].clone(), torch.cuda.Stream()
        first = torch.cuda.CUDAGraph()
        with torch.cuda.graph(first, stream=stream):
            prepared = attention.prepare(static, n_heads=HEADS)
            outs = _forward(layers, q, prepared)
        for turn in (1, 2, 0, 1):
            static.copy_(masks[turn])
            first.replay()
            eager = _forward(layers, q, prepared)
            torch.cuda.synchronize()
            with torch.cuda.stream(stream):
                aside = _forward(layers, q, prepared)
            torch.cuda.synchronize()
            assert _same(outs, want[turn]) and _same(eager, want[turn]) and _same(aside, want[turn]), turn
        second = torch.cuda.CUDAGraph()
        with torch.cuda.graph(second, stream=stream):
            again = _forward(layers, q, prepared)
        for turn in (2, 0, 1, 2):
            static.copy_(masks[turn])
            first.replay()
            second.replay()
            torch.cuda.synchronize()
            assert _same(outs, want[turn]) and _same(again, want[turn]), turn


@pytest.mark.parametrize("mode", [contextlib.nullcontext, torch.inference_mode])
@pytest.mark.parametrize("dtype,bits,dim", [(torch.bfloat16, 4, 128), (torch.float16, 8, 64), (torch.float32, 4, 32)])
def test_static_bits_and_plan(dtype, bits, dim, mode):
    """Bits and plan copied into those of a mask that eager calls and a captured graph use: both follow them."""
    from recurrent_drafting_amd import attention

    with mode():
        layers, q, masks = _setting(dtype, bits, dim)
        want = _wanted(layers, q, masks)
        fresh = [attention.prepare(m, n_heads=HEADS) for m in masks]
        static = attention.prepare(masks[0], n_heads=HEADS)
        assert _same(_forward(layers, q, static), want[0])
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            assert _same(_forward(layers, q, static), want[0])  # (a table of this stream before the capture on it)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            outs = _forward(layers, q, static)
        for turn in (1, 2, 0, 1):
            static.bits.copy_(fresh[turn].bits)
            static.plan.copy_(fresh[turn].plan)
            graph.replay()
            eager = _forward(layers, q, static)
            torch.cuda.synchronize()
            assert _same(outs, want[turn]) and _same(eager, want[turn]), turn


def test_bits_copied_by_a_replay():
    """The copy itself is captured: torch counts it once, the replays are not counted."""
    from recurrent_drafting_amd import attention

    layers, q, masks = _setting()
    want = _wanted(layers, q, masks)
    fresh = [attention.prepare(m, n_heads=HEADS) for m in masks]
    static = attention.prepare(masks[0], n_heads=HEADS)
    source = fresh[0].bits.clone(), fresh[0].plan.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        before = _forward(layers, q, static)
        static.bits.copy_(source[0])
        static.plan.copy_(source[1])
        outs = _forward(layers, q, static)
    last = 0
    for turn in (1, 2, 0, 1):
        source[0].copy_(fresh[turn].bits)
        source[1].copy_(fresh[turn].plan)
        graph.replay()
        eager = _forward(layers, q, static)
        torch.cuda.synchronize()
        assert _same(before, want[last]) and _same(outs, want[turn]) and _same(eager, want[turn]), turn
        last = turn


def test_the_bits_alone_rewritten_inside_the_same_keys():
    """Another tree over the same keys: the plan stays as it is, the bits are enough."""
    from recurrent_drafting_amd import attention

    layers, q, masks = _setting()
    prepared = attention.prepare(masks[0], n_heads=HEADS)
    _forward(layers, q, prepared)
    for turn in range(3):
        mask = masks[0].clone()
        mask[:, 1:, KV - N] = False          # (nobody but the root attends to the root)
        mask[:, turn + 2, 310 : 330 + turn] = False
        prepared.bits.copy_(attention.prepare(mask, n_heads=HEADS).bits)
        want = _forward(layers, q, attention.prepare(mask, n_heads=HEADS))
        assert _same(_forward(layers, q, prepared), want), turn


def test_a_forward_writes_one_table():
    """The layers of a forward, and the calls behind it, share the table as long as nobody writes the bits."""
    from recurrent_drafting_amd import _hip, attention

    layers, q, masks = _setting()
    with torch.inference_mode():
        prepared = attention.prepare(masks[0], n_heads=HEADS)
        _forward(layers, q, prepared)
        (table, *_), = prepared.spans.values()
        _forward(layers, q, prepared)
        assert len(prepared.spans) == 1 and prepared.spans[_hip.stream()][0] is table
