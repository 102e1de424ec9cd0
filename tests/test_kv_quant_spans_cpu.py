"""When the span table of a prepared mask is written anew and when an earlier one is read again: the host's
decision, with a stand-in for the library that counts the launches."""
import contextlib
import dataclasses

import pytest
import torch


class _Library:
    def __init__(self):
        self.capture, self.launches = 0, 0

    def rd_stream_capture_id(self, stream):
        return self.capture if stream else 0

    def rd_attn_bits_words(self, batch, n_q, kv_len):
        return batch * n_q * -(-kv_len // 64)

    def rd_attn_plan_ints(self, batch, n_q, kv_len):
        return 64

    def rd_attn_prepare(self, *_):
        return 0

    def rd_attn_spans_ints(self, batch, n_q):
        return 4 * batch * -(-n_q // 16)

    def rd_attn_spans(self, *_):
        self.launches += 1
        return 0


@pytest.fixture
def lib(monkeypatch):
    from recurrent_drafting_amd import _hip

    stand_in = _Library()
    stand_in.stream = 0
    monkeypatch.setattr(_hip, "lib", lambda: stand_in)
    monkeypatch.setattr(_hip, "stream", lambda: stand_in.stream)
    monkeypatch.setattr(_hip, "ptr", lambda t: None if t is None else t.data_ptr())
    monkeypatch.setattr(_hip, "check", lambda rc: None)
    return stand_in


def _prepare():
    from recurrent_drafting_amd import attention

    return attention.prepare(torch.ones(2, 3, 70, dtype=torch.bool))


def _use(lib, prepared, stream=0):
    """(launches of this use, its table)"""
    from recurrent_drafting_amd import attention

    before = lib.launches
    table = attention._spans(prepared, stream)
    return lib.launches - before, table


MODES = [contextlib.nullcontext, torch.inference_mode]


@pytest.mark.parametrize("mode", MODES)
def test_the_layers_of_a_forward_share_a_table(lib, mode):
    with mode():
        prepared = _prepare()
        launches, table = _use(lib, prepared)
        assert launches == 1 and table.numel() == 8
        for _ in range(3):
            again, same = _use(lib, prepared)
            assert again == 0 and same is table
        assert _use(lib, prepared, stream=7)[0] == 1 and _use(lib, prepared, stream=7)[0] == 0  # a table per stream
        assert _use(lib, _prepare())[0] == 1


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("write", ["copy", "fill", "item", "view", "out"])
def test_written_bits_are_read_anew_by_every_call(lib, write, mode):
    """Bits that anyone has written since `prepare` may be a static buffer, which replays write too: no table
    of theirs is kept."""
    with mode():
        prepared = _prepare()
        _use(lib, prepared)
        if write == "copy":
            prepared.bits.copy_(torch.ones_like(prepared.bits))
        elif write == "fill":
            prepared.bits.fill_(5)
        elif write == "item":
            prepared.bits[1, 2, 0] = 3
        elif write == "view":
            prepared.bits.view(-1)[:4].zero_()
        else:
            torch.add(prepared.bits, 1, out=prepared.bits)
        assert [_use(lib, prepared)[0] for _ in range(3)] == [1, 1, 1]


@pytest.mark.parametrize("mode", MODES)
def test_bits_of_a_capture_are_read_anew_by_every_eager_call(lib, mode):
    """A mask prepared inside a capture is written by every replay."""
    with mode():
        lib.stream, lib.capture = 7, 3
        prepared = _prepare()
        assert [_use(lib, prepared, 7)[0] for _ in range(3)] == [1, 0, 0]  # the layers of the capture
        lib.capture = 0
        assert [_use(lib, prepared, 7)[0] for _ in range(3)] == [1, 1, 1]
        lib.stream = 0
        assert [_use(lib, prepared, 0)[0] for _ in range(2)] == [1, 1]


def test_a_capture_writes_its_own_table(lib):
    """Never one that an eager call or another capture has written: a replay follows the bits it finds."""
    prepared = _prepare()
    _, eager = _use(lib, prepared, 7)
    tables = [eager]
    for capture in (11, 12):
        lib.capture = capture
        launches, table = _use(lib, prepared, 7)
        assert launches == 1 and all(table is not t for t in tables)
        assert _use(lib, prepared, 7) == (0, table)
        tables.append(table)
    prepared.bits.fill_(1)  # between two layers of the capture
    assert _use(lib, prepared, 7)[0] == 1
    lib.capture = 0
    assert [_use(lib, prepared, 7)[0] for _ in range(2)] == [1, 1]


def test_other_bits_and_masks_put_together_by_hand(lib):
    from recurrent_drafting_amd import attention

    prepared = _prepare()
    _use(lib, prepared)
    other = dataclasses.replace(prepared, bits=prepared.bits.clone())
    assert [_use(lib, other)[0] for _ in range(2)] == [1, 1] and _use(lib, prepared)[0] == 1
    assert _use(lib, prepared)[0] == 0
    prepared.bits = prepared.bits.clone()
    assert [_use(lib, prepared)[0] for _ in range(2)] == [1, 1]
    mine = attention.PreparedMask(other.bits, other.plan, 2, 3, 70)
    assert [_use(lib, mine)[0] for _ in range(2)] == [1, 1]
    with torch.inference_mode():
        mine = attention.PreparedMask(torch.zeros(2, 3, 2, dtype=torch.long), other.plan, 2, 3, 70)  # (no version to go by)
        assert [_use(lib, mine)[0] for _ in range(2)] == [1, 1]
