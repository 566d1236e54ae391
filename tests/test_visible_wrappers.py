"""What the torch wrappers of the visible-key attention calls refuse before anything is looked at on a device (no GPU)."""
import pytest
import torch

from fp8kv_amd import ops

T, D = 5, 128


def _calls():
    """(name, call taking q and out) of every visible-key attention call, with host tensors of one small batch."""
    kc = torch.zeros(1, 16, 2, D, dtype=torch.uint8)
    starts, lens, table = torch.tensor([0, T], dtype=torch.int32), torch.tensor([T], dtype=torch.int32), torch.zeros(1, 1, dtype=torch.int32)
    scales, one = torch.full((1, 1, 2, 2), 127, dtype=torch.uint8), torch.ones(1)
    b16 = kc.to(torch.bfloat16)
    yield "decode_window", lambda q, out: ops.decode_attention_window(q, kc, kc, out, starts, lens, table, one, one, 0.1, 4)
    yield "decode_window_bf16", lambda q, out: ops.decode_attention_window(q, b16, b16, out, starts, lens, table, None, None, 0.1, 4)
    yield "decode_blk", lambda q, out: ops.decode_attention_blk(q, kc, kc, out, starts, lens, table, scales, 0.1, max_seq_len=T)
    yield "prefill_window", lambda q, out: ops.prefill_attention_window(q, kc, kc, out, starts, lens, table, one, one, 0.1, 4, max_query_len=T)
    yield "prefill_window_bf16", lambda q, out: ops.prefill_attention_window(q, b16, b16, out, starts, lens, table, None, None, 0.1, 4,
                                                                             max_query_len=T)
    yield "prefill_blk", lambda q, out: ops.prefill_attention_blk(q, kc, kc, out, starts, lens, table, scales, 0.1, max_query_len=T)


@pytest.mark.parametrize("name", [n for n, _ in _calls()])
def test_out_with_fewer_rows_than_q_is_refused(name):
    """The kernels write every row of q in out: one row fewer would be a write past its end."""
    call = dict(_calls())[name]
    q = torch.zeros(T, 4, D, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="out has 4 rows, fewer than q's 5"):
        call(q, torch.zeros_like(q)[:T - 1])
    with pytest.raises(ValueError, match="out has 0 rows"):
        call(q, torch.zeros_like(q)[:0])
    for rows in (T, T + 3):                          # as many, and more: refused for being on the host alone
        with pytest.raises(ValueError, match="device tensor"):
            call(q, torch.zeros(rows, 4, D, dtype=torch.bfloat16))


def test_scratch_by_stream_and_by_capture(monkeypatch):
    """Eager calls of a stream share a zeroed buffer, which only grows; every capture has its own, whose tickets are zeroed
    within it; no two streams share one."""
    resets = []
    monkeypatch.setattr(ops, "_stream_scratch", {})
    monkeypatch.setattr(ops, "_capture_scratch", {})
    monkeypatch.setattr(ops, "decode_scratch_reset", resets.append)
    dev, least = torch.device("cpu", 0), ops.DECODE_SCRATCH_MIN_BYTES
    a, b = (ops._scratch_for(300 << 10, dev, s, 0) for s in (11, 12))
    assert a.data_ptr() != b.data_ptr() and a.numel() == b.numel() == least and int(a.sum()) == 0
    assert ops._scratch_for(least, dev, 11, 0) is a and ops._scratch_for(5, torch.device("cpu", 1), 11, 0) is not a
    grown = ops._scratch_for(least + 1, dev, 11, 0)
    assert grown.numel() >= 2 * least and int(grown.sum()) == 0 and ops._scratch_for(9, dev, 11, 0) is grown
    assert ops._scratch_for(9, dev, 12, 0) is b and resets == []
    first = ops._scratch_for(300 << 10, dev, 11, 1)
    assert first is not grown and ops._scratch_for(299 << 10, dev, 11, 1) is first
    assert [r.numel() for r in resets] == [256 << 10] and resets[0].data_ptr() == first.data_ptr()
    other, second = ops._scratch_for(300 << 10, dev, 12, 1), ops._scratch_for(300 << 10, dev, 11, 2)
    larger = ops._scratch_for(400 << 10, dev, 11, 2)
    assert len({x.data_ptr() for x in (first, other, second, larger)}) == 4 and larger.numel() == 400 << 10
    assert [r.data_ptr() for r in resets[1:]] == [other.data_ptr(), second.data_ptr(), larger.data_ptr()]
    assert ops._scratch_for(9, dev, 11, 0) is grown


def test_no_capture_without_a_stream(lib):
    assert lib.fp8kv_stream_capture(None) == 0
