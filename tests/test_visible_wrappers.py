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
