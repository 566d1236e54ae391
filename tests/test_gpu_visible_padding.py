"""Decode over visible keys of batches padded with sequences that own no row of q (query_start_loc does not move): they
write none of out."""
import pytest
import torch

from test_gpu_visible import KINDS, LONG, _case, _oracle, _run, _tolerance

pytestmark = pytest.mark.gpu

CUTS = {"one": dict(num_splits=1), "five": dict(num_splits=5), "forty": dict(num_splits=40),
        "parts": dict(num_splits=40, max_seq_len=LONG), "two_parts": dict(num_splits=2, max_seq_len=LONG)}
# (tokens, owns a row)
BATCHES = {"between": [(700, 1), (40, 0), (64, 1), (333, 1), (17, 0), (0, 0)], "first": [(90, 0), (0, 0), (500, 1), (3, 1)],
           "all": [(30, 0), (0, 0)], "long_without": [(10, 1), (6000, 0), (20, 1)],
           "padded": [(100 + 37 * i, 1) for i in range(9)] + [(0, 0)] * 60}


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("cut", CUTS.values(), ids=CUTS.keys())
@pytest.mark.parametrize("batch", BATCHES.values(), ids=BATCHES.keys())
def test_decode_of_sequences_without_a_row(kind, cut, batch):
    for window, sinks in ((0, 0), (200, 20)):
        c = _case(kind, [(n - 1, 1) for n, _ in batch], 8, 2, 16, window, sinks, seed=37)
        owners = [i for i, (_, own) in enumerate(batch) if own]
        want, *bounds = _oracle(c)
        tol = _tolerance(c, "decode", want, *bounds)[owners]
        owns = torch.tensor([own for _, own in batch])
        c["starts"] = torch.cat([torch.zeros(1, dtype=torch.int64), owns.cumsum(0)]).to(torch.int32)
        c["q"] = torch.cat([c["q"][owners], c["q"][:2]])              # two rows behind the last sequence
        for i, (_, own) in enumerate(batch):
            if not own:
                c["table"][i] = 0                                     # the block of NaN
        got = _run(c, "decode", **cut).double()
        assert ((got[:len(owners)] - want[owners]).abs() <= tol).all()
        assert (got[len(owners):] == 7).all()
