"""Decode over visible keys, several calls at once with the scratch that the wrappers choose: on two streams, in graphs
replayed beside one another, and eager beside them.  Every output equals that of the same call by itself, bit for bit (a
call's merges have a fixed order)."""
import math

import pytest
import torch

from fp8kv_amd import _lib, ops, workloads

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
D = 128


class Batch:
    """Sequences of `lens` over a block-scaled cache, and the call on it."""

    def __init__(self, lens, HQ, HKV, seed, **call):
        g = torch.Generator(device=DEV).manual_seed(seed)
        blocks = [-(-n // 16) for n in lens]
        pool = torch.randint(0, 0x78, (sum(blocks), HKV, 16, 2 * D), dtype=torch.uint8, device=DEV, generator=g)
        self.k, self.v = workloads.engine_views(pool, D)
        self.scales = torch.randint(110, 121, (sum(blocks), 1, HKV, 2), dtype=torch.uint8, device=DEV, generator=g)
        self.table = torch.zeros(len(lens), max(blocks), dtype=torch.int32, device=DEV)
        at = 0
        for s, n in enumerate(blocks):
            self.table[s, :n] = torch.arange(at, at + n)
            at += n
        self.lens = torch.tensor(lens, dtype=torch.int32, device=DEV)
        self.starts = torch.arange(len(lens) + 1, dtype=torch.int32, device=DEV)
        self.q = torch.randn(len(lens), HQ, D, device=DEV, generator=g).to(torch.bfloat16)
        self.call = dict(call)

    def run(self, out=None, **more):
        out = torch.full_like(self.q, 7.0) if out is None else out
        return ops.decode_attention_blk(self.q, self.k, self.v, out, self.starts, self.lens, self.table, self.scales,
                                        1 / math.sqrt(D), **self.call, **more)

    def alone(self):
        need = ops.decode_scratch_bytes(self.q.shape[0], self.q.shape[1], self.k.shape[2], 256)
        got = self.run(scratch=torch.zeros(need, dtype=torch.uint8, device=DEV))
        torch.cuda.synchronize()
        assert got.isfinite().all() and (got != 7).any()
        return got


def _batches():
    # splits of each sequence, parts of the batch, and a window: three layouts of records over the same scratch bytes
    return [Batch([4000 - 100 * i for i in range(16)], 16, 4, 1, num_splits=16, max_seq_len=4000),
            Batch([5000, 30, 700, 3000, 9000, 1], 8, 2, 2, num_splits=40, max_seq_len=1 << 24),
            Batch([300 * (i + 1) for i in range(12)], 24, 4, 3, num_splits=9, window=900, sinks=20)]


def test_streams_at_once():
    batches = _batches()
    want = [b.alone() for b in batches]
    streams = [torch.cuda.Stream() for _ in range(3)]
    for turn in range(4):
        outs = [[torch.empty_like(b.q) for _ in range(8)] for b in batches]
        torch.cuda.synchronize()
        for i in range(8):
            for j, s in enumerate(streams):
                with torch.cuda.stream(s):
                    b = (j + turn) % 3
                    batches[b].run(outs[b][i])
        torch.cuda.synchronize()
        for b in range(3):
            assert all(torch.equal(o, want[b]) for o in outs[b]), (turn, b)


def test_graphs_replayed_at_once_beside_eager_calls():
    """Graphs captured one after the other on one stream, with no call before the first."""
    batches = _batches()
    want = [b.alone() for b in batches]
    side = torch.cuda.Stream()
    graphs, outs = [], []
    for b in batches:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs.append([b.run(torch.empty_like(b.q)) for _ in range(6)])
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in range(3)]
    for turn in range(4):
        for o in sum(outs, []):
            o.fill_(7.0)
        eager = [torch.empty_like(batches[turn % 3].q) for _ in range(8)]
        torch.cuda.synchronize()
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
        with torch.cuda.stream(side):                     # the stream that they were captured on
            for e in eager:
                batches[turn % 3].run(e)
        torch.cuda.synchronize()
        for b in range(3):
            assert all(torch.equal(o, want[b]) for o in outs[b]), (turn, b)
        assert all(torch.equal(e, want[turn % 3]) for e in eager), turn


def test_a_fork_inside_a_capture():
    """Two streams of one capture run at once when it is replayed."""
    batches = _batches()[:2]
    want = [b.alone() for b in batches]
    side, other = torch.cuda.Stream(), torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        other.wait_stream(side)
        first = [batches[0].run(torch.empty_like(batches[0].q)) for _ in range(5)]
        with torch.cuda.stream(other):
            second = [batches[1].run(torch.empty_like(batches[1].q)) for _ in range(5)]
        side.wait_stream(other)
    for turn in range(3):
        for o in first + second:
            o.fill_(7.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, want[0]) for o in first), turn
        assert all(torch.equal(o, want[1]) for o in second), turn


def test_capture_numbers():
    """0 outside of a capture, the same number within one, another one for the next."""
    lib = _lib.load()
    side = torch.cuda.Stream()
    assert lib.fp8kv_stream_capture(None) == 0 and lib.fp8kv_stream_capture(side.cuda_stream) == 0
    seen = []
    x = torch.zeros(8, device=DEV)
    for _ in range(3):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            a = lib.fp8kv_stream_capture(torch.cuda.current_stream().cuda_stream)
            x.add_(1)
            b = lib.fp8kv_stream_capture(torch.cuda.current_stream().cuda_stream)
        assert a == b != 0
        seen.append(a)
    assert len(set(seen)) == 3 and lib.fp8kv_stream_capture(side.cuda_stream) == 0


def test_graphs_come_and_go():
    """Graphs that are dropped, one that stays, a shared pool, and eager calls between: a capture's scratch is its graph's."""
    batches = _batches()
    want = [b.alone() for b in batches]
    kept = torch.cuda.CUDAGraph()
    with torch.cuda.graph(kept):
        kept_out = [b.run(torch.empty_like(b.q)) for b in batches]          # each needs another size of scratch
    for i in range(6):
        graph = torch.cuda.CUDAGraph()
        b = i % 3
        with torch.cuda.graph(graph, pool=kept.pool() if i % 2 else None):
            out = batches[b].run(torch.empty_like(batches[b].q))
            wide = torch.full((1 << 20,), 3.0, device=DEV)                  # other memory of the graph's
            again = batches[b].run(torch.empty_like(batches[b].q))
        for _ in range(2):
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want[b]) and torch.equal(again, want[b]) and (wide == 3).all()
            assert torch.equal(batches[(b + 1) % 3].run(), want[(b + 1) % 3])
        del graph, out, wide, again
        if i % 2:
            torch.cuda.empty_cache()
        for o in kept_out:
            o.fill_(7.0)
        kept.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(kept_out, want)), i
