"""GPU parity of the rotation-and-append calls against the 64-bit oracle.

Bounds: a rotated element is at most two products and a sum in fp32, so it is within
3 * 2^-24 * (|a| + |b|) of the formula on the same table values (|cos|, |sin| <= 1); storing rounds once:
bf16 by at most 2^-8 of the value, e4m3 by 2^-4 of it or half a subnormal step (2^-10 code units).
Bytes that no new token owns are compared for equality, scale bytes likewise.
"""
import numpy as np
import pytest
import torch

from fp8kv_amd import ops, workloads
from oracle import formats, rope_append

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
F32 = 3 * 2.0 ** -24


def _tokens(g, T, HQ, HKV, D, spread=1.0):
    """q, key, value as slices of one projection output [T, (HQ + 2 HKV) D] on the device."""
    qkv = torch.randn(T, (HQ + 2 * HKV) * D, generator=g)
    qkv *= torch.exp(spread * torch.randn(T, 1, generator=g))
    qkv = qkv.to(torch.bfloat16).to(DEV)
    cut = lambda a, b: qkv[:, a * D:b * D].view(T, b - a, D)  # noqa: E731
    return cut(0, HQ), cut(HQ, HQ + HKV), cut(HQ + HKV, HQ + 2 * HKV)


def _f64(t):
    return t.detach().float().cpu().numpy().astype(np.float64)


def _room(x):
    """Bound on the fp32 error of rotated elements: any pair partner is at most the head's largest."""
    return F32 * 2 * np.abs(x).max(-1, keepdims=True) * np.ones_like(x)


def _pool(g, layout, NB, PBLK, HKV, D, dtype):
    if dtype == "bf16":
        kv = torch.randn(NB, HKV, PBLK, 2 * D, generator=g).to(torch.bfloat16).to(DEV)
    else:
        kv = torch.randint(0, 256, (NB, HKV, PBLK, 2 * D), dtype=torch.uint8, generator=g)
        kv[(kv & 0x7F) == 0x7F] = 0x10
        kv = kv.to(DEV)
    if layout == "engine":
        return workloads.engine_views(kv, D)
    k, v = workloads.engine_views(kv, D)
    return k.clone(memory_format=torch.contiguous_format), v.clone(memory_format=torch.contiguous_format)


def _bytes(t):
    return t.view(torch.uint8 if t.dtype != torch.bfloat16 else torch.int16).cpu().numpy().copy()


@pytest.mark.parametrize("dtype", ["fp8", "bf16"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("D,rot,table", [(128, 128, torch.float32), (128, 64, torch.bfloat16), (96, 16, torch.float32),
                                         (64, 48, torch.float32), (16, 16, torch.bfloat16)])
@pytest.mark.parametrize("layout,PBLK", [("engine", 16), ("standalone", 32)])
def test_rotate_and_append(dtype, interleaved, D, rot, table, layout, PBLK):
    g = torch.Generator().manual_seed(D + rot)
    T, HQ, HKV, NB = 37, 6, 2, 9
    q, key, value = _tokens(g, T, HQ, HKV, D)
    kc, vc = _pool(g, layout, NB, PBLK, HKV, D, dtype)
    cos_sin = ops.rope_table(5000, rot, DEV, dtype=table)
    pos = torch.randint(0, 5000, (T,), generator=g)
    slots = torch.randperm(NB * PBLK, generator=g)[:T].to(torch.int64)
    slots[::5] = -1
    slots[3] = NB * PBLK                                   # past the cache: skipped
    ks, vs = 0.037, 0.02
    before = _bytes(kc), _bytes(vc)
    out = ops.rope_append(q, key, value, kc, vc, pos.to(DEV), cos_sin, slots.to(DEV), ks, vs, interleaved=interleaved)
    torch.cuda.synchronize()
    tab = _f64(cos_sin)
    want = rope_append.rotate(_f64(q), pos.numpy(), tab, interleaved)
    assert (np.abs(_f64(out) - want) <= 2.0 ** -8 * np.abs(want) + _room(_f64(q))).all()
    for x, (cache, src, scale) in enumerate(((kc, key, ks), (vc, value, vs))):
        y = rope_append.rotate(_f64(src), pos.numpy(), None if x else tab, interleaved)
        room = 0 * y if x else _room(_f64(src))
        now = _bytes(cache)
        live = [(t, int(s)) for t, s in enumerate(slots) if 0 <= s < NB * PBLK]
        for t, s in live:
            row = now[s // PBLK, s % PBLK]
            if dtype == "bf16":
                got = _f64(torch.from_numpy(row.copy()).view(torch.bfloat16))
                assert (np.abs(got - y[t]) <= 2.0 ** -8 * np.abs(y[t]) + room[t]).all()
            else:
                f = float(np.float32(scale))
                got = formats.e4m3fn_table()[row]
                z = np.clip(y[t] / f, -448, 448)
                assert (np.abs(got - z) <= np.maximum(2.0 ** -4 * np.abs(z), 2.0 ** -10) + room[t] / f + 2.0 ** -23 * np.abs(z)).all()
            before[x][s // PBLK, s % PBLK] = row
        assert np.array_equal(now, before[x])              # nothing else moved


def test_without_rotation_the_bytes_are_those_of_cache_write():
    """Every bf16 pattern (NaN, infinities, subnormals), no table: the codes of ops.cache_write."""
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    T, HKV, D = 128, 4, 128
    key, value = bits.view(T, HKV, D).to(DEV), bits.flip(0).view(T, HKV, D).to(DEV)
    slots = torch.randperm(T, generator=torch.Generator().manual_seed(1)).to(DEV)
    a = [torch.zeros(T // 16, 16, HKV, D, dtype=torch.uint8, device=DEV) for _ in range(4)]
    ops.cache_write(key, value, a[0], a[1], slots, 0.0123, 3.7)
    assert ops.rope_append(None, key, value, a[2], a[3], None, None, slots, 0.0123, 3.7) is None
    assert torch.equal(a[0], a[2]) and torch.equal(a[1], a[3])
    b = [torch.zeros(T // 16, 16, HKV, D, dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    ops.rope_append(None, key, value, *b, None, None, slots)
    got = b[0].view(T, HKV, D)[slots].view(torch.int16)
    assert torch.equal(got[~key.isnan()], key.view(torch.int16)[~key.isnan()])
    assert b[0].view(T, HKV, D)[slots][key.isnan()].isnan().all()


def test_positions_outside_the_table_give_nan_only_there():
    g = torch.Generator().manual_seed(3)
    T, HQ, HKV, D, rot = 6, 2, 1, 128, 64
    q, key, value = _tokens(g, T, HQ, HKV, D)
    kc, vc = _pool(g, "standalone", 1, 16, HKV, D, "bf16")
    pos = torch.tensor([0, -1, 9, 10, 1 << 40, -(1 << 40)])
    cos_sin = ops.rope_table(10, rot, DEV)
    out = ops.rope_append(q, key, value, kc, vc, pos.to(DEV), cos_sin, torch.arange(T, device=DEV))
    bad = [1, 3, 4, 5]
    assert out[bad][..., :rot].isnan().all() and kc[0, bad][..., :rot].isnan().all()
    assert not out[[0, 2]].isnan().any() and not kc[0, [0, 2]].isnan().any()
    assert torch.equal(out[..., rot:], q[..., rot:]) and torch.equal(vc[0, :T], value)
    assert torch.equal(out[0], q[0])                       # position 0 turns nothing


def test_far_positions():
    """Angles of far positions come from the table, whose error is one rounding at any position."""
    pos = torch.tensor([0, 1, 131071, 1048575])
    tab = ops.rope_table(1 << 20, 128, DEV)[pos.to(DEV)].cpu().double()
    freq = 10000.0 ** (-np.arange(0, 128, 2) / 128)
    ang = pos.numpy()[:, None] * freq
    assert np.abs(tab.numpy() - np.concatenate([np.cos(ang), np.sin(ang)], 1)).max() <= 2.0 ** -24 + 1e-9


def test_in_place_and_single_token_with_odd_strides():
    g = torch.Generator().manual_seed(5)
    T, HQ, HKV, D = 19, 4, 2, 128
    q, key, value = _tokens(g, T, HQ, HKV, D)
    cos_sin = ops.rope_table(64, D, DEV)
    pos = torch.arange(T, device=DEV)
    kc, vc = _pool(g, "engine", 2, 16, HKV, D, "fp8")
    want = ops.rope_append(q.contiguous(), key, value, kc, vc, pos, cos_sin, pos, 0.1, 0.1)
    k1 = _bytes(kc)
    assert ops.rope_append(q, key, value, kc, vc, pos, cos_sin, pos, 0.1, 0.1, q_out=q) is q
    assert torch.equal(q, want) and np.array_equal(_bytes(kc), k1)
    # one token as [1, H, D] with a row stride that says nothing
    one = lambda t: t[:1].contiguous().as_strided((1, HKV, D), (8, D, 1))  # noqa: E731
    k0, v0 = one(key), one(value)
    assert k0.stride(0) == 8
    kc2, vc2 = _pool(g, "engine", 2, 16, HKV, D, "fp8")
    ops.rope_append(None, k0, v0, kc2, vc2, pos[:1], cos_sin, pos[:1], 0.1, 0.1)
    assert torch.equal(kc2[0, 0].view(torch.uint8), kc[0, 0].view(torch.uint8))
    empty = key[:0]
    assert ops.rope_append(q[:0], empty, empty, kc, vc, pos[:0], cos_sin, pos[:0], 0.1, 0.1).shape == (0, HQ, D)


# ---- block-scaled caches -------------------------------------------------------------------------

def _blk_case(g, lens, HQ, HKV, PBLK, layout="engine", spread=1.0, extra_rows=0):
    """lens: (earlier tokens, new tokens) of each sequence."""
    D = 128
    need = [max(0, -(-(a + b) // PBLK)) for a, b in lens]
    NB = sum(need) + 2
    table = torch.full((len(lens), max(need + [1])), -7, dtype=torch.int32)
    ids = torch.randperm(NB, generator=g).to(torch.int32)
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = ids[at:at + n]
        at += n
    starts = torch.tensor([0] + list(np.cumsum([b for _, b in lens])), dtype=torch.int32)
    T = int(starts[-1]) + extra_rows
    q, key, value = _tokens(g, T, HQ, HKV, D, spread)
    kc, vc = _pool(g, layout, NB, PBLK, HKV, D, "fp8")
    scales = torch.randint(110, 126, (NB, PBLK // 16, HKV, 2), dtype=torch.uint8, generator=g).to(DEV)
    pos = torch.zeros(T, dtype=torch.int64)
    for s, (a, b) in enumerate(lens):
        pos[int(starts[s]):int(starts[s]) + b] = torch.arange(a, a + b)
    return dict(q=q, key=key, value=value, kc=kc, vc=vc, scales=scales, pos=pos.clamp(min=0), starts=starts,
                seq_lens=torch.tensor([a + b for a, b in lens], dtype=torch.int32), table=table, PBLK=PBLK, T=T)


def _blk_run(c, cos_sin, interleaved=False, q_out=None):
    return ops.rope_append_blk(c["q"], c["key"], c["value"], c["kc"], c["vc"], c["scales"], c["pos"].to(DEV), cos_sin,
                               c["starts"].to(DEV), c["seq_lens"].to(DEV), c["table"].to(DEV), q_out=q_out,
                               interleaved=interleaved)


def _blk_check(c, cos_sin, interleaved=False):
    before = _bytes(c["kc"]), _bytes(c["vc"]), c["scales"].cpu().numpy().copy()
    fill = torch.full_like(c["q"].contiguous(), 7.0)
    out = _blk_run(c, cos_sin, interleaved, fill)
    torch.cuda.synchronize()
    tab = None if cos_sin is None else _f64(cos_sin)
    live = int(c["starts"][-1])
    want = rope_append.rotate(_f64(c["q"]), c["pos"].numpy(), tab, interleaved)
    tol = 2.0 ** -8 * np.abs(want) + _room(_f64(c["q"]))
    assert (np.abs(_f64(out) - want) <= tol)[:live].all() and (out[live:] == 7.0).all()
    key = rope_append.rotate(_f64(c["key"]), c["pos"].numpy(), tab, interleaved)
    k, v, sc = rope_append.append_blk(key, _f64(c["value"]), *before, c["starts"].numpy(), c["seq_lens"].numpy(),
                                      c["table"].numpy(), c["PBLK"])
    assert np.array_equal(c["scales"].cpu().numpy(), sc)
    dec = formats.e4m3fn_table()
    # V takes no arithmetic before its rounding: equal.  K may fall on the other side of a rounding tie by its fp32 error.
    got_v = dec[_bytes(c["vc"])]
    assert np.array_equal(got_v, v, equal_nan=True)
    got_k = dec[_bytes(c["kc"])]
    if cos_sin is None:
        assert np.array_equal(got_k, k, equal_nan=True)
    else:
        off = np.abs(got_k - k)
        assert (off <= np.maximum(2.0 ** -3 * np.abs(k), 2.0 ** -9)).all() and (off > 0).mean() < 1e-4


LENS = {
    "fresh": [(0, 1), (0, 16), (0, 17), (0, 33)],
    "inside_a_group": [(5, 3), (15, 1), (1, 14), (3, 200), (31, 2)],
    "at_borders": [(16, 16), (32, 1), (15, 17), (48, 31)],
    "empty_between": [(0, 0), (20, 0), (7, 1), (0, 0), (9, 40), (100, 0)],
    "fewer_tokens_than_new_rows": [(-3, 5), (0, 2), (-20, 18), (-1, 1)],
}


@pytest.mark.parametrize("lens", LENS.values(), ids=LENS.keys())
@pytest.mark.parametrize("PBLK", [16, 64])
@pytest.mark.parametrize("interleaved,rot", [(False, 128), (True, 32)])
def test_blk_append(lens, PBLK, interleaved, rot):
    g = torch.Generator().manual_seed(len(lens) + PBLK)
    c = _blk_case(g, lens, 6, 2, PBLK, extra_rows=3)
    _blk_check(c, ops.rope_table(400, rot, DEV), interleaved)


@pytest.mark.parametrize("NS", [1, 63, 64, 65, 200])
def test_blk_many_sequences(NS):
    """Decode batches and mixed ones past one probe of the sequence search."""
    g = torch.Generator().manual_seed(NS)
    n = torch.randint(0, 4, (NS,), generator=g).tolist()
    a = torch.randint(0, 60, (NS,), generator=g).tolist()
    c = _blk_case(g, list(zip(a, n if NS > 64 else [1] * NS)), 2, 1, 16)
    _blk_check(c, ops.rope_table(100, 128, DEV))


def test_blk_search_past_two_probes():
    g = torch.Generator().manual_seed(9)
    lens = [(i % 23, 1 if i % 3 == 0 else 0) for i in range(4200)]
    c = _blk_case(g, lens, 1, 1, 16)
    _blk_check(c, None)


@pytest.mark.parametrize("layout", ["engine", "standalone"])
def test_blk_growing_scale_rerounds_earlier_tokens_once(layout):
    """Token by token with growing norms: each step equals the oracle's step on the bytes before it."""
    g = torch.Generator().manual_seed(11)
    D, HKV = 128, 2
    c = _blk_case(g, [(0, 1)], 2, HKV, 16, layout)
    for t in range(20):
        step = dict(c, **{k: v for k, v in _blk_case(g, [(t, 1)], 2, HKV, 32, layout, 2.0).items() if k in ("q", "key", "value", "pos", "starts", "seq_lens")})
        step["table"] = torch.tensor([[0, 1]], dtype=torch.int32)
        _blk_check(step, None)


def test_blk_non_finite_rows_and_zeros():
    g = torch.Generator().manual_seed(12)
    c = _blk_case(g, [(0, 16), (4, 12), (0, 16), (2, 3)], 2, 1, 16)
    key, value = c["key"], c["value"]
    key[3, 0, 5] = float("nan")
    key[4, 0, 6] = float("inf")
    value[20, 0, 0:8] = float("-inf")
    value[28:44] = 0.0                                      # a whole group of zeros: the smallest scale
    key[44:47] = float("nan")                               # no finite element beside earlier tokens
    _blk_check(c, None)
    part = c["scales"][int(c["table"][2, 0]), 0, 0, 1]
    assert int(part) == 127 - 100


def test_blk_bad_blocks_are_skipped():
    """Block ids outside the cache and columns past the table write nothing."""
    g = torch.Generator().manual_seed(13)
    c = _blk_case(g, [(0, 40), (10, 20), (0, 5)], 2, 2, 16)
    c["table"][0, 1] = -1
    c["table"][1, 1] = 1 << 30
    c["table"][2, 0] = c["kc"].shape[0]
    c["table"] = c["table"][:, :2].contiguous()
    _blk_check(c, ops.rope_table(64, 128, DEV))


def test_on_another_stream_and_in_a_graph():
    g = torch.Generator().manual_seed(14)
    cos_sin = ops.rope_table(256, 128, DEV)
    c = _blk_case(g, [(5, 30), (100, 1), (0, 17)], 4, 2, 16)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _blk_check(c, cos_sin)
    torch.cuda.current_stream().wait_stream(side)

    dev = {k: c[k].to(DEV) for k in ("starts", "seq_lens", "table", "pos")}
    kc, vc = _pool(g, "engine", c["kc"].shape[0], 16, 2, 128, "fp8")
    q_out = torch.empty_like(c["q"].contiguous())

    def call(k, v, sc, out):
        return ops.rope_append_blk(c["q"], c["key"], c["value"], k, v, sc, dev["pos"], cos_sin, dev["starts"],
                                   dev["seq_lens"], dev["table"], q_out=out)
    scales = c["scales"].clone()
    call(kc, vc, scales, q_out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(kc, vc, scales, q_out)
    for i in range(4):
        c["key"].copy_(torch.randn_like(c["key"].float()) * (3.0 ** i))
        c["q"].mul_(1.25)
        k2, v2, s2 = kc.clone(), vc.clone(), scales.clone()
        want = call(k2, v2, s2, torch.empty_like(q_out))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(q_out, want) and torch.equal(scales, s2)
        assert torch.equal(kc.view(torch.uint8), k2.view(torch.uint8))
        assert torch.equal(vc.view(torch.uint8), v2.view(torch.uint8))


def test_refusals():
    T, HQ, HKV, D = 4, 4, 2, 128
    q = torch.zeros(T, HQ, D, dtype=torch.bfloat16, device=DEV)
    k = torch.zeros(T, HKV, D, dtype=torch.bfloat16, device=DEV)
    kc = torch.zeros(2, 16, HKV, D, dtype=torch.uint8, device=DEV)
    sc = torch.zeros(2, 1, HKV, 2, dtype=torch.uint8, device=DEV)
    pos = torch.arange(T, device=DEV)
    tab = ops.rope_table(8, D, DEV)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    seqs = (i32(0, T), i32(T), i32(0).view(1, 1))
    ok = ops.rope_append(q, k, k, kc, kc.clone(), pos, tab, pos, 1.0, 1.0)
    assert ok.shape == q.shape
    for bad in (
        lambda: ops.rope_append(q, k, k, kc, kc, pos, tab, pos),                                # no scales
        lambda: ops.rope_append(q.half(), k, k, kc, kc, pos, tab, pos, 1.0, 1.0),
        lambda: ops.rope_append(q[:3], k, k, kc, kc, pos, tab, pos, 1.0, 1.0),
        lambda: ops.rope_append(q, k, k[:, :1], kc, kc, pos, tab, pos, 1.0, 1.0),
        lambda: ops.rope_append(q, k, k, kc, kc[:, :, :1], pos, tab, pos, 1.0, 1.0),
        lambda: ops.rope_append(q, k, k, kc, kc, pos.int(), tab, pos, 1.0, 1.0),
        lambda: ops.rope_append(q, k, k, kc, kc, None, tab, pos, 1.0, 1.0),
        lambda: ops.rope_append(q, k, k, kc, kc, pos, tab.double(), pos, 1.0, 1.0),
        lambda: ops.rope_append(q, k, k, kc, kc, pos, tab, pos[:3], 1.0, 1.0),
        lambda: ops.rope_append(None, k, k, kc, kc, pos, tab, pos, 1.0, 1.0, q_out=q),
        lambda: ops.rope_append_blk(q, k, k, kc, kc, sc[:1], pos, tab, *seqs),
        lambda: ops.rope_append_blk(q, k, k, kc, kc, sc.float(), pos, tab, *seqs),
        lambda: ops.rope_append_blk(q, k, k, kc, kc, sc, pos, tab, seqs[0][:1], *seqs[1:]),
        lambda: ops.rope_append_blk(q, k, k, kc, kc, sc, pos, tab, seqs[0], seqs[1].long(), seqs[2]),
    ):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(Exception, match="status 2"):       # an odd rotary width
        ops.rope_append(q, k, k, kc, kc, pos, tab[:, :20], pos, 1.0, 1.0)
