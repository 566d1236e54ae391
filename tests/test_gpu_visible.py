"""GPU parity of windowed attention and of attention over block-scaled caches against the 64-bit oracle.

Bound of an output element o = sum w v: its bf16 rounding, 2^-8 |o|, and on the weights, times sum w |v|:
  * their rounding in P.V: 2^-16 (decode, two bf16 parts of 8 bits each) or twice 2^-8 (prefill: bf16, the weight
    and, as the sum is that of the rounded weights, the sum);
  * the scores' fp32 error: 128 products and the k-parts' sums, at most 140 * 2^-24 of sum |q k|, twice (weight and
    sum of weights), the split query's 2^-22 included, and exp2 and the running sums, some 2^-20.
Every slot that no query sees holds NaN, and block-table entries of blocks that none needs point to a block of NaN.
"""
import math

import numpy as np
import pytest
import torch

from fp8kv_amd import ops, workloads
from oracle import rope_append, visible

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
D = 128
PARTS = {"decode": 2.0 ** -16, "prefill": 2.0 ** -7}


def _case(kind, lens, HQ, HKV, PBLK, window, sinks, seed=0, spread=1.0):
    """lens: (earlier tokens, new tokens).  Block 0 is the NaN block."""
    g = torch.Generator().manual_seed(seed)
    total = [a + b for a, b in lens]
    need = [max(0, -(-t // PBLK)) for t in total]
    NB = sum(need) + 1
    bf16 = kind == "bf16"
    x = torch.randn(NB, HKV, PBLK, 2 * D, generator=g) * torch.exp(spread * torch.randn(NB, HKV, PBLK, 1, generator=g))
    scales = torch.full((NB, PBLK // 16, HKV, 2), 127, dtype=torch.uint8)
    if bf16:
        pool = x.to(torch.bfloat16)
        bad = torch.tensor([float("nan"), float("inf"), float("-inf")]).to(torch.bfloat16)[torch.randint(0, 3, x.shape, generator=g)]
        ks = vs = 1.0
    else:
        ks, vs = 0.011, 0.017
        if kind == "blk":
            e = torch.randint(-9, -4, scales.shape, generator=g)
            e[..., 1] -= torch.randint(0, 30, scales.shape[:-1], generator=g)
            scales = (e + 127).to(torch.uint8)
            f = torch.exp2(e.float()).repeat_interleave(16, 1).permute(0, 2, 1, 3)       # [NB, HKV, PBLK, 2]
            f = f.repeat_interleave(D, -1)
            x[..., D:] *= f[..., D:] * 2.0 ** 6                # values of a block go with its scale
        else:
            f = torch.cat([torch.full((D,), ks), torch.full((D,), vs)])
        pool = (x / f).clamp(-448, 448).to(torch.float8_e4m3fn)
        bad = torch.full(x.shape, 0x7F, dtype=torch.uint8).view(torch.float8_e4m3fn)
    table = torch.zeros(len(lens), max(need + [1]), dtype=torch.int32)
    ids = 1 + torch.randperm(NB - 1, generator=g).to(torch.int32)
    seen = torch.zeros(NB, PBLK, dtype=torch.bool)
    at = 0
    for s, (a, b) in enumerate(lens):
        row = ids[at:at + need[s]]
        at += need[s]
        some = torch.zeros(need[s] * PBLK, dtype=torch.bool)
        for p in range(max(a, 0), a + b):
            some[visible.visible(p, total[s], window, sinks)] = True
        used = some.view(-1, PBLK).any(1)
        table[s, :need[s]] = torch.where(used, row, torch.zeros_like(row))
        seen[row.long()] = some.view(-1, PBLK)
    hide = ~seen[:, None, :, None].expand(x.shape)
    if bf16:
        pool = torch.where(hide, bad, pool)
    else:
        pool = torch.where(hide, bad.view(torch.uint8), pool.view(torch.uint8))
    starts = torch.tensor([0] + list(np.cumsum([b for _, b in lens])), dtype=torch.int32)
    q = (1.5 * torch.randn(int(starts[-1]), HQ, D, generator=g)).to(torch.bfloat16)
    return dict(kind=kind, q=q, pool=pool, scales=scales, ks=ks, vs=vs, table=table, starts=starts,
                seq_lens=torch.tensor(total, dtype=torch.int32), window=window, sinks=sinks, sm=1 / math.sqrt(D))


def _run(c, form, out=None, **more):
    d = {k: c[k].to(DEV) for k in ("q", "pool", "scales", "table", "starts", "seq_lens")}
    k, v = workloads.engine_views(d["pool"], D)
    out = torch.full_like(d["q"], 7.0) if out is None else out
    scales = (d["scales"],) if c["kind"] == "blk" else (c["ks"], c["vs"])
    call = getattr(ops, f"{form}_attention_" + ("blk" if c["kind"] == "blk" else "window"))
    got = call(d["q"], k, v, out, d["starts"], d["seq_lens"], d["table"], *scales, c["sm"], window=c["window"],
               sinks=c["sinks"], **more)
    torch.cuda.synchronize()
    return got.cpu()


def _oracle(c):
    k, v = workloads.engine_views(c["pool"], D)
    ks, vs = ((c["scales"], 0), (c["scales"], 1)) if c["kind"] == "blk" else (c["ks"], c["vs"])
    return visible.attention(c["q"], k, v, c["starts"], c["seq_lens"], c["table"], ks, vs, c["sm"], c["window"], c["sinks"])


def _tolerance(c, form, want, mass, reach):
    return 2.0 ** -8 * want.abs() + (PARTS[form] + 280 * 2.0 ** -24 * reach[..., None] + 2.0 ** -20) * mass + 1e-30


def _check(c, form, **more):
    want, *bounds = _oracle(c)
    assert want.isfinite().all()                     # the planted NaN are nobody's
    got = _run(c, form, **more).double()
    assert got.isfinite().all()
    off = (got - want).abs() - _tolerance(c, form, want, *bounds)
    assert (off <= 0).all(), f"{(off > 0).sum()} of {off.numel()} out of bounds, worst by {off.max():.3g}"


KINDS = ["fp8", "bf16", "blk"]
DECODE_LENS = [0, 1, 15, 16, 17, 47, 300, 777]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (1, 1), (16, 4), (17, 16), (100, 0), (100, 33), (300, 300), (5000, 4), (33, 700)])
def test_decode_masks(kind, window, sinks):
    lens = [(n - 1, 1) for n in DECODE_LENS]
    for PBLK, splits in ((16, None), (64, 3)):
        _check(_case(kind, lens, 8, 2, PBLK, window, sinks, seed=window + sinks), "decode", num_splits=splits)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("HQ,HKV", [(3, 3), (4, 2), (3, 1), (5, 1), (12, 2), (7, 1), (16, 2), (11, 1), (16, 1)])
def test_decode_heads_and_splits(kind, HQ, HKV):
    lens = [(1200, 1), (3, 1), (450, 1)]
    for window, sinks, splits in ((0, 0, 8), (700, 4, 5), (700, 20, 40), (64, 0, None)):
        _check(_case(kind, lens, HQ, HKV, 32, window, sinks, seed=HQ), "decode", num_splits=splits, max_seq_len=1201)


@pytest.mark.parametrize("kind", KINDS)
def test_decode_many_sequences_and_long_context(kind):
    lens = [((37 * i) % 500, 1) for i in range(150)]
    _check(_case(kind, lens, 4, 2, 16, 120, 4), "decode")
    _check(_case(kind, [(20000, 1), (9000, 1)], 4, 1, 128, 0, 0), "decode", max_seq_len=20001)
    _check(_case(kind, [(20000, 1), (9000, 1)], 4, 1, 128, 6000, 50), "decode")


PART_LENS = {
    "ragged": [5000, 1, 0, 16, 17, 700, 0, 2300, 33],
    "no_keys": [0, -3, 0, 0, 0],
    "one_token": [1, 1, 1],
    "long_last": [3, 0, 0, 9000],
    "fewer_groups_than_parts": [100, 16, 40],
    "one_group_more": [1040, 1024, 1024, 1023],
    "many": [(37 * i) % 400 for i in range(200)],
    "most": [(11 * i) % 60 for i in range(255)] + [700],
    "too_many_to_share": [(11 * i) % 60 for i in range(257)],
}
LONG = 1 << 24                  # a longest context for which any batch is cut into parts


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("lens", PART_LENS.values(), ids=PART_LENS.keys())
def test_decode_parts(kind, lens):
    """The walks of a batch in equal parts: boundaries inside sequences, parts of many sequences, sequences of many parts."""
    lens = [(n - 1, 1) for n in lens]
    for HQ, HKV, window, sinks in ((8, 2, 0, 0), (3, 1, 0, 0), (16, 16, 0, 0), (16, 16, 4000, 500), (2, 1, 4000, 500)):
        if len(lens) > 50 and HKV > 2:
            continue
        c = _case(kind, lens, HQ, HKV, 32, window, sinks, seed=HKV)
        splits = ops.decode_visible_splits(len(lens), HKV, LONG, window, sinks, kind == "bf16")
        for n in {splits, 2, 3, 7}:
            _check(c, "decode", num_splits=n, max_seq_len=LONG)


def test_decode_parts_share_scratch():
    """One scratch for calls of either shape and any lengths, in turn and replayed from a graph; same results every time."""
    lens = [900, 1, 0, 3000, 64, 17]
    c = _case("blk", [(n - 1, 1) for n in lens], 8, 2, 16, 0, 0, seed=5)
    want, *bounds = _oracle(c)
    d = {k: c[k].to(DEV) for k in ("q", "pool", "scales", "table", "starts", "seq_lens")}
    k, v = workloads.engine_views(d["pool"], D)
    splits = ops.decode_visible_splits(len(lens), 2, LONG)
    scratch = ops.decode_scratch(ops.decode_scratch_bytes(len(lens), 8, 2, max(splits, 16), D), DEV)

    def call(n, longest, lens=d["seq_lens"]):
        out = torch.full_like(d["q"], 7.0)
        return ops.decode_attention_blk(d["q"], k, v, out, d["starts"], lens, d["table"], d["scales"], c["sm"],
                                        num_splits=n, max_seq_len=longest, scratch=scratch)
    first = call(splits, LONG)
    assert ((first.cpu().double() - want).abs() <= _tolerance(c, "decode", want, *bounds)).all()
    moving = d["seq_lens"].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        replayed = call(splits, LONG, moving)
    for i in range(4):
        moving.copy_(torch.tensor([900 - 200 * i, 1, 0, 3000 - 7 * i, 64, 17 - i], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(replayed, call(splits, LONG, moving))
        call(16, 3000)                                         # splits of each sequence over the same records
        assert torch.equal(first, call(splits, LONG))


PREFILL_LENS = {
    "short": [(0, 1), (0, 16), (0, 17), (0, 37), (0, 0), (5, 3)],
    "after_cached": [(200, 33), (5, 100), (31, 1), (64, 64)],
    "negative_positions": [(-3, 10), (-20, 18), (0, 5), (-16, 40)],
    "one": [(130, 250)],
}


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("lens", PREFILL_LENS.values(), ids=PREFILL_LENS.keys())
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (1, 3), (16, 4), (33, 0), (40, 20), (100, 33), (4000, 4)])
def test_prefill_masks(kind, lens, window, sinks):
    for HQ, HKV, PBLK in ((6, 1, 16), (4, 2, 64)):
        c = _case(kind, lens, HQ, HKV, PBLK, window, sinks, seed=window + sinks)
        _check(c, "prefill")


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("HQ,HKV", [(3, 3), (4, 2), (3, 1), (8, 2), (5, 1), (12, 2), (7, 1), (16, 2), (11, 1), (12, 1), (14, 1), (16, 1)])
def test_prefill_heads(kind, HQ, HKV):
    for lens, window, sinks in (([(0, 90), (70, 40)], 0, 0), ([(300, 70)], 50, 4)):
        _check(_case(kind, lens, HQ, HKV, 16, window, sinks, seed=HQ), "prefill")


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("window,sinks", [(0, 0), (90, 5)])
def test_prefill_more_than_one_round(kind, window, sinks):
    """Enough blocks for several rounds of workgroups; checked on a sample of the rows."""
    c = _case(kind, [(0, 900), (40, 700), (11, 500)], 16, 8, 16, window, sinks)
    got = _run(c, "prefill").double()
    pick = sorted(set(range(0, c["q"].shape[0], 61)) | {899, 900, 1599, 1600, 2099})
    k, v = workloads.engine_views(c["pool"], D)
    for row in pick:
        s = int(torch.bucketize(torch.tensor(row), c["starts"][1:].long(), right=True))
        a, b = int(c["starts"][s]), int(c["starts"][s + 1])
        n = int(c["seq_lens"][s]) - (b - 1 - row)
        one = dict(c, q=c["q"][row:row + 1], starts=torch.tensor([0, 1]), seq_lens=torch.tensor([n]), table=c["table"][s:s + 1])
        want, *bounds = _oracle(one)
        assert ((got[row:row + 1] - want).abs() <= _tolerance(c, "prefill", want, *bounds)).all(), row


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("HQ,HKV", [(6, 1), (1, 1), (2, 1), (4, 1), (8, 1), (16, 1)])
def test_non_finite_values_reach_the_rows_that_see_them_and_no_other(kind, HQ, HKV):
    """A NaN (an infinity) in V, element 40, of token 70: rows 70 .. 70 + window - 1 have it there, all others and all
    other elements stay in bounds.  The same in K of token 90: rows that see it are NaN throughout."""
    window, sinks = 48, 4
    for what, where in (("v", 70), ("v", 2), ("k", 90)):
        for val in (float("nan"), float("inf")):
            if kind != "bf16" and val == float("inf"):
                continue
            c = _case(kind, [(0, 200)], HQ, HKV, 16, window, sinks, seed=3)
            want, *bounds = _oracle(c)
            tol = _tolerance(c, "prefill", want, *bounds)
            blk, slot = int(c["table"][0, where // 16]), where % 16
            at = (D if what == "v" else 0) + 40
            c["pool"] = c["pool"].clone()
            c["pool"][blk, :, slot, at] = val if kind == "bf16" else 0x7F
            got = _run(c, "prefill").double()
            t = torch.arange(200)
            sees = (t >= where) & ((t < where + window) | (where < sinks))
            if what == "v":
                col = got[:, :, 40]
                assert (col[sees].isnan() if val != val else col[sees] == val).all()
                keep = torch.ones(200, HQ, D, dtype=torch.bool)
                keep[sees, :, 40] = False
            else:
                if val != val:
                    assert got[sees].isnan().all()
                keep = (~sees)[:, None, None].expand(200, HQ, D)
            assert ((got - want).abs() <= tol)[keep].all()


def test_block_scales_far_apart():
    """Neighbouring blocks whose V differ by up to 2^20 and blocks of tiny and of large values."""
    c = _case("blk", [(0, 120), (700, 60)], 6, 1, 16, 0, 0, seed=5)
    g = torch.Generator().manual_seed(6)
    c["scales"][..., 1] = 127 + torch.randint(-20, 1, c["scales"].shape[:-1], generator=g).to(torch.uint8)
    _check(c, "prefill")
    for e in (27, 60, 200, 230):
        c["scales"][..., 1] = e
        _check(c, "prefill")
    c = _case("blk", [(999, 1), (40, 1)], 6, 1, 16, 0, 0, seed=5)
    for e in (27, 60, 200, 230):
        c["scales"][..., 1] = e
        _check(c, "decode", num_splits=3)


@pytest.mark.parametrize("form", ["decode", "prefill"])
def test_large_scores_of_one_sign_and_zero_scale(form):
    for kind in KINDS:
        c = _case(kind, [(99, 1), (30, 1)], 4, 2, 16, 20, 2, seed=8)
        c["q"] = c["q"] * 0 + 3.0
        for sm in (50.0, -50.0, 0.0):
            c["sm"] = sm
            want, *bounds = _oracle(c)
            got = _run(c, form).double()
            # at such scores the fp32 rounding of a score (2^-24 of it) is what moves the weights; the bound has it
            assert ((got - want).abs() <= _tolerance(c, form, want, *bounds)).all(), (kind, sm)


@pytest.mark.parametrize("kind", KINDS)
def test_largest_window_and_sinks(kind):
    """Windows and sinks at the top of their range hide nothing, behind rows of negative position too."""
    for window, sinks in ((2 ** 31 - 1, 0), (2 ** 31 - 1, 2 ** 31 - 1), (1, 2 ** 31 - 1), (2 ** 30, 5)):
        _check(_case(kind, [(-20, 70), (100, 33), (-5, 9)], 4, 2, 16, window, sinks, seed=13), "prefill")
        _check(_case(kind, [(0, 1), (400, 1), (-1, 1), (70, 1)], 4, 2, 16, window, sinks, seed=14), "decode")


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("form", ["decode", "prefill"])
def test_huge_scores_pick_their_key(form, kind):
    """Scores from 10^6 to 10^20: half a unit in the last place of one is more than a weight's whole range, and still
    every row whose best key is best by more than the scores' error is that key's V."""
    c = _case(kind, [(230, 1 if form == "decode" else 70), (31, 1 if form == "decode" else 40)], 6, 2, 16, 0, 0, seed=12)
    for sm in (1e4, 1e6, 1e7, 3e7, 1e8, 1e10, -1e10, 1e18, -1e18):
        c["sm"] = sm
        want, _, reach = _oracle(c)
        got = _run(c, form).double()
        assert got.isfinite().all(), sm
        k, _ = workloads.engine_views(c["pool"], D)
        scale = (c["scales"], 0) if kind == "blk" else c["ks"]
        clear = 0
        for s in range(2):
            a, b, length = int(c["starts"][s]), int(c["starts"][s + 1]), int(c["seq_lens"][s])
            for i in range(a, b):
                for h in range(2):
                    keys = visible.rows(k, c["table"][s], torch.arange(length - (b - a) + i - a + 1), h, scale)
                    best = (c["q"][i, 3 * h:3 * h + 3].double() @ keys.T * sm).sort(-1).values
                    for r in range(3):
                        row = 3 * h + r
                        if best.shape[1] > 1 and best[r, -1] - best[r, -2] > 560 * 2.0 ** -24 * reach[i, row] + 20:
                            clear += 1
                            assert ((got[i, row] - want[i, row]).abs() <= 2.0 ** -8 * want[i, row].abs() + 1e-6).all(), (sm, i, row)
        assert clear > 0.8 * 6 * int(c["starts"][-1])


@pytest.mark.parametrize("kind", KINDS)
def test_strided_rows_and_untouched_output(kind):
    """q and out as slices of wider rows; only the rows of the sequences are written."""
    c = _case(kind, [(50, 20), (0, 9)], 4, 2, 16, 30, 4, seed=9)
    want, *bounds = _oracle(c)
    T = c["q"].shape[0]
    wide = torch.full((T + 5, 3, 4, D), 3.0, dtype=torch.bfloat16, device=DEV)
    q = torch.zeros(T + 5, 2, 4, D, dtype=torch.bfloat16, device=DEV)
    q[:T, 1] = c["q"].to(DEV)
    d = {k: c[k].to(DEV) for k in ("pool", "scales", "table", "starts", "seq_lens")}
    k, v = workloads.engine_views(d["pool"], D)
    scales = (d["scales"],) if kind == "blk" else (c["ks"], c["vs"])
    call = ops.prefill_attention_blk if kind == "blk" else ops.prefill_attention_window
    call(q[:, 1], k, v, wide[:, 1], d["starts"], d["seq_lens"], d["table"], *scales, c["sm"], window=30, sinks=4,
         max_query_len=33)
    got = wide.cpu().double()
    assert ((got[:T, 1] - want).abs() <= _tolerance(c, "prefill", want, *bounds)).all()
    assert (got[:, 0] == 3).all() and (got[:, 2] == 3).all() and (got[T:] == 3).all()


@pytest.mark.parametrize("kind", ["fp8", "bf16"])
def test_whole_context_agrees_with_the_unwindowed_calls(kind):
    """Window 0, and one wider than the context, are the attention of decode_attention / prefill_attention_varlen."""
    for form, lens in (("decode", [(300, 1), (40, 1)]), ("prefill", [(300, 50), (0, 40)])):
        a = _run(_case(kind, lens, 8, 2, 16, 0, 0), form)
        c = _case(kind, lens, 8, 2, 16, 1 << 30, 7)
        b = _run(c, form)
        assert torch.equal(a, b)
        want, *bounds = _oracle(c)
        d = {k: c[k].to(DEV) for k in ("q", "pool", "table", "starts", "seq_lens")}
        k, v = workloads.engine_views(d["pool"], D)
        out = torch.empty_like(d["q"])
        args = (d["q"], k, v, out, d["starts"], d["seq_lens"], d["table"], c["ks"], c["vs"], c["sm"])
        ops.decode_attention(*args) if form == "decode" else ops.prefill_attention_varlen(*args)
        old = out.cpu().double()
        assert ((old - b.double()).abs() <= 2.0 ** -7 * want.abs() + 2.0 ** -7 * bounds[0]).all()


def test_offsets_past_32_bits():
    """Blocks at the end of a cache of 5 GB: append, prefill and decode there."""
    HKV, PBLK = 4, 16
    NB = 5 * (1 << 30) // (HKV * PBLK * 2 * D)
    pool = torch.empty(NB, HKV, PBLK, 2 * D, dtype=torch.uint8, device=DEV)
    small = _case("blk", [(0, 60)], 8, HKV, PBLK, 0, 0, seed=4)
    k, v = workloads.engine_views(pool, D)
    scales = torch.zeros(NB, 1, HKV, 2, dtype=torch.uint8, device=DEV)
    ids = small["table"].long()[0]
    far = torch.arange(NB - 4, NB, device=DEV)
    pool[far] = small["pool"].to(DEV)[ids.to(DEV)]
    scales[far] = small["scales"].to(DEV)[ids.to(DEV)]
    table = far.to(torch.int32).view(1, 4)
    want, *bounds = _oracle(small)
    for form, rows in (("prefill", 60), ("decode", 1)):
        q = small["q"][60 - rows:].to(DEV)
        out = torch.empty_like(q)
        call = ops.prefill_attention_blk if form == "prefill" else ops.decode_attention_blk
        call(q, k, v, out, torch.tensor([0, rows], dtype=torch.int32, device=DEV), small["seq_lens"].to(DEV), table, scales,
             small["sm"])
        tol = _tolerance(small, form, want, *bounds)[60 - rows:]
        assert ((out.cpu().double() - want[60 - rows:]).abs() <= tol).all()
    # a bf16 and a per-tensor append at the last slots, and a block-scaled one
    g = torch.Generator().manual_seed(1)
    kv = torch.randn(2, 3, HKV, D, generator=g).to(torch.bfloat16).to(DEV)
    slots = torch.tensor([NB * PBLK - 3, NB * PBLK - 1, NB * PBLK - 2], device=DEV)
    ops.rope_append(None, kv[0], kv[1], k, v, None, None, slots, 0.01, 0.01)
    ref = [torch.zeros(1, PBLK, HKV, D, dtype=torch.uint8, device=DEV) for _ in range(2)]
    ops.cache_write(kv[0], kv[1], *ref, slots - (NB - 1) * PBLK, 0.01, 0.01)
    assert torch.equal(k[NB - 1, 13:].view(torch.uint8), ref[0][0, 13:]) and torch.equal(v[NB - 1, 13:].view(torch.uint8), ref[1][0, 13:])
    ops.rope_append_blk(None, kv[0], kv[1], k, v, scales, None, None, torch.tensor([0, 3], dtype=torch.int32, device=DEV),
                        torch.tensor([51], dtype=torch.int32, device=DEV), table)
    e = rope_append.needed_exp(kv[1][:, 0].float().cpu().numpy())
    assert int(scales[NB - 1, 0, 0, 1]) == e + 127


@pytest.mark.parametrize("kind", ["fp8", "bf16", "blk"])
def test_graph_replays_and_streams(kind):
    """Captured without a warm-up call, replayed with changed queries and lengths; two streams with a scratch each."""
    lens = [(700, 1), (40, 1), (333, 1)]
    c = _case(kind, lens, 8, 2, 16, 400, 4, seed=2)
    d = {k: c[k].to(DEV) for k in ("q", "pool", "scales", "table", "starts", "seq_lens")}
    k, v = workloads.engine_views(d["pool"], D)
    scales = (d["scales"],) if kind == "blk" else tuple(torch.tensor([x], device=DEV) for x in (c["ks"], c["vs"]))
    name = "blk" if kind == "blk" else "window"
    outs = [torch.empty_like(d["q"]) for _ in range(2)]

    def call(out, lens, scratch=None):
        getattr(ops, "decode_attention_" + name)(d["q"], k, v, out, d["starts"], lens, d["table"], *scales, c["sm"],
                                                 window=400, sinks=4, num_splits=4, scratch=scratch)
        return out

    def pre(out, lens):
        getattr(ops, "prefill_attention_" + name)(d["q"], k, v, out, d["starts"], lens, d["table"], *scales, c["sm"],
                                                  window=400, sinks=4, max_query_len=1)
        return out
    lens_dev = d["seq_lens"].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(outs[0], lens_dev)
        pre(outs[1], lens_dev)
    for i in range(4):
        d["q"].copy_(torch.randn_like(d["q"].float()))
        lens_dev.copy_(torch.tensor([700 - i, 41 - i, 334 - 5 * i], dtype=torch.int32))
        # hidden slots hold NaN: shorter lengths see a window that begins earlier, so give the tokens there values
        if kind == "bf16":
            d["pool"].nan_to_num_(0.5, 0.5, 0.5)
        else:
            d["pool"][(d["pool"] & 0x7F) == 0x7F] = 0x30
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], call(torch.empty_like(d["q"]), lens_dev))
        assert torch.equal(outs[1], pre(torch.empty_like(d["q"]), lens_dev))
    need = ops.decode_scratch_bytes(3, 8, 2, 4)
    streams = [torch.cuda.Stream() for _ in range(2)]
    bufs = [torch.zeros(need, dtype=torch.uint8, device=DEV) for _ in range(2)]
    res = [torch.empty_like(d["q"]) for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(3):
        for s, b, r in zip(streams, bufs, res):
            with torch.cuda.stream(s):
                call(r, lens_dev, b)
    torch.cuda.synchronize()
    assert torch.equal(res[0], outs[0]) and torch.equal(res[1], outs[0])


@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 4)])
@pytest.mark.parametrize("kind", KINDS)
def test_a_prompt_then_single_tokens(kind, window, sinks):
    """As an engine runs them: append and attend over a prompt, then token by token, on caches that the appends
    wrote; every output against the oracle on the cache as it stands, and against unquantised attention."""
    g = torch.Generator().manual_seed(21)
    HQ, HKV, PBLK, prompts, steps = 6, 2, 16, [37, 5, 64], 20
    NS = len(prompts)
    NB = sum(-(-(n + steps) // PBLK) for n in prompts) + 1
    dtype = torch.bfloat16 if kind == "bf16" else torch.uint8
    pool = torch.zeros(NB, HKV, PBLK, 2 * D, dtype=dtype, device=DEV)
    kc, vc = workloads.engine_views(pool, D)
    kv_scales = torch.zeros(NB, 1, HKV, 2, dtype=torch.uint8, device=DEV)
    ids = torch.randperm(NB, generator=g).to(torch.int32)
    table = torch.zeros(NS, max(-(-(n + steps) // PBLK) for n in prompts), dtype=torch.int32)
    at = 0
    for s, n in enumerate(prompts):
        m = -(-(n + steps) // PBLK)
        table[s, :m] = ids[at:at + m]
        at += m
    table_d = table.to(DEV)
    cos_sin = ops.rope_table(256, D, DEV)
    ks = vs = 0.02
    keys = [[] for _ in prompts]
    lens = [0] * NS
    for step in range(steps + 1):
        new = prompts if step == 0 else [1] * NS
        T = sum(new)
        qkv = torch.randn(T, (HQ + 2 * HKV) * D, generator=g).to(torch.bfloat16).to(DEV)
        q, key, value = (x.view(T, -1, D) for x in qkv.split([HQ * D, HKV * D, HKV * D], 1))
        pos = torch.cat([torch.arange(lens[s], lens[s] + n) for s, n in enumerate(new)])
        seq = torch.repeat_interleave(torch.arange(NS), torch.tensor(new))
        slots = table[seq, pos // PBLK].long() * PBLK + pos % PBLK
        lens = [a + b for a, b in zip(lens, new)]
        starts = torch.tensor([0] + list(np.cumsum(new)), dtype=torch.int32)
        lens_t = torch.tensor(lens, dtype=torch.int32)
        if kind == "blk":
            rot = ops.rope_append_blk(q, key, value, kc, vc, kv_scales, pos.to(DEV), cos_sin, starts.to(DEV),
                                      lens_t.to(DEV), table_d)
        else:
            rot = ops.rope_append(q, key, value, kc, vc, pos.to(DEV), cos_sin, slots.to(DEV), ks, vs)
        out = torch.empty_like(rot)
        form = "prefill" if step == 0 else "decode"
        call = getattr(ops, f"{form}_attention_" + ("blk" if kind == "blk" else "window"))
        sc = (kv_scales,) if kind == "blk" else (ks, vs)
        call(rot, kc, vc, out, starts.to(DEV), lens_t.to(DEV), table_d, *sc, 1 / math.sqrt(D), window=window, sinks=sinks)
        c = dict(kind=kind, q=rot.cpu(), pool=pool.cpu(), scales=kv_scales.cpu(), ks=float(np.float32(ks)), vs=float(np.float32(vs)),
                 table=table, starts=starts, seq_lens=lens_t, window=window, sinks=sinks, sm=1 / math.sqrt(D))
        want, *bounds = _oracle(c)
        assert ((out.cpu().double() - want).abs() <= _tolerance(c, form, want, *bounds)).all(), step
        tab = cos_sin.cpu().double().numpy()
        turned = rope_append.rotate(key.double().cpu().numpy(), pos.numpy(), tab, False)
        for s in range(NS):
            a, b = int(starts[s]), int(starts[s + 1])
            keys[s].append((torch.from_numpy(turned[a:b]), value[a:b].cpu().double()))
        if step in (0, steps):
            turned_q = torch.from_numpy(rope_append.rotate(q.double().cpu().numpy(), pos.numpy(), tab, False))
            for s in range(NS):
                k, v = (torch.cat([x[i] for x in keys[s]]) for i in range(2))
                row = int(starts[s + 1]) - 1
                seen = visible.visible(lens[s] - 1, lens[s], window, sinks)
                for h in range(HQ):
                    w = torch.softmax(turned_q[row, h] @ k[seen, h // 3].T / math.sqrt(D), -1)
                    plain = w @ v[seen, h // 3]
                    # e4m3 is off by 2^-4 of an element at most (bf16 2^-8): values directly, keys through the scores
                    half = 2.0 ** -8 if kind == "bf16" else 2.0 ** -4
                    err = half * (w @ v[seen, h // 3].abs()).max() + (math.expm1(2 * half * float((turned_q[row, h].abs() @ k[seen, h // 3].abs().T).max()) / math.sqrt(D))) * v[seen, h // 3].abs().max()
                    assert ((out[row, h].cpu().double() - plain).abs() <= err + 2.0 ** -7 * plain.abs() + 1e-3).all()


def test_refusals():
    c = _case("fp8", [(20, 4)], 4, 2, 16, 8, 0)
    d = {k: c[k].to(DEV) for k in ("q", "pool", "scales", "table", "starts", "seq_lens")}
    k, v = workloads.engine_views(d["pool"], D)
    out = torch.empty_like(d["q"])
    good = [d["q"], k, v, out, d["starts"], d["seq_lens"], d["table"], 1.0, 1.0, 0.1, 8, 0]
    blk = good[:7] + [d["scales"], 0.1, 8, 0]
    for call, args, changes in (
            (ops.decode_attention_window, good, {0: d["q"].half(), 1: k[:, :, :1], 3: out[:, :1], 4: d["starts"].long(),
                                                 5: d["seq_lens"][:0], 6: d["table"].long(), 10: -1, 11: -1}),
            (ops.prefill_attention_window, good, {0: d["q"][:, :, :64], 2: v[:1], 4: d["starts"][:1], 10: -1, 11: -3}),
            (ops.decode_attention_blk, blk, {1: k.view(torch.uint8).to(torch.bfloat16), 7: d["scales"][:1], 9: -1}),
            (ops.prefill_attention_blk, blk, {7: d["scales"].int(), 10: -1})):
        for i, bad in changes.items():
            with pytest.raises(ValueError):
                call(*args[:i], bad, *args[i + 1:])
    with pytest.raises(Exception, match="status 2"):           # GQA past 16
        q = torch.zeros(4, 34, D, dtype=torch.bfloat16, device=DEV)
        ops.decode_attention_window(q, k, v, torch.empty_like(q), *good[4:])
    with pytest.raises(ValueError, match="scratch"):
        ops.decode_attention_window(*good, num_splits=4, scratch=torch.zeros(16, dtype=torch.uint8, device=DEV))
    with pytest.raises(ValueError, match="scratch"):
        ops.decode_attention_window(*good, num_splits=4, scratch=torch.zeros(2, 1 << 20, dtype=torch.uint8, device=DEV).t())
    for n in (0, -1, 257, 1 << 40):
        with pytest.raises(Exception, match="status 1"):
            ops.decode_attention_window(*good, num_splits=n)
    with pytest.raises(Exception, match="status 1"):
        ops.prefill_attention_window(*good[:10], 1 << 40)
    for i, bad in ((7, None), (8, torch.ones(1, device=DEV).half()), (3, None), (9, "one"), (10, 1.5)):
        with pytest.raises((ValueError, TypeError)):
            ops.prefill_attention_window(*good[:i], bad, *good[i + 1:])
    none = d["table"][:0]
    assert ops.decode_attention_window(d["q"], k, v, out, d["starts"][:1], d["seq_lens"][:0], none, *good[7:]) is out
    assert ops.prefill_attention_blk(d["q"], k, v, out, d["starts"][:1], d["seq_lens"][:0], none, *blk[7:]) is out
