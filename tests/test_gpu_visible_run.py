"""The append and visible-key attention calls in a run, as an engine makes them, against attention over the tokens that
were handed in (not over the cache as it was written).

The keys and values have four significant bits and the rotations are quarter turns, so every cache kind holds every
token exactly, and the outputs are held to the bounds of test_gpu_visible.py: no quantisation error hides a wrong slot,
position, scale or head.  That an output of zeros, of another head or of a shifted window breaks them is asserted too."""
import math

import numpy as np
import pytest
import torch

from fp8kv_amd import ops, workloads
from oracle import rope_append, visible
from test_gpu_visible import D, DEV, KINDS, PARTS

pytestmark = pytest.mark.gpu

HQ, HKV, PBLK, PROMPTS, STEPS = 6, 2, 16, [37, 5, 64, 130], 18


def _four_bits(g, *shape, low=-3, high=1):
    """Numbers of either sign with four significant bits and exponents in [low, high)."""
    mantissa = torch.randint(8, 16, shape, generator=g).double() / 8
    sign = 1 - 2 * torch.randint(0, 2, shape, generator=g).double()
    return (sign * mantissa * torch.exp2(torch.randint(low, high, shape, generator=g).double())).to(torch.bfloat16)


def _quarter_turns(positions, rot):
    """cos then sin of p (i + 1) quarter turns."""
    turn = torch.arange(positions)[:, None] * torch.arange(1, rot // 2 + 1) % 4
    cos, sin = torch.tensor([1., 0., -1., 0.]), torch.tensor([0., 1., 0., -1.])
    return torch.cat([cos[turn], sin[turn]], 1)


def _attend(q, k, v, seen):
    """(out, sum w |v|, largest sum |q k|) of one query row q [D] over the keys `seen` of k, v [n, D]."""
    k, v = k[seen], v[seen]
    w = torch.softmax(k @ q / math.sqrt(D), -1)
    return w @ v, w @ v.abs(), float((k.abs() @ q.abs()).max()) / math.sqrt(D)


@pytest.mark.parametrize("window,sinks,interleaved", [(0, 0, False), (40, 4, False), (25, 20, True)])
@pytest.mark.parametrize("kind", KINDS)
def test_outputs_are_those_of_the_tokens(kind, window, sinks, interleaved):
    g = torch.Generator().manual_seed(41)
    NS, rot = len(PROMPTS), 96
    need = [-(-(n + STEPS) // PBLK) for n in PROMPTS]
    NB = sum(need) + 1
    pool = torch.zeros(NB, HKV, PBLK, 2 * D, dtype=torch.bfloat16 if kind == "bf16" else torch.uint8, device=DEV)
    kc, vc = workloads.engine_views(pool, D)
    kv_scales = torch.zeros(NB, 1, HKV, 2, dtype=torch.uint8, device=DEV)
    ids = torch.randperm(NB, generator=g).to(torch.int32)
    table = torch.zeros(NS, max(need), dtype=torch.int32)
    at = 0
    for s, m in enumerate(need):
        table[s, :m] = ids[at:at + m]
        at += m
    cos_sin = _quarter_turns(256, rot)
    ks, vs = 2.0 ** -7, 2.0 ** -6          # keys up to 1.875 / ks = 240 and values up to 1.875 * 2 / vs = 240, both below 448
    told = [(torch.zeros(0, HKV, D, dtype=torch.float64),) * 2 for _ in PROMPTS]          # keys (rotated) and values so far
    lens = [0] * NS
    checked = strict = 0
    for step in range(STEPS + 1):
        new = PROMPTS if step == 0 else [1] * NS
        T = sum(new)
        q = torch.randn(T, HQ, D, generator=g).to(torch.bfloat16)
        key = _four_bits(g, T, HKV, D)
        # later values are larger, so that block scales grow inside of groups
        value = _four_bits(g, T, HKV, D, low=-3 + step // 4, high=1 + step // 4) / 8
        pos = torch.cat([torch.arange(lens[s], lens[s] + n) for s, n in enumerate(new)])
        seq = torch.repeat_interleave(torch.arange(NS), torch.tensor(new))
        lens = [a + b for a, b in zip(lens, new)]
        starts = torch.tensor([0] + list(np.cumsum(new)), dtype=torch.int32)
        meta = (starts.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV), table.to(DEV))
        head = (q.to(DEV), key.to(DEV), value.to(DEV), kc, vc)
        if kind == "blk":
            rotated = ops.rope_append_blk(*head, kv_scales, pos.to(DEV), cos_sin.to(DEV), *meta, interleaved=interleaved)
        else:
            slots = table[seq, pos // PBLK].long() * PBLK + pos % PBLK
            rotated = ops.rope_append(*head, pos.to(DEV), cos_sin.to(DEV), slots.to(DEV), ks, vs, interleaved=interleaved)
        form = "prefill" if step == 0 else "decode"
        call = getattr(ops, f"{form}_attention_" + ("blk" if kind == "blk" else "window"))
        got = call(rotated, kc, vc, torch.empty_like(rotated), *meta, *((kv_scales,) if kind == "blk" else (ks, vs)),
                   1 / math.sqrt(D), window=window, sinks=sinks).cpu().double()
        tab = cos_sin.double().numpy()
        q64, k64 = (torch.from_numpy(rope_append.rotate(x.double().numpy(), pos.numpy(), tab, interleaved)) for x in (q, key))
        assert torch.equal(rotated.cpu().double(), q64)
        for s in range(NS):
            rows = slice(int(starts[s]), int(starts[s + 1]))
            told[s] = tuple(torch.cat([a, b]) for a, b in zip(told[s], (k64[rows], value[rows].double())))
            n = int(starts[s + 1] - starts[s])
            for i in sorted({0, n // 3, n - 2, n - 1} & set(range(n))):
                row, p = int(starts[s]) + i, lens[s] - n + i
                seen = visible.visible(p, lens[s], window, sinks)
                for h in range(HQ):
                    k, v = (x[:, h // 3] for x in told[s])
                    want, mass, reach = _attend(q64[row, h], k, v, seen)
                    tol = 2.0 ** -8 * want.abs() + (PARTS[form] + 280 * 2.0 ** -24 * reach + 2.0 ** -20) * mass
                    assert ((got[row, h] - want).abs() <= tol).all(), (step, s, i, h)
                    checked += 1
                    other = _attend(q64[row, (h + 1) % HQ], k, v, seen)[0]
                    late = _attend(q64[row, h], k, v, seen[1:] if len(seen) > 1 else seen)[0]
                    strict += bool((want.abs() > tol).any() and (len(seen) < 2 or ((want - other).abs() > tol).any() and
                                                                  ((want - late).abs() > tol).any()))
    assert checked > 300 and strict >= 0.98 * checked
