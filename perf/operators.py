"""Operators around the paged KV cache, as cases to be measured.

A serving program appends the new tokens of every step to its cache and attends over what the
cache holds.  Three families of calls, each for one token per sequence and for packed prompts:

  * ``append``  rotate queries and keys to their positions and append keys and values to a paged
                cache: e4m3 with one scale per tensor or bf16 (``ops.rope_append``), or e4m3 with a
                power-of-two scale per 16 tokens and kv head (``ops.rope_append_blk``);
  * ``blk``     attention over the cache with a scale per 16 tokens and kv head
                (``ops.decode_attention_blk``, ``ops.prefill_attention_blk``);
  * ``win``     attention with a sliding window and a few first tokens that stay visible
                (``ops.decode_attention_window``, ``ops.prefill_attention_window``).

Caches have the engine's layout: one [blocks, kv heads, block size, 2 D] tensor with K and V side
by side, read through strided views; queries, keys and values are slices of one projection's
output.  Where ``own`` is false every operator is computed in its plain form, elementary tensor
operations in 32 bits; where it is true by the framework's calls.
"""
import math
import os
import random
import sys

import torch

own = False

D = 128                       # head size
E4M3_MAX = 448.0
GROUP = 16                    # tokens that share a scale
SCALE_MIN_EXP = -100          # smallest exponent of such a scale


# ------------------------------------------------------------------------------ the cases

def listed():
    return [
        # one conversation's next token: the smallest call, all latency
        {"name": "append_decode_b1", "op": "append", "kind": "fp8", "seqs": 1, "new_lo": 1, "new_hi": 1, "cached_lo": 776,
         "cached_hi": 776, "heads": 24, "kv_heads": 4, "block": 16, "rot": 128, "interleaved": False},
        # a busy server's decode step into scaled blocks that are partly full
        {"name": "append_decode_b64_blk", "op": "append", "kind": "blk", "seqs": 64, "new_lo": 1, "new_hi": 1, "cached_lo": 0,
         "cached_hi": 8191, "heads": 32, "kv_heads": 8, "block": 16, "rot": 128, "interleaved": False},
        # prompts of unequal length that arrived together, behind cached prefixes that end inside a block
        {"name": "append_prompts_6_blk", "op": "append", "kind": "blk", "seqs": 6, "new_lo": 37, "new_hi": 900, "cached_lo": 150,
         "cached_hi": 200, "heads": 24, "kv_heads": 4, "block": 32, "rot": 128, "interleaved": False},
        # a long prompt into a bf16 cache, half of each head rotated in adjacent pairs
        {"name": "append_prompt_4096_bf16", "op": "append", "kind": "bf16", "seqs": 1, "new_lo": 4096, "new_hi": 4096,
         "cached_lo": 0, "cached_hi": 0, "heads": 28, "kv_heads": 4, "block": 16, "rot": 64, "interleaved": True},
        # one short conversation over a block-scaled cache
        {"name": "blk_decode_b1_short", "op": "blk", "kind": "blk", "seqs": 1, "new_lo": 1, "new_hi": 1, "cached_lo": 776,
         "cached_hi": 776, "heads": 24, "kv_heads": 4, "block": 16, "window": 0, "sinks": 0},
        # many sequences with long, unequal contexts
        {"name": "blk_decode_b32", "op": "blk", "kind": "blk", "seqs": 32, "new_lo": 1, "new_hi": 1, "cached_lo": 511,
         "cached_hi": 8191, "heads": 32, "kv_heads": 8, "block": 16, "window": 0, "sinks": 0},
        # the second chunk of a long prompt
        {"name": "blk_prefill_2048_after_2048", "op": "blk", "kind": "blk", "seqs": 1, "new_lo": 2048, "new_hi": 2048,
         "cached_lo": 2048, "cached_hi": 2048, "heads": 24, "kv_heads": 4, "block": 16, "window": 0, "sinks": 0},
        # several prompts of unequal length after short cached prefixes
        {"name": "blk_prefill_varlen_6", "op": "blk", "kind": "blk", "seqs": 6, "new_lo": 37, "new_hi": 900, "cached_lo": 200,
         "cached_hi": 200, "heads": 24, "kv_heads": 4, "block": 32, "window": 0, "sinks": 0},
        # long conversations of a model that attends to a window and keeps the first tokens visible
        {"name": "win_decode_b16", "op": "win", "kind": "fp8", "seqs": 16, "new_lo": 1, "new_hi": 1, "cached_lo": 900,
         "cached_hi": 32767, "heads": 32, "kv_heads": 8, "block": 16, "window": 1024, "sinks": 4},
        # a few sequences over a bf16 cache, one query head per kv head, a wide window
        {"name": "win_decode_b3_bf16", "op": "win", "kind": "bf16", "seqs": 3, "new_lo": 1, "new_hi": 1, "cached_lo": 1000,
         "cached_hi": 9000, "heads": 16, "kv_heads": 16, "block": 64, "window": 4096, "sinks": 0},
        # a long prompt's chunk behind cached tokens
        {"name": "win_prefill_4096_after_1000", "op": "win", "kind": "fp8", "seqs": 1, "new_lo": 4096, "new_hi": 4096,
         "cached_lo": 1000, "cached_hi": 1000, "heads": 24, "kv_heads": 4, "block": 16, "window": 1024, "sinks": 4},
        # prompts of unequal length over a bf16 cache, a window shorter than most of them
        {"name": "win_prefill_varlen_5_bf16", "op": "win", "kind": "bf16", "seqs": 5, "new_lo": 100, "new_hi": 1500,
         "cached_lo": 0, "cached_hi": 300, "heads": 32, "kv_heads": 8, "block": 16, "window": 512, "sinks": 16},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "append", "blk", "blk", "win", "win"])
    heads, kv = rng.choice([(24, 4), (24, 4), (32, 8), (32, 8), (28, 4), (16, 2), (16, 16), (48, 8), (12, 4), (40, 4)])
    prompts = rng.random() < 0.5
    case = {"op": op, "heads": heads, "kv_heads": kv, "block": rng.choice([16, 16, 32, 64, 128])}
    case["kind"] = "blk" if op == "blk" else rng.choice(["fp8", "bf16", "blk"])
    if op == "append":
        case.update(rot=rng.choice([128, 128, 64, 96, 32]), interleaved=rng.random() < 0.3)
    else:
        limited = op == "win" or rng.random() < 0.3
        case.update(window=_log_int(rng, 17, 4096) if limited else 0, sinks=rng.choice([0, 4, 4, 16, 33]) if limited else 0)
    if prompts:
        seqs = rng.choice([1, 1, 2, 3, 5, 8, 12])
        hi = _log_int(rng, 33, (2048 if seqs == 1 else 4000 // seqs))
        cached = rng.choice([0, _log_int(rng, 1, 2048 if seqs == 1 else 3000 // seqs)])
        case.update(seqs=seqs, new_lo=rng.randint(max(1, hi // 8), hi) if seqs > 1 else hi, new_hi=hi,
                    cached_lo=rng.randint(cached // 2, cached), cached_hi=cached)
    else:
        seqs = _log_int(rng, 1, 64)
        most = min(16384, int(1.0e8 / (2 * D * kv * (2 if case["kind"] == "bf16" else 1)) / seqs))
        hi = _log_int(rng, 33, max(most, 64))
        case.update(seqs=seqs, new_lo=1, new_hi=1, cached_lo=rng.randint(hi // 8, hi), cached_hi=hi)
    if case["seqs"] == 1:
        case["cached_lo"] = case["cached_hi"]
    return case


def _spread(n, lo, hi, salt):
    """n lengths from `lo` to `hi`, both of them present, in an order of no kind."""
    if n == 1:
        return [hi]
    got = [lo + (hi - lo) * i // (n - 1) for i in range(n)]
    random.Random(n * 1000003 + hi + salt).shuffle(got)
    return got


def _lengths(case):
    """(new tokens, cached tokens) of every sequence."""
    return (_spread(case["seqs"], case["new_lo"], case["new_hi"], 0),
            _spread(case["seqs"], case["cached_lo"], case["cached_hi"], 1))


# ------------------------------------------------------------------------------ inputs

def _values(g, *shape):
    """Keys and values as layers produce them: tokens of unequal norm (the last axis is the head)."""
    x = torch.randn(*shape, device="cuda", generator=g)
    return x * torch.exp(0.5 * torch.randn(*shape[:-1], 1, device="cuda", generator=g))


def _group_scales(x):
    """e8m0 bytes [NB, groups, HKV] of x [NB, HKV, block, D]: the smallest power of two that keeps a group's 16 rows within e4m3."""
    nb, hkv, block, _ = x.shape
    amax = x.reshape(nb, hkv, block // GROUP, GROUP * D).abs().amax(-1)
    return (_needed_exp(amax) + 127).to(torch.uint8).transpose(1, 2).contiguous()


def _pool(g, nb, kv, block, kind):
    """A cache of `nb` blocks in which every slot holds some token."""
    shape = (nb, kv, block, 2 * D)
    if kind == "bf16":
        pool = torch.empty(shape, dtype=torch.bfloat16, device="cuda")
        for h in range(2):
            pool[..., h * D:(h + 1) * D] = _values(g, nb, kv, block, D)
        return {"pool": pool, "k_scale": torch.ones(1, device="cuda"), "v_scale": torch.ones(1, device="cuda")}
    pool, scales = torch.empty(shape, dtype=torch.uint8, device="cuda"), []
    for h in range(2):
        x = _values(g, nb, kv, block, D)
        if kind == "blk":
            s = _group_scales(x)
            x = x / torch.exp2(s.transpose(1, 2).float() - 127).repeat_interleave(GROUP, 2)[..., None]
        else:
            s = (x.abs().max() / E4M3_MAX).reshape(1)
            x = x / s
        pool[..., h * D:(h + 1) * D] = x.clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn).view(torch.uint8)
        scales.append(s)
    if kind == "blk":
        return {"pool": pool, "kv_scales": torch.stack(scales, -1).contiguous()}
    return {"pool": pool, "k_scale": scales[0], "v_scale": scales[1]}


def _views(pool):
    k, v = pool.transpose(1, 2).split(D, dim=-1)
    return (k, v) if pool.dtype == torch.bfloat16 else (k.view(torch.float8_e4m3fn), v.view(torch.float8_e4m3fn))


def _table(g, case, total):
    """Block table of sequences of `total` tokens, blocks handed out in no order.  Blocks that no query sees
    any more have been given back: their entries are block 0, which no sequence owns."""
    block, window, sinks = case["block"], case.get("window", 0), case.get("sinks", 0)
    new, _ = _lengths(case)
    held = []
    for n, t in zip(new, total):
        first = max(0, t - n - window + 1) // block if window else 0
        held.append([b for b in range(-(-t // block)) if b >= first or b * block < sinks])
    count = 1 + sum(len(h) for h in held)
    ids = (1 + torch.randperm(count - 1, device="cuda", generator=g)).to(torch.int32)
    rows, cols = [], []
    for s, h in enumerate(held):
        rows += [s] * len(h)
        cols += h
    table = torch.zeros(len(total), max(1, max(-(-t // block) for t in total)), dtype=torch.int32, device="cuda")
    table[torch.tensor(rows, device="cuda"), torch.tensor(cols, device="cuda")] = ids
    return table, count


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _starts(lengths):
    got = [0]
    for n in lengths:
        got.append(got[-1] + n)
    return got


def _ops():
    path = os.path.join(os.getcwd(), "gfx1201-tuning-log_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from fp8kv_amd import ops
    return ops


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    new, cached = _lengths(case)
    total = [a + b for a, b in zip(new, cached)]
    heads, kv, block = case["heads"], case["kv_heads"], case["block"]
    table, blocks = _table(g, case, total)
    state = dict(case, **_pool(g, blocks, kv, block, case["kind"]), table=table, starts=_i32(_starts(new)),
                 seq_lens=_i32(total), longest_new=max(new), longest=max(total))
    state["k_cache"], state["v_cache"] = _views(state["pool"])
    tokens = sum(new)
    if case["op"] == "append":
        rot, most = case["rot"], max(total)
        qkv = torch.empty(tokens, (heads + 2 * kv) * D, dtype=torch.bfloat16, device="cuda")
        qkv[:, :heads * D] = torch.randn(tokens, heads * D, device="cuda", generator=g)
        qkv[:, heads * D:] = _values(g, tokens, 2 * kv, D).reshape(tokens, -1)
        at = lambda a, b: qkv[:, a * D:b * D].view(tokens, b - a, D)  # noqa: E731
        seq = torch.repeat_interleave(torch.arange(len(new), device="cuda"), _i32(new))
        pos = torch.arange(tokens, device="cuda") - state["starts"].long()[seq] + _i32(cached).long()[seq]
        freq = 1e4 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
        angle = torch.arange(most, dtype=torch.float64, device="cuda")[:, None] * freq
        state.update(q=at(0, heads), key=at(heads, heads + kv), value=at(heads + kv, heads + 2 * kv), positions=pos,
                     cos_sin=torch.cat([angle.cos(), angle.sin()], 1).float(),
                     slots=table[seq, pos // block].long() * block + pos % block,
                     q_out=torch.empty(tokens, heads, D, dtype=torch.bfloat16, device="cuda"))
    else:
        state["q"] = torch.randn(tokens, heads, D, device="cuda", generator=g).to(torch.bfloat16)
        state["out"] = torch.empty_like(state["q"])
        state["sm_scale"] = 1.0 / math.sqrt(D)
    return state


# ------------------------------------------------------------------------------ plain forms

def _rotate(x, positions, cos_sin, interleaved):
    """x [T, H, D] in 32 bits with the first R elements of each head rotated to the token's position."""
    half = cos_sin.shape[1] // 2
    c, s = cos_sin[positions, None, :half], cos_sin[positions, None, half:]
    x = x.float()
    part, rest = x[..., :2 * half], x[..., 2 * half:]
    a, b = (part[..., 0::2], part[..., 1::2]) if interleaved else (part[..., :half], part[..., half:])
    y, z = a * c - b * s, b * c + a * s
    return torch.cat([torch.stack([y, z], -1).flatten(-2) if interleaved else torch.cat([y, z], -1), rest], -1)


def _codes(x):
    return x.clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)


def _needed_exp(amax):
    """Exponent of the smallest power of two s >= 2^SCALE_MIN_EXP with amax / s <= 448."""
    mant, exp = torch.frexp((amax / E4M3_MAX).clamp(min=2.0 ** SCALE_MIN_EXP))
    return torch.where(mant == 0.5, exp - 1, exp)


def _append_plain(s):
    q = _rotate(s["q"], s["positions"], s["cos_sin"], s["interleaved"])
    s["q_out"].copy_(q)
    k = _rotate(s["key"], s["positions"], s["cos_sin"], s["interleaved"])
    v = s["value"].float()
    block, slots = s["block"], s["slots"]
    if s["kind"] != "blk":
        at = (slots // block, slots % block)
        if s["kind"] == "bf16":
            s["k_cache"][at], s["v_cache"][at] = k.to(torch.bfloat16), v.to(torch.bfloat16)
        else:
            s["k_cache"].view(torch.uint8)[at] = _codes(k / s["k_scale"]).view(torch.uint8)
            s["v_cache"].view(torch.uint8)[at] = _codes(v / s["v_scale"]).view(torch.uint8)
        return s["q_out"], s["pool"] if s["kind"] == "bf16" else s["pool"].view(torch.float8_e4m3fn)
    # the groups that get new tokens, the new tokens' rows in them, and the rows that were there before
    pos = s["positions"]
    group, member = torch.unique(slots // GROUP, return_inverse=True)
    kv = torch.stack([k, v], 2)                                            # [T, HKV, 2, D]
    fresh = torch.zeros(group.numel(), GROUP, kv.shape[1], 2, D, device=kv.device)
    fresh[member, pos % GROUP] = kv
    is_new = torch.zeros(group.numel(), GROUP, dtype=torch.bool, device=kv.device)
    is_new[member, pos % GROUP] = True
    first = torch.full((group.numel(),), GROUP, device=kv.device).scatter_reduce(0, member, pos % GROUP, "amin")
    is_old = torch.arange(GROUP, device=kv.device) < first[:, None]
    need = _needed_exp(fresh.abs().amax((1, 4)))                           # [groups, HKV, 2]
    scales = s["kv_scales"]
    blk, part = group * GROUP // block, group * GROUP % block // GROUP
    before = scales[blk, part].int() - 127
    exp = torch.where((first > 0)[:, None, None], torch.maximum(before, need), need)
    pool = s["pool"].view(-1, s["kv_heads"], block // GROUP, GROUP, 2, D)
    held = pool[blk, :, part].view(torch.float8_e4m3fn).float().permute(0, 2, 1, 3, 4)     # [groups, 16, HKV, 2, D]
    kept = _codes(held * torch.exp2((before - exp).float())[:, None, :, :, None])
    codes = _codes(fresh * torch.exp2(-exp.float())[:, None, :, :, None])
    now = torch.where(is_new[:, :, None, None, None], codes.view(torch.uint8), kept.view(torch.uint8))
    was = pool[blk, :, part].permute(0, 2, 1, 3, 4)
    pool[blk, :, part] = torch.where((is_new | is_old)[:, :, None, None, None], now, was).permute(0, 2, 1, 3, 4)
    scales[blk, part] = (exp + 127).to(torch.uint8)
    return s["q_out"], s["pool"].view(torch.float8_e4m3fn), scales.view(torch.float8_e8m0fnu)


def _attend_plain(s):
    dev, block, window, sinks = s["q"].device, s["block"], s["window"], s["sinks"]
    starts, lens = s["starts"].long(), s["seq_lens"].long()
    tokens, heads, _ = s["q"].shape
    kv, seqs, most = s["kv_heads"], lens.numel(), s["longest_new"]
    # queries as one row of `most` per sequence, and their positions
    row = torch.arange(most, device=dev)
    new = starts[1:] - starts[:-1]
    take = (starts[:-1, None] + row).clamp(max=tokens - 1)
    q = s["q"][take].float().view(seqs, most, kv, heads // kv, D).permute(0, 2, 3, 1, 4).reshape(seqs, kv, -1, D)
    qpos = (lens - new)[:, None] + row
    # the key positions that some query of the sequence sees
    if window and most == 1:
        near = lens[:, None] - window + torch.arange(window, device=dev)
        kpos = torch.cat([torch.arange(sinks, device=dev).expand(seqs, -1), near], 1)
        real = torch.cat([torch.arange(sinks, device=dev) < near[:, :1].clamp(min=0), near >= 0], 1)
    else:
        kpos = torch.arange(s["longest"], device=dev).expand(seqs, -1)
        real = torch.ones_like(kpos, dtype=torch.bool)
    real = real & (kpos < lens[:, None])
    kpos = torch.where(real, kpos, lens[:, None] - 1)
    blk, slot = s["table"].gather(1, kpos // block).long(), kpos % block
    k, v = s["k_cache"][blk, slot].float(), s["v_cache"][blk, slot].float()      # [seqs, keys, HKV, D]
    if s["kind"] == "blk":
        scale = torch.exp2(s["kv_scales"][blk, slot // GROUP].float() - 127)
        k, v = k * scale[..., 0, None], v * scale[..., 1, None]
    elif s["kind"] == "fp8":
        k, v = k * s["k_scale"], v * s["v_scale"]
    score = torch.matmul(q, k.permute(0, 2, 3, 1).contiguous()) * s["sm_scale"]
    seen = real[:, None] & (kpos[:, None] <= qpos[:, :, None])
    if window:
        seen = seen & ((kpos[:, None] > qpos[:, :, None] - window) | (kpos[:, None] < sinks))
    score = score.view(seqs, kv, heads // kv, most, -1).masked_fill(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(seqs, kv, -1, p.shape[-1]), v.permute(0, 2, 1, 3).contiguous())
    out = out.view(seqs, kv, -1, most, D) / torch.where(total > 0, total, torch.ones_like(total))
    seq = torch.bucketize(torch.arange(tokens, device=dev), starts[1:], right=True)
    out = out.permute(0, 3, 1, 2, 4).reshape(seqs, most, heads, D)[seq, torch.arange(tokens, device=dev) - starts[seq]]
    s["out"].copy_(out)
    return s["out"]


# ------------------------------------------------------------------------------ one pass

def _append_own(s):
    ops = _ops()
    if s["kind"] == "blk":
        ops.rope_append_blk(s["q"], s["key"], s["value"], s["k_cache"], s["v_cache"], s["kv_scales"], s["positions"],
                            s["cos_sin"], s["starts"], s["seq_lens"], s["table"], q_out=s["q_out"],
                            interleaved=s["interleaved"])
        return s["q_out"], s["pool"].view(torch.float8_e4m3fn), s["kv_scales"].view(torch.float8_e8m0fnu)
    ops.rope_append(s["q"], s["key"], s["value"], s["k_cache"], s["v_cache"], s["positions"], s["cos_sin"], s["slots"],
                    s["k_scale"], s["v_scale"], q_out=s["q_out"], interleaved=s["interleaved"])
    return s["q_out"], s["pool"] if s["kind"] == "bf16" else s["pool"].view(torch.float8_e4m3fn)


def _attend_own(s):
    ops = _ops()
    decode = s["longest_new"] == 1
    if s["kind"] == "blk":
        call = ops.decode_attention_blk if decode else ops.prefill_attention_blk
        scales = (s["kv_scales"],)
    else:
        call = ops.decode_attention_window if decode else ops.prefill_attention_window
        scales = (s["k_scale"], s["v_scale"])
    bound = {"max_seq_len": s["longest"]} if decode else {"max_query_len": s["longest_new"]}
    return call(s["q"], s["k_cache"], s["v_cache"], s["out"], s["starts"], s["seq_lens"], s["table"], *scales,
                s["sm_scale"], window=s["window"], sinks=s["sinks"], **bound)


def run(state):
    if state["op"] == "append":
        return _append_own(state) if own else _append_plain(state)
    return _attend_own(state) if own else _attend_plain(state)


def _visible(case):
    """(visible pairs of a query and a key, keys that some query of their sequence sees)."""
    window, sinks = case.get("window", 0), case.get("sinks", 0)
    pairs = keys = 0
    for n, c in zip(*_lengths(case)):
        for p in range(c, c + n):
            low = max(0, p - window + 1) if window else 0
            pairs += p + 1 - low + min(sinks, low)
        low = max(0, c - window + 1) if window else 0
        keys += c + n - low + min(sinks, low)
    return pairs, keys


def work(case):
    new, _ = _lengths(case)
    tokens, heads, kv = sum(new), case["heads"], case["kv_heads"]
    if case["op"] == "append":
        wide = 2 if case["kind"] == "bf16" else 1
        groups = sum(n // GROUP + 1 for n in new) if case["kind"] == "blk" else 0
        return {"bytes": tokens * (4 * heads * D + 2 * kv * D * (2 + wide) + 4 * case["rot"] + 16) + 4 * groups * kv,
                "flops": tokens * (heads + kv) * case["rot"] * 3}
    pairs, keys = _visible(case)
    per_key = 2 * D * kv * (2 if case["kind"] == "bf16" else 1) + (2 * kv / GROUP if case["kind"] == "blk" else 0)
    return {"bytes": 4 * tokens * heads * D + keys * per_key + keys / case["block"] * 4, "flops": 4 * D * heads * pairs}


# ------------------------------------------------------------------------------ in 64 bits

def _round_e4m3(x):
    """The e4m3 number nearest to x (ties to even, saturating), in 64 bits."""
    _, exp = torch.frexp(x)
    step = torch.ldexp(torch.ones_like(x), (exp - 1).clamp(min=-6) - 3)
    return (torch.round(x / step) * step).clamp(-E4M3_MAX, E4M3_MAX)


def _exact_append(s, case):
    x = {n: s[n].double() for n in ("q", "key", "value")}
    half, table = case["rot"] // 2, s["cos_sin"].double()[s["positions"]]
    for name in ("q", "key"):
        turned = x[name].clone()
        for i in range(half):
            a, b = (2 * i, 2 * i + 1) if case["interleaved"] else (i, i + half)
            c, w = table[:, None, i], table[:, None, half + i]
            turned[..., a] = x[name][..., a] * c - x[name][..., b] * w
            turned[..., b] = x[name][..., a] * w + x[name][..., b] * c
        x[name] = turned
    block, pool = case["block"], s["pool"]
    tokens = torch.stack([x["key"], x["value"]], 2)                        # [T, HKV, 2, D]
    if case["kind"] != "blk":
        held = (pool if case["kind"] == "bf16" else pool.view(torch.float8_e4m3fn)).double()
        if case["kind"] == "fp8":
            tokens = _round_e4m3(tokens / torch.stack([s["k_scale"], s["v_scale"]], 1).double()[0][:, None])
        held[s["slots"] // block, :, s["slots"] % block] = tokens.flatten(-2)
        return x["q"], held
    held, exps = pool.view(torch.float8_e4m3fn).double(), s["kv_scales"].double() - 127
    new, cached = _lengths(case)
    for i, (n, c) in enumerate(zip(new, cached)):
        rows = tokens[int(s["starts"][i]):int(s["starts"][i]) + n]
        for g in range(c // GROUP, (c + n - 1) // GROUP + 1):
            lo, hi = max(c, g * GROUP), min(c + n, g * GROUP + GROUP)
            b, at = int(s["table"][i, lo // block]), g * GROUP % block
            fresh = rows[lo - c:hi - c]
            exp = torch.ceil(torch.log2((fresh.abs().amax((0, 3)) / E4M3_MAX).clamp(min=2.0 ** SCALE_MIN_EXP)))
            old = lo - g * GROUP
            if old:
                was = exps[b, at // GROUP].clone()
                exp = torch.maximum(exp, was)
                there = held[b, :, at:at + old].view(-1, old, 2, D)
                there = _round_e4m3(there * torch.exp2(was - exp)[:, None, :, None])
                held[b, :, at:at + old] = there.flatten(-2)
            exps[b, at // GROUP] = exp
            held[b, :, at + old:at + hi - g * GROUP] = _round_e4m3(fresh / torch.exp2(exp)[..., None]).permute(1, 0, 2, 3).flatten(-2)
    return x["q"], held, torch.exp2(exps)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "append":
        return _exact_append(s, case)
    new, cached = _lengths(case)
    kv, group, block = case["kv_heads"], case["heads"] // case["kv_heads"], case["block"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    start = 0
    for i, (n, c) in enumerate(zip(new, cached)):
        pos = torch.arange(c + n, device="cuda")
        blk = s["table"][i].long()[pos // block]
        query = torch.arange(c, c + n, device="cuda")[:, None]
        hidden = pos > query
        if case["window"]:
            hidden = hidden | ((pos <= query - case["window"]) & (pos >= case["sinks"]))
        for h in range(kv):
            k, v = (t[blk, pos % block, h].double() for t in (s["k_cache"], s["v_cache"]))
            if case["kind"] == "blk":
                e = s["kv_scales"][blk, pos % block // GROUP, h].double() - 127
                k, v = k * torch.exp2(e[:, :1]), v * torch.exp2(e[:, 1:])
            elif case["kind"] == "fp8":
                k, v = k * s["k_scale"].double(), v * s["v_scale"].double()
            for j in range(h * group, (h + 1) * group):
                score = (s["q"][start:start + n, j].double() @ k.T) * s["sm_scale"]
                weight = torch.softmax(score.masked_fill(hidden, -math.inf), -1)
                out[start:start + n, j] = weight @ v
        start += n
    return out
