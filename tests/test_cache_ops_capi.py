"""Argument rejection of the append and visible-key attention calls, before any launch (no GPU; the pointers are
never followed), and checks of their oracles."""
import ctypes
import struct

import numpy as np
import pytest
import torch

from fp8kv_amd import _lib
from oracle import attention, formats, rope_append, visible

A = 0x10000
# q, q_out, key, value with strides, caches, strides (engine layout of 4 kv heads, blocks of 16), rotation
LEAD = [A, 4096, A, 4096, A, 4096, A, 4096, A, A + 128, 16384, 256, 4096, 16384, 256, 4096, A, A, 128, 0, 1000, 128, 0]
TAIL = [0, 24, 4, 128, 16, 100, None]                        # no tokens: nothing is launched


def _lead(elem=1, **at):
    args = list(LEAD)
    if elem == 2:
        args[9] = A + 256
    for i, v in at.items():
        args[int(i[1:])] = v
    return args


CHECKS = [
    (dict(_4=None), 1), (dict(_6=None), 1), (dict(_8=None), 1), (dict(_2=None), 1), (dict(_16=None), 1), (dict(_20=0), 1),
    (dict(_21=24), 2), (dict(_21=144), 2), (dict(_21=8), 2), (dict(_0=A + 8), 3), (dict(_1=4100), 3), (dict(_2=A + 8), 3),
    (dict(_4=A + 8), 3), (dict(_5=516), 3), (dict(_5=256), 1), (dict(_1=512), 1), (dict(_17=A + 8), 3), (dict(_18=130), 3),
    (dict(_18=64), 1), (dict(_8=A + 8), 3), (dict(_10=16392), 3), (dict(_14=252), 3)]


@pytest.mark.parametrize("change,code", CHECKS)
def test_append_rejects_before_launch(lib, change, code):
    assert lib.fp8kv_rope_append(*_lead(**change), A, A, A, *TAIL) == code
    blk = [A, A, A, A, 64, 64, 1]
    assert lib.fp8kv_rope_append_blk(*_lead(**change), *blk, *TAIL) == code


@pytest.mark.parametrize("change,code", [c for c in CHECKS if "_10" not in c[0] and "_14" not in c[0]] + [(dict(_14=252), 3), (dict(_9=A + 8), 3)])
def test_append_bf16_rejects_before_launch(lib, change, code):
    assert lib.fp8kv_rope_append_bf16(*_lead(2, **change), A, *TAIL) == code


@pytest.mark.parametrize("tail,code", [
    ([-1, 24, 4, 128, 16, 100, None], 1), ([0, 0, 4, 128, 16, 100, None], 1), ([0, 24, 0, 128, 16, 100, None], 1),
    ([0, 24, 4, 128, 16, -1, None], 1), ([0, 24, 4, 120, 16, 100, None], 2), ([0, 24, 4, 128, 24, 100, None], 2),
    ([1 << 24, 24, 4, 128, 16, 100, None], 2)])
def test_append_sizes(lib, tail, code):
    assert lib.fp8kv_rope_append(*LEAD, A, A, A, *tail) == code
    assert lib.fp8kv_rope_append_blk(*LEAD, A, A, A, A, 64, 64, 1, *tail) == code


def test_append_without_what_it_needs(lib):
    assert lib.fp8kv_rope_append(*LEAD, None, A, A, *TAIL) == 1
    assert lib.fp8kv_rope_append(*LEAD, A, None, A, *TAIL) == 1
    assert lib.fp8kv_rope_append_bf16(*_lead(2), None, *TAIL) == 1
    for i in range(4):
        blk = [A, A, A, A, 64, 64, 1]
        blk[i] = None
        assert lib.fp8kv_rope_append_blk(*LEAD, *blk, *TAIL) == 1
    assert lib.fp8kv_rope_append_blk(*LEAD, A, A, A, A, 64, 64, -1, *TAIL) == 1
    assert lib.fp8kv_rope_append_blk(*LEAD, A, A, A, A, 64, 64, 1, 0, 24, 4, 64, 16, 100, None) == 2   # head size
    assert lib.fp8kv_rope_append_blk(*LEAD, A, A, A, A, 64, 64, 1, 0, 24, 4, 128, 8, 100, None) == 2   # block size


def test_append_of_nothing_is_a_no_op(lib):
    assert lib.fp8kv_rope_append(*LEAD, A, A, A, *TAIL) == 0
    assert lib.fp8kv_rope_append_bf16(*_lead(2), A, *TAIL) == 0
    assert lib.fp8kv_rope_append_blk(*LEAD, A, A, A, A, 64, 64, 1, *TAIL) == 0
    assert lib.fp8kv_rope_append_blk(*LEAD, A, A, A, A, 64, 64, 0, 8, 24, 4, 128, 16, 100, None) == 0
    # without queries and without rotation the arguments that belong to them are not looked at
    assert lib.fp8kv_rope_append(*_lead(_0=None, _1=0, _2=None, _3=0, _16=None, _17=None, _18=0, _20=0, _21=0), A, A, A, 0, 0, 4, 128,
                                 16, 100, None) == 0


# q .. bt_stride of the attention calls: 24 / 4 heads, the engine's layout with blocks of 16
ATT = [A, 24 * 128, A, A + 128, 16384, 256, 4096, 16384, 256, 4096, A, 24 * 128, A, A, A, 64]
GEO = [8, 24, 4, 128, 16]


def _att(elem=1, **at):
    args = list(ATT)
    if elem == 2:
        args[3] = A + 256
    for i, v in at.items():
        args[int(i[1:])] = v
    return args


ATT_CHECKS = [(dict(_0=None), 1), (dict(_2=None), 1), (dict(_10=None), 1), (dict(_12=None), 1), (dict(_13=None), 1),
              (dict(_14=None), 1), (dict(_15=-1), 1), (dict(_0=A + 8), 3), (dict(_2=A + 8), 3), (dict(_3=A + 4), 3), (dict(_1=3076), 3),
              (dict(_5=264), 3), (dict(_8=260), 3), (dict(_5=-256), 2)]
GEO_CHECKS = [([0, 24, 4, 128, 16], 1), ([8, 0, 4, 128, 16], 1), ([8, 24, 0, 128, 16], 1), ([8, 25, 4, 128, 16], 2), ([8, 68, 4, 128, 16], 2),
              ([8, 24, 4, 64, 16], 2), ([8, 24, 4, 128, 8], 2), ([8, 24, 4, 128, 48], 2), ([65536, 24, 4, 128, 16], 2)]


def _forms(lib):
    """(decode call, prefill call, element bytes, scale arguments) of every cache kind."""
    return ((lib.fp8kv_decode_attn_window, lib.fp8kv_prefill_attn_window, 1, [A, A]),
            (lib.fp8kv_decode_attn_window_bf16, lib.fp8kv_prefill_attn_window_bf16, 2, []),
            (lib.fp8kv_decode_attn_blk, lib.fp8kv_prefill_attn_blk, 1, [A]))


@pytest.mark.parametrize("change,code", ATT_CHECKS)
def test_visible_attention_rejects_before_launch(lib, change, code):
    for dec, pre, elem, scales in _forms(lib):
        if elem == 2 and "_5" in change and change["_5"] == 264:
            change = dict(_5=260)
        args = _att(elem, **change)
        assert dec(*args, *scales, 0.1, *GEO, 4, None, 0, 64, 4, 0, None) == code
        assert pre(*args, *scales, 0.1, *GEO, 64, 4, 0, 0, None) == code


@pytest.mark.parametrize("geo,code", GEO_CHECKS)
def test_visible_attention_geometry(lib, geo, code):
    for dec, pre, elem, scales in _forms(lib):
        assert dec(*_att(elem), *scales, 0.1, *geo, 4, None, 0, 64, 4, 0, None) == code
        assert pre(*_att(elem), *scales, 0.1, *geo, 64, 4, 0, 0, None) == code


def test_visible_attention_window_splits_and_scales(lib):
    for dec, pre, elem, scales in _forms(lib):
        args = _att(elem)
        for win in ((-1, 0), (0, -1)):
            assert dec(*args, *scales, 0.1, *GEO, 1, None, 0, *win, 0, None) == 1
            assert pre(*args, *scales, 0.1, *GEO, *win, 0, 0, None) == 1
        assert dec(*args, *scales, 0.1, *GEO, 0, None, 0, 64, 4, 0, None) == 1
        assert dec(*args, *scales, 0.1, *GEO, 257, None, 0, 64, 4, 0, None) == 1
        assert dec(*args, *scales, 0.1, *GEO, 4, A, 100, 64, 4, 0, None) == 5
        assert pre(*args, *scales, 0.1, *GEO, 64, 4, -1, 0, None) == 1
        assert pre(*args, *scales, 0.1, *GEO, 64, 4, 0, -1, None) == 1
        for i in range(len(scales)):
            missing = scales[:i] + [None] + scales[i + 1:]
            assert dec(*args, *missing, 0.1, *GEO, 1, None, 0, 64, 4, 0, None) == 1
            assert pre(*args, *missing, 0.1, *GEO, 64, 4, 0, 0, None) == 1
        assert pre(*args, *scales, 0.1, *GEO, 64, 4, 0, 0, None) == 0                    # no queries: nothing is launched
    assert lib.fp8kv_decode_attn_blk(*_att(), A + 1, 0.1, *GEO, 1, None, 0, 64, 4, 0, None) == 3
    assert lib.fp8kv_prefill_attn_blk(*_att(), A + 1, 0.1, *GEO, 64, 4, 0, 0, None) == 3


# ---- the oracle itself ---------------------------------------------------------------------------

def test_oracle_rotation_keeps_norms_and_composes():
    rng = np.random.default_rng(0)
    x = rng.standard_normal((5, 2, 16))
    ang = np.arange(40)[:, None] * 10000.0 ** (-np.arange(0, 12, 2) / 12)
    table = np.concatenate([np.cos(ang), np.sin(ang)], 1)
    for inter in (False, True):
        y = rope_append.rotate(x, np.arange(5) + 3, table, inter)
        assert np.allclose(np.linalg.norm(y[..., :12], axis=-1), np.linalg.norm(x[..., :12], axis=-1))
        assert np.array_equal(y[..., 12:], x[..., 12:])
        # by p then by r is by p + r; scores depend on the distance alone
        z = rope_append.rotate(y, np.full(5, 7), table, inter)
        assert np.allclose(z, rope_append.rotate(x, np.arange(5) + 10, table, inter))
        a, b = (rope_append.rotate(x[:1], [p], table, inter)[0, 0] for p in (4, 20))
        c, d = (rope_append.rotate(x[1:2], [p], table, inter)[0, 0] for p in (9, 25))
        assert np.isclose(a @ c, b @ d)


def test_oracle_exponents_and_rounding():
    for top, e in ((448.0, 0), (448.0001, 1), (447.9, 0), (7.0, -6), (3.5, -7), (1e-40, -100), (0.0, -100), (3e38, 120)):
        assert rope_append.needed_exp(np.array([0.0, -top, np.nan, np.inf])) == e, top
    codes = formats.e4m3fn_table()
    fine = codes[np.isfinite(codes)]
    assert np.array_equal(rope_append.round_e4m3(fine), fine)
    mids = (np.sort(np.unique(fine))[1:] + np.sort(np.unique(fine))[:-1]) / 2
    from oracle.kv_cache import encode_e4m3fn_satfinite
    assert np.array_equal(rope_append.round_e4m3(mids), codes[encode_e4m3fn_satfinite(mids.astype(np.float32))])


def test_oracle_visible_keys():
    assert visible.visible(9, 10, 0, 3).tolist() == list(range(10))
    assert visible.visible(9, 10, 4, 2).tolist() == [0, 1, 6, 7, 8, 9]
    assert visible.visible(9, 10, 1, 0).tolist() == [9]
    assert visible.visible(2, 10, 5, 9).tolist() == [0, 1, 2]
    assert visible.visible(-1, 10, 5, 9).numel() == 0 and visible.visible(4, 0, 0, 0).numel() == 0


def test_oracle_agrees_with_the_whole_context_oracle_and_with_masked_softmax():
    from fp8kv_amd import workloads
    c = workloads.prefill_case([9, 4], [20, 0], HQ=4, HKV=2, seed=1)
    args = (c["q"], c["k_cache"], c["v_cache"], c["cu_seqlens_q"], c["seq_lens"], c["block_table"], c["k_scale"], c["v_scale"], c["sm_scale"])
    whole = attention.varlen_prefill_attention(*args)
    assert torch.allclose(visible.attention(*args)[0], whole, atol=1e-12)
    assert torch.allclose(visible.attention(*args, window=100, sinks=3)[0], whole, atol=1e-12)
    got = visible.attention(*args, window=6, sinks=2)[0]
    k, v = (attention.gather_kv(c[n], c["block_table"][0], 29, 1) for n in ("k_cache", "v_cache"))
    for i in range(9):
        p = 20 + i
        hidden = torch.tensor([t > p or (t <= p - 6 and t >= 2) for t in range(29)])
        s = (c["q"][i, 3].double() @ k.T * c["sm_scale"] * c["k_scale"]).masked_fill(hidden, -float("inf"))
        assert torch.allclose(got[i, 3], torch.softmax(s, -1) @ v * c["v_scale"], atol=1e-12)
    # scales that are powers of two: the block-scaled form of the same values
    sc = torch.full((c["k_cache"].shape[0], 1, 2, 2), 127, dtype=torch.uint8)
    sc[..., 0] += 3
    a = visible.attention(*args[:6], (sc, 0), (sc, 1), c["sm_scale"], 6, 2)[0]
    b = visible.attention(*args[:6], 8.0, 1.0, c["sm_scale"], 6, 2)[0]
    assert torch.allclose(a, b, atol=1e-12)


@pytest.mark.parametrize("ns,hkv,ctx,window,sinks,bf16,want", [
    (32, 8, 2559, 0, 0, 0, 1), (32, 8, 2560, 0, 0, 0, 2), (32, 8, 100000, 2000, 559, 0, 1), (32, 8, 100000, 2000, 560, 0, 2),
    (32, 8, 1279, 0, 0, 1, 1), (32, 8, 1280, 0, 0, 1, 2), (16, 4, 10239, 0, 0, 0, 4), (16, 4, 10240, 0, 0, 0, 5),
    (24, 8, 2047, 0, 0, 0, 2), (24, 8, 2048, 0, 0, 0, 3), (128, 8, 2047, 0, 0, 0, 1), (128, 8, 2048, 0, 0, 0, 2),
    (1, 4, 1 << 24, 0, 0, 0, 32), (257, 8, 1 << 24, 0, 0, 0, 1), (2, 1, 1 << 24, 0, 0, 0, 129), (2, 257, 1 << 24, 0, 0, 0, 1),
    (2, 1, 1 << 30, 0, 0, 0, 32), (64, 8, 0, 0, 0, 0, 1), (64, 8, 0, 4096, 4, 0, 2), (64, 8, 0, 1 << 30, 4, 0, 1)])
def test_decode_visible_split_plan(lib, ns, hkv, ctx, window, sinks, bf16, want):
    """Both sides of the lines between splits of a sequence and equal parts of the batch; a count that a call takes."""
    assert lib.fp8kv_decode_visible_splits(ns, hkv, ctx, window, sinks, bf16) == want
    assert 1 <= want <= 256


def test_prefill_visible_plan(lib):
    out = (ctypes.c_int * 5)()
    for hq, hkv in ((4, 4), (8, 4), (12, 4), (24, 4), (32, 4), (64, 4), (11, 1), (7, 7)):
        for ns, longest, tokens in ((1, 1, 1), (1, 4096, 4096), (6, 900, 0), (40, 512, 3000), (200, 16, 3200), (65535, 1, 65535)):
            for window, sinks in ((0, 0), (1024, 4), (16, 0)):
                for bf16 in (0, 1):
                    assert lib.fp8kv_prefill_visible_plan(hq, hkv, ns, longest, tokens, window, sinks, bf16, out) == 0
                    sets, groups, blocks, paired, ranks = out
                    assert sets in (2, 3) and groups in (2, 4, 8) and blocks >= 1 and ranks >= 1
                    assert blocks * (hq // hkv) <= sets * groups                          # every row has a place
                    assert (1 + paired) * ranks * blocks * 16 >= longest                  # and every token a workgroup
    assert lib.fp8kv_prefill_visible_plan(3, 2, 1, 1, 1, 0, 0, 0, out) != 0


DECODE = [A, 4096, A, A + 128, 16384, 256, 4096, 16384, 256, 4096, A, 4096, A, A, A, 64]
GEOMETRY = [2, 24, 4, 64, 16]                                # a head size that is refused
BY_WORDS = {
    "fp8kv_rope_append": (LEAD + [A, A, A] + TAIL, 0), "fp8kv_rope_append_bf16": (_lead(2) + [A] + TAIL, 0),
    "fp8kv_rope_append_blk": (LEAD + [A, A, A, A, 64, 64, 1] + TAIL, 0),
    "fp8kv_decode_attn_window": (DECODE + [A, A, 0.5] + GEOMETRY + [1, 0, 0, 64, 4, 100, 0], 2),
    "fp8kv_decode_attn_window_bf16": (DECODE + [0.5] + GEOMETRY + [1, 0, 0, 64, 4, 100, 0], 2),
    "fp8kv_decode_attn_blk": (DECODE + [A, 0.5] + GEOMETRY + [1, 0, 0, 64, 4, 100, 0], 2),
    "fp8kv_prefill_attn_window": (DECODE + [A, A, 0.5] + GEOMETRY + [64, 4, 10, 20, 0], 2),
    "fp8kv_prefill_attn_window_bf16": (DECODE + [0.5] + GEOMETRY + [64, 4, 10, 20, 0], 2),
    "fp8kv_prefill_attn_blk": (DECODE + [A, 0.5] + GEOMETRY + [64, 4, 10, 20, 0], 2),
}


@pytest.mark.parametrize("name", BY_WORDS)
def test_call_by_words(lib, name):
    """The call's own answer, and a refusal where the words are too few or one is too large for its argument."""
    args, code = BY_WORDS[name]
    types = _lib.SIGNATURES[name][1]
    assert len(types) == len(args)
    entry = lib.fp8kv_call_entry(name.encode())
    pack = struct.Struct("<" + "".join("f4x" if t is ctypes.c_float else "q" for t in types)).pack
    args = [0 if x is None else x for x in args]
    assert getattr(lib, name)(*args) == lib.fp8kv_call(entry, pack(*args), len(args)) == code
    assert lib.fp8kv_call(entry, pack(*args), len(args) - 1) == 1
    assert lib.fp8kv_call(entry, None, len(args)) == 1
    for i, t in enumerate(types):
        if t in (ctypes.c_int, ctypes.c_size_t):
            wrong = [(1 << 32) + args[i], -(1 << 40)] if t is ctypes.c_int else [-1]
            for x in wrong:
                assert lib.fp8kv_call(entry, pack(*args[:i], x, *args[i + 1:]), len(args)) == 1, (i, x)


def test_call_entries(lib):
    assert sorted(lib.fp8kv_call_entry(n.encode()) for n in BY_WORDS) == list(range(len(BY_WORDS)))
    assert lib.fp8kv_call_entry(b"fp8kv_cache_write") == lib.fp8kv_call_entry(None) == -1
    assert lib.fp8kv_call(len(BY_WORDS), b"", 0) == lib.fp8kv_call(-1, b"", 0) == 1


def test_wrappers_refuse_host_tensors():
    """The checks of the torch wrappers are native: tensors that are not on a device never reach the library."""
    from fp8kv_amd import ops
    x = torch.zeros(2, 4, 128, dtype=torch.bfloat16)
    kc, slots, i32 = torch.zeros(1, 16, 4, 128, dtype=torch.uint8), torch.zeros(2, dtype=torch.int64), torch.zeros(2, dtype=torch.int32)
    one, scales, table = torch.ones(1), torch.full((1, 1, 4, 2), 127, dtype=torch.uint8), torch.zeros(1, 1, dtype=torch.int32)
    for call in (lambda: ops.rope_append(x, x, x, kc, kc, None, None, slots, one, one),
                 lambda: ops.rope_append_blk(x, x, x, kc, kc, scales, None, None, i32, i32[:1], table),
                 lambda: ops.decode_attention_window(x, kc, kc, x, i32, i32[:1], table, one, one, 0.1, 4),
                 lambda: ops.decode_attention_blk(x, kc, kc, x, i32, i32[:1], table, scales, 0.1),
                 lambda: ops.prefill_attention_window(x, kc, kc, x, i32, i32[:1], table, one, one, 0.1, 4),
                 lambda: ops.prefill_attention_blk(x, kc, kc, x, i32, i32[:1], table, scales, 0.1, max_query_len=2)):
        with pytest.raises(ValueError, match="device tensor"):
            call()
    native = _lib.load_calls()
    for name in ("rope_append", "rope_append_blk", "decode", "decode_blk", "prefill", "prefill_blk"):
        with pytest.raises(TypeError, match="arguments"):
            getattr(native, name)(x, x)
    with pytest.raises(ValueError, match="tensor"):
        native.rope_append(0, 1, 0, None, 3, x, kc, kc, None, None, None, False, slots, one, one)
