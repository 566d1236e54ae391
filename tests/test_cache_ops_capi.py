"""Argument rejection of the append calls, before any launch (no GPU; the pointers are never followed)."""
import numpy as np
import pytest

from oracle import formats, rope_append

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
