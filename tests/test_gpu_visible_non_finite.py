"""NaN and infinities in what the visible-key attention calls read: they reach the rows that see them, as they do in the
formula, and no other row, head or element.

Finite elements are held to the bounds of test_gpu_visible.py, whose terms are taken from the case without the planted
value (a planted one enters a finite element's sums with weight 0 alone)."""
import pytest
import torch

from test_gpu_visible import D, KINDS, LONG, _case, _oracle, _run, _tolerance

pytestmark = pytest.mark.gpu

NAN, INF = float("nan"), float("inf")
# how a batch of two kv heads is cut: one split, several, more than the merge keeps in registers, parts of the batch
CUTS = {"one": dict(num_splits=1), "two": dict(num_splits=2), "five": dict(num_splits=5), "forty": dict(num_splits=40),
        "parts": dict(num_splits=40, max_seq_len=LONG)}
LENS = [(700, 1), (40, 1), (333, 1)]


def _plant(c, seq, token, head, element, value):
    """Sets element `element` (K below D, V from D on) of kv head `head` of a token.  e4m3: a code for NaN."""
    c["pool"] = c["pool"].clone()
    block = c["pool"].shape[2]
    code = value if c["kind"] == "bf16" else 0x7F if value != value else value
    c["pool"][int(c["table"][seq, token // block]), head, token % block, element] = code


def _agrees(got, want, tol):
    """NaN where it is wanted, the same infinities, and the rest within `tol`."""
    assert torch.equal(got.isnan(), want.isnan())
    inf = want.isinf()
    assert torch.equal(got[inf], want[inf])
    rest = want.isfinite()
    off = (got - want).abs()[rest] - tol[rest]
    assert (off <= 0).all(), f"worst by {off.max():.3g}"


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("cut", CUTS.values(), ids=CUTS.keys())
@pytest.mark.parametrize("window,sinks", [(0, 0), (200, 20)])
def test_decode_nan_in_keys_and_queries(kind, cut, window, sinks):
    """A NaN in one kv head's key makes that head's queries NaN, one in a query that query."""
    c = _case(kind, LENS, 8, 2, 16, window, sinks, seed=31)
    want, *bounds = _oracle(c)
    tol = _tolerance(c, "decode", want, *bounds)
    for token in (650, 5, 700):                           # inside the window, a first one, the newest
        if window and sinks <= token <= 700 - window:
            continue
        bad = dict(c, q=c["q"].clone())
        _plant(bad, 0, token, 1, 40, NAN)
        bad["q"][1, 2, 127] = NAN
        bad["q"][2, 7, 0] = INF                           # inf - inf, as K has elements of either sign
        then = want.clone()
        then[0, 4:] = then[1, 2] = then[2, 7] = NAN
        _agrees(_run(bad, "decode", **cut).double(), then, tol)


@pytest.mark.parametrize("cut", CUTS.values(), ids=CUTS.keys())
@pytest.mark.parametrize("window,sinks", [(0, 0), (200, 20)])
def test_decode_infinite_keys(cut, window, sinks):
    """A score of +inf makes its row NaN (inf - inf), one of -inf takes the key out of the sums."""
    c = _case("bf16", LENS, 8, 2, 16, window, sinks, seed=32)
    _plant(c, 0, 640, 0, 9, INF)
    _plant(c, 2, 333, 1, 70, -INF)
    want, mass, _ = _oracle(c)
    reach = _oracle(_case("bf16", LENS, 8, 2, 16, window, sinks, seed=32))[2]
    assert 0 < want.isnan().all(-1).sum() < 8             # some of either
    tol = _tolerance(c, "decode", want, mass, reach)
    _agrees(_run(c, "decode", **cut).double(), want, tol)


@pytest.mark.parametrize("cut", CUTS.values(), ids=CUTS.keys())
@pytest.mark.parametrize("window,sinks", [(0, 0), (200, 20)])
def test_decode_nan_scale(cut, window, sinks):
    """Every row that sees a key is NaN, a row that sees none zero."""
    lens = LENS + [(-1, 1)]
    for name in ("ks", "vs"):
        c = _case("fp8", lens, 8, 2, 16, window, sinks, seed=33)
        c[name] = NAN
        got = _run(c, "decode", **cut)
        assert got[:3].isnan().all() and (got[3] == 0).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("HQ,HKV", [(6, 1), (4, 4), (16, 2)])
def test_prefill_nan_in_queries(kind, HQ, HKV):
    """A NaN or an infinity in one query's head makes that row NaN and no other."""
    c = _case(kind, [(100, 60), (0, 20)], HQ, HKV, 16, 50, 4, seed=34)
    want, *bounds = _oracle(c)
    c["q"] = c["q"].clone()
    for row, head, element, value in ((3, 0, 0, NAN), (59, HQ - 1, 127, INF), (70, HQ // 2, 64, -INF)):
        c["q"][row, head, element] = value
        want[row, head] = NAN
    _agrees(_run(c, "prefill").double(), want, _tolerance(c, "prefill", want, *bounds))


@pytest.mark.parametrize("cut", CUTS.values(), ids=CUTS.keys())
@pytest.mark.parametrize("window,sinks", [(0, 0), (200, 20)])
def test_decode_infinite_values(cut, window, sinks):
    """An infinity in V is that infinity in its element of the output; two of either sign are NaN."""
    c = _case("bf16", LENS, 8, 2, 16, window, sinks, seed=35, spread=0.3)
    want, *bounds = _oracle(c)
    tol = _tolerance(c, "decode", want, *bounds)
    for value in (INF, -INF):
        bad = dict(c)
        _plant(bad, 0, 640, 1, D + 40, value)
        _plant(bad, 0, 12, 0, D + 3, value)
        _plant(bad, 1, 40, 0, D + 127, value)
        _plant(bad, 2, 300, 1, D, value)
        _plant(bad, 2, 180, 1, D, -value)
        then = want.clone()
        then[0, 4:, 40] = then[0, :4, 3] = then[1, :4, 127] = value
        then[2, 4:, 0] = NAN
        _agrees(_run(bad, "decode", **cut).double(), then, tol)


# e4m3 codes whose value times 2^(byte - 127) is 2^128 or more, the least of them first
TOO_LARGE = {247: (0x78, 0x7E), 248: (0x70, 0xF0, 0x7E), 250: (0x60, 0xFE), 254: (0x40, 0xC0, 0x7E)}


@pytest.mark.parametrize("byte", TOO_LARGE)
def test_values_past_32_bits_count_as_infinite(byte):
    """Elements of a block-scaled V that leave the range of 32 bits: infinite for the rows that see them, nothing for the
    others; the largest that stays within it is like any other."""
    for form, lens in (("prefill", [(0, 200)]), ("decode", [(199, 1)])):
        c = _case("blk", lens, 6, 1, 16, 48, 4, seed=36)
        token = 70 if form == "prefill" else 170
        c["pool"], c["scales"] = c["pool"].clone(), c["scales"].clone()
        block = int(c["table"][0, token // 16])
        c["pool"][block, :, :, D:] = 0
        c["scales"][block, :, :, 1] = byte
        want, *bounds = _oracle(c)
        tol = _tolerance(c, form, want, *bounds)
        first = 200 - c["q"].shape[0]
        t = torch.arange(first, 200)
        sees = (t >= token) & (t < token + 48)
        assert sees.any()
        for code in TOO_LARGE[byte]:
            bad = dict(c)
            _plant(bad, 0, token, 0, D + 40, code)
            _plant(bad, 0, token, 0, D + 41, 0x7F)
            then = want.clone()
            then[sees, :, 40] = -INF if code & 0x80 else INF
            then[sees, :, 41] = NAN
            _agrees(_run(bad, form).double(), then, tol)
        # the largest finite one, where only rows that do not see it are looked at, and finite for those that do
        bad = dict(c)
        _plant(bad, 0, token, 0, D + 40, (TOO_LARGE[byte][0] & 0x7F) - 1)
        got = _run(bad, form).double()
        assert ((got - want).abs() <= tol)[~sees].all() and not got[sees].isnan().any()
