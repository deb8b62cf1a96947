"""The cache in pages, the attention over it, probabilities and verification where their inputs contradict themselves or reach the ends of their ranges."""
import ctypes as C
from fractions import Fraction

import numpy as np
import pytest

import paged_plain as pp
import quant_np as qn
from conftest import load_pkg
from device_data import Dev
from paged_plain import BF16, E4M3, F16, F32, I8
from test_paged_gpu import Step, error_word, padded, run_verify

pytestmark = pytest.mark.gpu
pkg = load_pkg()

BACKWARDS = [([10, 12, 0, 5], [100, 30, 40]), ([0, 3, 50, 60, 20, 100], [9, 60, 70, 30, 300]), ([0, 40, 8, 9], [41, 3, 200])]


# ---- starts that decrease ---------------------------------------------------------------------

@pytest.mark.parametrize("kind", [BF16, I8], ids=pp.NAMES.get)
@pytest.mark.parametrize("starts,lens", BACKWARDS + [([5, 0], [64])])
def test_an_append_whose_starts_decrease_leaves_old_rows_alone(gpu, kind, starts, lens):
    """A row is looked up by its number among the starts: where they decrease it must not be taken for a row of a sequence that does not hold it."""
    rng = np.random.default_rng(len(starts))
    c = pp.Cache(rng, lens, 2, 64, kind, 16).fill(rng)
    tokens = max(starts)
    before = [x.copy() for x in c.data + c.scales]
    with Dev(gpu) as d:
        a = c.upload(d, starts)
        x = rng.standard_normal((tokens, 128)).astype(np.float32) * 9
        pkg.check(gpu.lib.lv_paged_append(gpu.handle, C.byref(a), d.f32(x), d.f32(-x), F32, 128, None, 0, 0, tokens))
        error_word(gpu)
        data, scales = c.download(gpu)
    for s, n in enumerate(lens):                                         # (the new places of the sequences that are in order may be written)
        m = starts[s + 1] - starts[s]
        if 0 < m <= n:
            p, r = c.place(s, np.arange(n - m, n))
            for old, got in zip(before, data + scales):
                old[p, :, r] = got[p, :, r]
    for old, got in zip(before, data + scales):
        assert np.array_equal(old, got, equal_nan=old.dtype == np.float32)


@pytest.mark.parametrize("out", [F32, BF16], ids=["to-f32", "to-bf16"])
@pytest.mark.parametrize("window", [0, 64])
@pytest.mark.parametrize("starts,lens", BACKWARDS)
def test_an_attention_whose_starts_decrease_stays_inside_its_scratch(gpu, starts, lens, window, out):
    """The parts of a row are joined by its number of parts, which a sequence that does not hold the row does not know."""
    rng = np.random.default_rng(len(starts))
    lens = [n + 3000 for n in lens]                                      # (several parts)
    c = pp.Cache(rng, lens, 1, 64, BF16, 16).fill(rng)
    tokens = max(starts)
    with Dev(gpu) as d:
        st = Step(d, c, [tokens], 4, out=out, window=window, behind=0, max_new=tokens, max_len=max(lens))
        st.a.cache = c.upload(d, starts)
        st.bytes = gpu.lib.lv_paged_attention_scratch_bytes(gpu.handle, C.byref(st.a))
        guard = 4096
        st.scratch = d.up(np.full(st.bytes + guard, 0xFF, np.uint8))
        st.launch()
        error_word(gpu)
        got = pp.values(gpu.download(st.dout, st.blank.dtype, st.blank.size), out).reshape(tokens, st.ld)
        assert (gpu.download(st.scratch, np.uint8, st.bytes + guard)[st.bytes:] == 0xFF).all()
    held = np.zeros(tokens, bool)
    for a, b in zip(starts, starts[1:]):
        if a < b:
            held[a:b] = True
    assert (got[~held] == -7.0).all() and (got[:, 4 * 64:] == -7.0).all()


# ---- what an append is told ---------------------------------------------------------------------

@pytest.mark.parametrize("seqs", [3, 700])
@pytest.mark.parametrize("change", ["beyond the rows", "too long", "before the beginning", "behind all rows"])
def test_an_append_reports_every_sequence_that_contradicts_itself(gpu, seqs, change):
    """One of them; the others are written, also where no row of the step is the bad one's."""
    rng = np.random.default_rng(seqs)
    lens, new = rng.integers(1, 40, seqs), rng.integers(0, 2, seqs)
    new[-1] = 1
    lens[-1] = 20
    c = pp.Cache(rng, lens, 1, 64, E4M3, 8).fill(rng)
    starts = np.cumsum([0] + list(new))
    tokens, told, bad = int(starts[-1]), lens.copy(), seqs - 1
    if change == "beyond the rows":                                      # the last sequence's only row
        tokens -= 1
    elif change == "too long":
        bad = int(np.argmin(new))                                        # (no new token: nothing else looks at it)
        told[bad] = c.width * 8 + 1
        assert new[bad] == 0
    elif change == "before the beginning":
        told[bad] = 0
    else:
        starts[-1] = 0xFFFFFFF0
        told[bad] = 5
    x = rng.standard_normal((max(tokens, 1), 64)).astype(np.float32)
    with Dev(gpu) as d:
        a = c.upload(d, starts, told)
        pkg.check(gpu.lib.lv_paged_append(gpu.handle, C.byref(a), d.f32(x), d.f32(-x), F32, 64, None, 0, 0, tokens))
        error_word(gpu)
        data, scales = c.download(gpu)
    for s in range(seqs):
        if s != bad and new[s]:
            c.write(s, [lens[s] - 1], 0, x[starts[s]].reshape(1, 1, 64))
            c.write(s, [lens[s] - 1], 1, -x[starts[s]].reshape(1, 1, 64))
    for want, got in zip(c.data + c.scales, data + scales):
        assert np.array_equal(want, got, equal_nan=want.dtype == np.float32)


# ---- what is behind a contradiction -----------------------------------------------------------------

def contradictions(d):
    """The paged calls that find their data at odds, by name: each reports and is otherwise in order."""
    rng = np.random.default_rng(1)
    c = pp.Cache(rng, [20, 30], 1, 64, BF16, 16).fill(rng)
    a = c.upload(d, [0, 1, 2], [c.width * 16 + 1, 30])
    x, out = d.f32(rng.standard_normal((2, 64))), d.zeros(2 * 30 * 64 * 4)
    lib, h = d.gpu.lib, d.gpu.handle
    few, many = Step(d, c, [1, 1], 1, behind=0), Step(d, c, [20, 30], 2, behind=0)
    for st in (few, many):
        st.a.cache.lens = a.lens
    v = pkg.VerifyArgs(target=d.f32(np.full((1, 8), 0.125)).value, target_ld=8, vocab=8, drafted=d.u32([0]).value, starts=d.u32([0, 1]).value, seqs=1, rows=1, accept=d.f32([0.5]).value,
                       pick=d.f32([2.0]).value, tokens=d.u32([0]).value, accepted=d.u32([0]).value)
    return {"append": lambda: lib.lv_paged_append(h, C.byref(a), x, x, F32, 64, None, 0, 0, 2), "read": lambda: lib.lv_paged_read(h, C.byref(a), out, out, F32, 30 * 64, 0, 64, 0, 30),
            "attention of few rows": lambda: few.launch() and 0, "attention of many": lambda: many.launch() and 0, "verification": lambda: lib.lv_verify_drafts(h, C.byref(v))}


@pytest.mark.parametrize("call", ["append", "read", "attention of few rows", "attention of many", "verification"])
def test_a_contradiction_does_not_end_the_waits_of_what_follows(gpu, call):
    """A product whose activations come behind a long launch: all of its rows are there, although a sequence of the step was left out."""
    rows, cols, batch, lib, h = 23680, 1024, 40, gpu.lib, gpu.handle
    rng = np.random.default_rng(70)
    W = np.tile(qn.quantize((rng.standard_normal((32, cols)) * 0.02).astype(np.float32), qn.Q8_0).reshape(32, -1), (rows // 32, 1))
    x, n = rng.standard_normal((batch, cols)).astype(np.float32), 1 << 23
    with Dev(gpu) as d:
        dW, dx, xh, long_row, norm, out = d.up(W), d.f32(x), d.zeros(lib.lv_act_split_bytes(cols, batch)), d.zeros(n * 4), d.zeros(n * 4), d.zeros(batch * rows * 4)
        pkg.check(lib.lv_act_split_f16(h, xh, dx, None, cols, batch))
        pkg.check(lib.lv_gemm_tc(h, out, dW, qn.Q8_0, xh, rows, cols, batch, 0))
        gpu.sync()
        want = d.get(out, (batch, rows))
        bad = contradictions(d)[call]
        gpu.sync()
        pkg.check(lib.lv_memset(h, out, 255, batch * rows * 4))
        pkg.check(bad())
        pkg.check(lib.lv_norm_f32(h, norm, long_row, long_row, n, 1))    # one thread block
        pkg.check(lib.lv_gemm_tc(h, out, dW, qn.Q8_0, xh, rows, cols, batch, 0))
        error_word(gpu)
        assert np.array_equal(d.get(out, (batch, rows)), want)


@pytest.mark.parametrize("kind", [BF16, E4M3], ids=pp.NAMES.get)
@pytest.mark.parametrize("lens,new", [([9000, 40, 12001], [70, 40, 33]), ([2500], [900])], ids=["split", "whole"])
def test_an_earlier_index_out_of_range_does_not_end_the_waits_of_many_rows(gpu, kind, lens, new):
    rng = np.random.default_rng(len(lens))
    c = pp.Cache(rng, lens, 1, 64, kind, 64).fill(rng)
    with Dev(gpu) as d:
        st = Step(d, c, new, 2, out=F16)
        cache, row = d.zeros(128), d.f32(np.zeros(64))
        pkg.check(gpu.lib.lv_kv_append_f16(gpu.handle, cache, row, d.u32([8]), 64, 1, 1))        # row 8 of a cache of one row
        st.launch()
        error_word(gpu)
        st.check()


# ---- verification: the bounds between runs --------------------------------------------------------

def sums_by_halves(s):
    """Running sums in float64 that add up in pairs of runs, so that each has brackets of its own."""
    run, o = [float(x) for x in s], 1
    while o < len(run):
        run = [run[i] + run[i - o] if i >= o else run[i] for i in range(len(run))]
        o *= 2
    return run


def rows_with_a_gap():
    """(weights of 16 runs, weights behind them, run): half of the whole weight is the running sum behind `run`, where the next one, without any weight, has a larger one by halves."""
    cases = []
    for seed in range(400):
        rng = np.random.default_rng(seed)
        s = (rng.random(16) * 2.0 ** rng.integers(-40, 0, 16)).astype(np.float32)
        s[rng.integers(8, 15):] = 0
        p = sums_by_halves(s)
        for i in range(15):
            if s[i + 1] == 0 and p[i + 1] > p[i]:
                rest, left = [], 2 * p[i] - p[15]
                for _ in range(3):
                    h = np.float32(left)
                    h = np.nextafter(h, np.float32(0)) if float(h) > left else h
                    rest.append(h)
                    left -= float(h)
                if left == 0 and p[15] + (2 * p[i] - p[15]) == 2 * p[i]:
                    cases.append((s, rest, i))
                break
    return cases


def test_a_pick_between_two_runs_draws_a_token(gpu):
    """Each warp sums a run of 128 values (a vocabulary of 16384 is 8 x 16 of them) and asks whether the target lies in its run: between the bounds of one and the next there
    must be no gap, and none at all around a run without weight."""
    cases = rows_with_a_gap()
    assert len(cases) > 30
    target = np.zeros((len(cases), 16384), np.float32)
    for row, (s, rest, _) in zip(target, cases):
        row[np.arange(16) * 128] = s
        row[np.arange(16, 16 + len(rest)) * 128] = rest
    n = len(cases)
    accepted, tokens, _, failed = run_verify(gpu, target, None, np.zeros(n, np.uint32), np.arange(n + 1), np.zeros(n, np.float32), np.full(n, 0.5, np.float32))
    assert failed is None and (accepted == 0).all()
    for row, token in zip(target, tokens):
        assert token < 16384 and row[token] > 0                          # (77 where nothing was written)
        before = sum((Fraction(float(x)) for x in row[:token]), Fraction(0))
        whole = sum((Fraction(float(x)) for x in row), Fraction(0))
        slack = whole / 2 ** 50                                          # (19 additions of 2^-53 each)
        assert before <= whole / 2 + slack and before + Fraction(float(row[token])) > whole / 2 - slack


# ---- probabilities: temperatures at the ends --------------------------------------------------------

@pytest.mark.parametrize("vocab", [1, 50, 32000, 40001, 300002])
@pytest.mark.parametrize("rows", [1, 60])
def test_probabilities_at_the_largest_temperatures(gpu, vocab, rows):
    """A temperature without end leaves no differences but that -infinity has no weight; 3e38 next to none."""
    x = (np.random.default_rng(vocab).standard_normal((rows, vocab)) * 5).astype(np.float32)
    if vocab > 1:
        x[:, ::3] = -np.inf
        x[:, 1] = 1e30
    there = np.isfinite(x)
    want = there / there.sum(1, keepdims=True)
    with Dev(gpu) as d:
        dx = d.f32(x)
        for T in (np.inf, 3e38, 1.5e38):
            out = d.zeros(x.nbytes)
            d.call("lv_probabilities", out, vocab, dx, vocab, vocab, rows, d.f32(np.full(rows, T)))
            got = d.get(out, x.shape)
            # exponents are at most 1e30 / 1.5e38 < 2^-26; equal values sum to whole numbers of up to 2^24 in any order, the quotient is rounded twice
            assert (got[~there] == 0).all() and (np.abs(got - want) <= 2.0 ** -22 * want).all()


def test_temperatures_that_are_none(gpu):
    """Negative or not a number: not a number, beside rows that are in order; minus zero is zero."""
    for vocab in (700, 200001):
        x = np.random.default_rng(vocab).standard_normal((5, vocab)).astype(np.float32)
        x[1, 3] = -np.inf
        with Dev(gpu) as d:
            out = d.zeros(x.nbytes)
            d.call("lv_probabilities", out, vocab, d.f32(x), vocab, vocab, 5, d.f32([np.nan, -1.0, -np.inf, -0.0, 1.0]))
            got = d.get(out, x.shape)
        assert np.isnan(got[:3]).all()
        assert got[3, x[3].argmax()] == 1.0 and got[3].sum() == 1.0
        e = np.exp(x[4].astype(np.float64) - x[4].max())
        assert np.abs(got[4] - e / e.sum()).max() <= 1e-6


@pytest.mark.parametrize("vocab", [1, 3, 700, 32000, 40001, 300002])
def test_the_first_minus_infinity_of_a_row_without_numbers(gpu, vocab):
    """At temperature 0 it is the maximum of a row of -infinity and NaN, wherever it lies, also where the values of a thread end behind it."""
    places = sorted({0, vocab // 3, vocab // 2, vocab - 2, vocab - 1} & set(range(vocab)))
    x = np.full((len(places) + 1, vocab), np.nan, np.float32)
    for r, at in enumerate(places):
        x[r, at:] = np.where(np.arange(vocab - at) % 2 == 0, -np.inf, np.nan)
    with Dev(gpu) as d:
        out = d.zeros(x.nbytes)
        d.call("lv_probabilities", out, vocab, d.f32(x), vocab, vocab, len(x), d.f32(np.zeros(len(x))))
        got = d.get(out, x.shape)
    want = np.zeros(x.shape)
    want[np.arange(len(x)), places + [0]] = 1.0
    assert np.array_equal(got, want)


# ---- verification: lengths ----------------------------------------------------------------------------

def test_lengths_shorter_than_what_is_rejected(gpu):
    """They stay as they are and are reported; the tokens are drawn all the same, and other sequences' lengths shortened."""
    target, draft = np.full((9, 16), 1 / 16, np.float32), np.full((9, 16), 1 / 16, np.float32)
    draft[:, 3] = 1.0
    starts, drafted, accept = [0, 4, 8, 9], np.full(9, 3, np.uint32), np.full(9, 0.9, np.float32)        # (0.9 is above 1 / 16: all rejected)
    for lens, want, wrong in (([2, 10, 0], [2, 7, 0], True), ([3, 3, 0], [0, 0, 0], False)):
        n, t, left, failed = run_verify(gpu, target, draft, drafted, starts, accept, np.full(3, 0.5, np.float32), lens)
        assert list(n) == [0, 0, 0] and list(left) == want and failed == (pkg.LV_ERR_DEVICE_WAIT if wrong else None)
        assert (t[[0, 4, 8]] < 16).all() and (t[[1, 2, 3, 5, 6, 7]] == 0xFFFFFFFF).all()


# ---- attention: as many bits as the header says --------------------------------------------------------

def attend_tight(c, starts, q, heads, scale, out_kind, uq, up, terms, angles=None):
    """(out, bound) like paged_plain.attend, for queries and weights whose relative errors are at most uq and up, and queries with `terms` values that are not zero.

    A product of |q| |k| is exact in f32 where one number has 8 or 11 bits and within 2^-24 elsewhere, `terms` products and planes add up with one rounding of the running sum each, the
    factors take four more: a score is off by d = (uq + (3 terms + 8) 2^-24) scale sum |q| |k|; f16 queries also by 2^-25 of the row's largest value per key value (they are
    whole multiples of that).  A quotient of weights is off by 2 d, by 2^-22 |s| + 2^-19 for the exponentials, and n 2^-24 for the sums; the numerator's weights by up, f16 weights also by 2^-35 of the
    largest one each (see paged_plain).  Together times sum p |v|, and the rounding of the result."""
    x = pp.rotate(q, angles).astype(np.float64)
    G, dim = heads // c.H, c.dim
    out, bound = np.zeros((2,) + x.shape)
    for s, n in enumerate(c.lens):
        m = int(starts[s + 1]) - int(starts[s])
        k, v = (c.read(s, np.arange(n), w) for w in range(2))
        for i in range(m):
            t, at = int(starts[s]) + i, n - m + i
            for h in range(heads):
                kk, vv = k[:at + 1, h // G], v[:at + 1, h // G]
                z = scale * (kk @ x[t, h])
                p = np.exp(z - z.max())
                p /= p.sum()
                size = scale * (np.abs(kk) @ np.abs(x[t, h])).max()
                d = (uq + (3 * terms + 8) * 2.0 ** -24) * size
                floor = 0.0
                if c.kind != BF16:
                    d += 2.0 ** -25 * scale * np.abs(x[t, h]).max() * np.abs(kk).sum(1).max()
                    floor = len(z) * 2.0 ** -35 * np.abs(vv).max()
                out[t, h] = p @ vv
                bound[t, h] = floor + (np.expm1(2 * d) + up + 2.0 ** -19 + 2.0 ** -22 * size + len(z) * 2.0 ** -24) * (p @ np.abs(vv))
    bound += pp.HALF_STEP[out_kind] * (np.abs(out) + bound) + 1e-30 + (2.0 ** -25 if out_kind == F16 else 0)
    return out, bound


@pytest.mark.parametrize("out", [BF16, F16], ids=["to-bf16", "to-f16"])
@pytest.mark.parametrize("scale", [None, 0.1, 0.9])
def test_queries_that_fit_enter_many_rows_unrounded(gpu, out, scale):
    """bf16 queries without a rotation over a bf16 cache: the scale is applied to the scores, so that large ones are off by the sums' roundings alone."""
    rng = np.random.default_rng(9)
    c = pp.Cache(rng, [160, 90], 1, 64, BF16, 16).fill(rng)
    with Dev(gpu) as d:
        st = Step(d, c, [50, 40], 2, out=out, given=BF16, size=30.0 * 0.125 / (scale or 0.125), scale=scale, behind=0)
        got = st.launch().result()
        want, bound = attend_tight(c, st.starts, st.q.reshape(90, 2, 64), 2, st.scale, out, 0.0, pp.HALF_STEP[BF16], 64)
        worst = (np.abs(got - want) / bound).max()
        assert worst <= 1.0, worst


@pytest.mark.parametrize("kind", [F16, BF16, I8], ids=pp.NAMES.get)
@pytest.mark.parametrize("new", [2, 50])
@pytest.mark.parametrize("out", [F32, BF16], ids=["to-f32", "to-bf16"])
@pytest.mark.parametrize("scale", [1e-45, 1e-30, 3e38])
def test_rows_of_zeros_at_any_scale(gpu, kind, new, out, scale):
    """All scores are zero: the mean of the values, whatever the scale."""
    rng = np.random.default_rng(new)
    c = pp.Cache(rng, [140], 1, 64, kind, 16).fill(rng)
    with Dev(gpu) as d:
        st = Step(d, c, [new], 2, out=out, scale=scale, size=0.0, behind=0)
        got = st.launch().result()
        want, bound = attend_tight(c, st.starts, st.q.reshape(new, 2, 64), 2, st.scale, out, 0.0, pp.HALF_STEP[BF16 if kind == BF16 else F16], 64)
        assert (np.abs(got - want) <= bound).all()


# relative error of what enters the products for up to 32 rows: the numbers that a value enters as leave 2^-11 (f16) or 2^-8 (bf16) of it each
FEW = {(BF16, F32): 2.0 ** -24, (BF16, BF16): 2.0 ** -16, (BF16, F16): 2.0 ** -16, (F16, F32): 2.0 ** -22, (F16, F16): 2.0 ** -22, (F16, BF16): 2.0 ** -11, (I8, F32): 2.0 ** -22,
       (I8, F16): 2.0 ** -11, (I8, BF16): 2.0 ** -11, (E4M3, F32): 2.0 ** -22, (E4M3, F16): 2.0 ** -11, (E4M3, BF16): 2.0 ** -11}


@pytest.mark.parametrize("kind,out", FEW, ids=[f"{pp.NAMES[k]}-to-{pp.NAMES[o]}" for k, o in FEW])
@pytest.mark.parametrize("size", [0.3, 150.0])
def test_few_rows_have_the_bits_that_the_header_states(gpu, kind, out, size):
    """Queries of two values, so that sums hide nothing: with large scores a number that is missing from the queries shows, with small ones and few keys one that is
    missing from the weights."""
    rng = np.random.default_rng(31)
    lens = [2, 3, 4, 3, 2, 4, 5, 7] * 3
    c = pp.Cache(rng, lens, 1, 64, kind, 16).fill(rng)
    u = FEW[kind, out]
    with Dev(gpu) as d:
        st = Step(d, c, [1] * len(lens), 4, out=out, size=size, behind=0)
        q = st.q.reshape(len(lens), 4, 64)
        q[..., [i for i in range(64) if i not in (3, 40)]] = 0
        st.a.q = d.up(padded(q.reshape(len(lens), -1), st.ld, F32, 0.0)).value
        got = st.launch().result()
        want, bound = attend_tight(c, st.starts, q, 4, st.scale, out, u, u, 2)
        worst = (np.abs(got - want) / bound).max()
        assert worst <= 1.0, worst


def test_f32_results_of_many_rows_have_them_too(gpu):
    rng = np.random.default_rng(32)
    for kind in (F16, BF16, I8, E4M3):
        c = pp.Cache(rng, [60, 9], 1, 64, kind, 16).fill(rng)
        with Dev(gpu) as d:
            st = Step(d, c, [40, 9], 4, out=F32, size=20.0, behind=0)
            q = st.q.reshape(49, 4, 64)
            q[..., 2:] = 0
            st.a.q = d.up(padded(q.reshape(49, -1), st.ld, F32, 0.0)).value
            got = st.launch().result()
            want, bound = attend_tight(c, st.starts, q, 4, st.scale, F32, FEW[kind, F32], FEW[kind, F32], 2)
            assert (np.abs(got - want) <= bound).all()


# ---- where the kernels of few rows and of many meet -------------------------------------------------

@pytest.mark.parametrize("kind", [BF16, F16, I8, E4M3], ids=pp.NAMES.get)
@pytest.mark.parametrize("rows", [24, 32, 33, 40, 95, 96, 97, 98, 128, 129])
def test_rows_on_both_sides_of_the_kernels_border(gpu, kind, rows):
    """One query head, so that rows are tokens; a second sequence has a row of its own, a third none."""
    rng = np.random.default_rng(rows)
    c = pp.Cache(rng, [rows + 70, 40, 9], 1, 128, kind, 16).fill(rng)
    with Dev(gpu) as d:
        for out in (BF16, F16):
            Step(d, c, [rows, 1, 0], 1, out=out, pairs=32, sink=out == F16).launch().check()


@pytest.mark.parametrize("kind", [I8, E4M3], ids=pp.NAMES.get)
@pytest.mark.parametrize("page,dim,heads,H,lens,new", [(8, 16, 4, 1, [90, 40], [31, 25]), (24, 48, 4, 2, [200, 1, 60], [70, 1, 35]), (40, 112, 4, 1, [700], [33]), (128, 128, 1, 1, [129, 128], [129, 128]),
                                                       (256, 64, 5, 1, [600, 34], [60, 7]), (8, 128, 8, 2, [1, 300, 0, 257], [1, 64, 0, 65]), (16, 80, 1, 1, [1300], [100])])
def test_many_rows_of_8_bit_pages(gpu, kind, page, dim, heads, H, lens, new):
    """More than 96 rows of the longest: boxes of 8 to 128 rows, head sizes that do not fill a block of columns, windows that begin inside a box."""
    rng = np.random.default_rng(page + dim)
    c = pp.Cache(rng, lens, H, dim, kind, page).fill(rng)
    with Dev(gpu) as d:
        for window, out in ((0, BF16), (37, F16)):
            Step(d, c, new, heads, out=out, window=window, sink=bool(window), pairs=dim // 2 if window else 0).launch().check()


@pytest.mark.parametrize("rows", [24, 25, 37, 38])
@pytest.mark.parametrize("vocab", [65536, 65540, 70001, 131072, 200000])
def test_probabilities_on_both_sides_of_the_clusters_border(gpu, rows, vocab):
    rng = np.random.default_rng(rows)
    x = (rng.standard_normal((rows, vocab)) * 4).astype(np.float32)
    with Dev(gpu) as d:
        out = d.zeros(x.nbytes)
        d.call("lv_probabilities", out, vocab, d.f32(x), vocab, vocab, rows, None)
        got = d.get(out, x.shape)
    z = x.astype(np.float64) - x.max(1, keepdims=True).astype(np.float64)
    e = np.exp(z)
    e /= e.sum(1, keepdims=True)
    # an exponential's argument is off by 2^-22 of itself, the exponential by 2^-22, the sum by the mean of both and its longest chain of additions
    tol = np.abs(z) * 2.0 ** -22 + 2.0 ** -22 + (np.abs(z) * e).sum(1, keepdims=True) * 2.0 ** -22 + (128 + vocab / 1024) * 2.0 ** -24
    assert (np.abs(got - e) <= tol * e).all()


# ---- the largest and the most, and what is recorded ----------------------------------------------------

def test_the_most_sequences(gpu):
    """65535 of one position each: a result is the value itself."""
    n, dim = 65535, 16
    rng = np.random.default_rng(5)
    k, v, q = (rng.standard_normal((n, dim)).astype(np.float32) for _ in range(3))
    v = pp.rounded(v, F16)
    with Dev(gpu) as d:
        cache = pkg.PagedCache(k=d.zeros(n * dim * 2).value, v=d.zeros(n * dim * 2).value, type=F16, pages=n, page_rows=1, kv_heads=1, dim=dim, table=d.u32(rng.permutation(n)).value, table_ld=1,
                               lens=d.u32(np.ones(n)).value, starts=d.u32(np.arange(n + 1)).value, seqs=n)
        d.call("lv_paged_append", C.byref(cache), d.f32(k), d.f32(v), F32, dim, None, 0, 0, n)
        out = d.zeros(n * dim * 4)
        a = pkg.PagedAttentionArgs(cache=cache, q=d.f32(q).value, q_type=F32, q_ld=dim, heads=1, tokens=n, max_new=1, max_len=1, scale=0.25, out=out.value, out_type=F32, out_ld=dim)
        nbytes = gpu.lib.lv_paged_attention_scratch_bytes(gpu.handle, C.byref(a))
        d.call("lv_paged_attention", C.byref(a), d.zeros(nbytes), nbytes)
        # a weight of 2^10 is exact, the quotient is rounded twice
        assert (np.abs(d.get(out, (n, dim)) - v) <= 2.0 ** -22 * np.abs(v)).all()


@pytest.mark.parametrize("kind", [F16, I8], ids=pp.NAMES.get)
@pytest.mark.parametrize("new", [1, 3, 200])
def test_positions_near_the_largest(gpu, kind, new):
    """One page of 2^20 rows that a table names 2047 times, and a window over the last positions below 2^31."""
    page, dim, slots, window = 1 << 20, 16, 2047, 70
    length = slots * page
    rng = np.random.default_rng(new)
    width = new + window - 1
    x, v = (rng.standard_normal((width, 1, dim)).astype(np.float32) for _ in range(2))
    eight = kind in pp.TOP
    with Dev(gpu) as d:
        bufs = [d.zeros(page * dim * (1 if eight else 2)) for _ in range(2)] + [d.zeros(page * 4) for _ in range(2)]
        lens = d.u32([length])
        cache = pkg.PagedCache(k=bufs[0].value, v=bufs[1].value, k_scale=bufs[2].value if eight else None, v_scale=bufs[3].value if eight else None, type=kind, pages=1, page_rows=page, kv_heads=1,
                               dim=dim, table=d.u32(np.zeros(slots)).value, table_ld=slots, lens=lens.value, starts=d.u32([0, width]).value, seqs=1)
        d.call("lv_paged_append", C.byref(cache), d.f32(x), d.f32(v), F32, dim, None, 0, 0, width)
        c = pp.Cache(rng, [width], 1, dim, kind, 256)                    # the same rows as a short sequence
        c.write(0, np.arange(width), 0, x)
        c.write(0, np.arange(width), 1, v)
        for out in (F32, BF16):
            q = rng.standard_normal((new, 1, dim)).astype(np.float32)
            to = d.zeros(new * dim * 4)
            cache.starts = d.u32([0, new]).value
            a = pkg.PagedAttentionArgs(cache=cache, q=d.f32(q).value, q_type=F32, q_ld=dim, heads=1, tokens=new, max_new=new, max_len=length, scale=0.25, window=window, out=to.value, out_type=out,
                                       out_ld=dim)
            nbytes = gpu.lib.lv_paged_attention_scratch_bytes(gpu.handle, C.byref(a))
            d.call("lv_paged_attention", C.byref(a), d.zeros(nbytes), nbytes)
            got = pp.values(gpu.download(to, np.float32 if out == F32 else np.uint16, new * dim), out).reshape(new, 1, dim)
            want, bound = pp.attend(c, [0, new], q, 1, 0.25, window, out_kind=out)
            assert (np.abs(got - want) <= bound).all()


def test_the_largest_vocabulary(gpu):
    n = 1 << 24
    rng = np.random.default_rng(24)
    x = rng.standard_normal((2, n)).astype(np.float32)
    with Dev(gpu) as d:
        p = d.zeros(2 * n * 4)
        d.call("lv_probabilities", p, n, d.f32(x), n, n, 2, None)
        got = d.get(p, (2, n))
    e = np.exp(x.astype(np.float64))
    e /= e.sum(1, keepdims=True)
    assert np.abs(got / e - 1).max() <= 2.0 ** -18                      # (arguments of at most 11 in magnitude, sums of 2^20 terms in chains of 2^11)
    drafted, accept, pick = np.array([n - 1, 0], np.uint32), np.array([0.999, 0.0], np.float32), np.array([0.73], np.float32)
    draft = np.zeros((2, n), np.float32)
    draft[0, n - 1] = 1.0
    k, t, _, failed = run_verify(gpu, got, draft, drafted, [0, 2], accept, pick)
    assert failed is None and list(k) == [0]
    cum = np.cumsum(np.maximum(got[0].astype(np.float64) - draft[0], 0))
    at = int(t[0])
    assert cum[at] > 0.73 * cum[-1] * (1 - 1e-6) and (at == 0 or cum[at - 1] <= 0.73 * cum[-1] * (1 + 1e-6))
    k, t, _, failed = run_verify(gpu, got, None, drafted, [0, 2], np.zeros(2, np.float32), pick)
    assert failed is None and list(k) == [1] and t[0] == n - 1


@pytest.mark.parametrize("rows,vocab", [(3, 200), (5, 70001), (20, 140000), (60, 33000)])
def test_probabilities_and_verification_in_a_recorded_step(gpu, rows, vocab):
    """Recorded once, replayed with other logits, drafts, random numbers and lengths."""
    rng = np.random.default_rng(vocab)
    starts = np.array([0, rows // 2, rows])
    lib, h = gpu.lib, gpu.handle
    with Dev(gpu) as d:
        dx, dp, dt = d.zeros(rows * vocab * 4), d.zeros(rows * vocab * 4), d.f32(np.full(rows, 0.8))
        drafted, accept, pick, tok, acc, lens = d.zeros(rows * 4), d.zeros(rows * 4), d.zeros(8), d.zeros(rows * 4), d.zeros(8), d.zeros(8)
        a = pkg.VerifyArgs(target=dp.value, target_ld=vocab, vocab=vocab, drafted=drafted.value, starts=d.u32(starts).value, seqs=2, rows=rows, accept=accept.value, pick=pick.value,
                           tokens=tok.value, accepted=acc.value, lens=lens.value)
        pkg.check(lib.lv_graph_begin_capture(h))
        pkg.check(lib.lv_probabilities(h, dp, vocab, dx, vocab, vocab, rows, dt))
        pkg.check(lib.lv_verify_drafts(h, C.byref(a)))
        g = C.c_void_p()
        pkg.check(lib.lv_graph_end_capture(h, C.byref(g)))
        for step in range(3):
            x = (rng.standard_normal((rows, vocab)) * 3).astype(np.float32)
            drafts, u, picks = x.argmax(1).astype(np.uint32), rng.random(rows).astype(np.float32) * np.float32(0.3), rng.random(2).astype(np.float32)
            for b, host in ((dx, x), (drafted, drafts), (accept, u), (pick, picks), (lens, np.full(2, 100, np.uint32))):
                pkg.check(lib.lv_upload(h, b, np.ascontiguousarray(host).ctypes.data_as(C.c_void_p), host.nbytes))
            pkg.check(lib.lv_graph_launch(h, g))
            gpu.sync()
            p = d.get(dp, (rows, vocab))
            z = x.astype(np.float64) / np.float64(np.float32(0.8))
            e = np.exp(z - z.max(1, keepdims=True))
            e /= e.sum(1, keepdims=True)
            assert (np.abs(p - e) <= (40 * 2.0 ** -21 + (128 + vocab / 1024) * 2.0 ** -24) * e + 1e-37).all()          # (arguments of at most 40 in magnitude, see test_probabilities)
            wn, wt = pp.verify(p, None, drafts, starts, u, picks)
            n = gpu.download(acc, np.uint32, 2)
            assert np.array_equal(n, wn) and np.array_equal(gpu.download(tok, np.uint32, rows), wt)
            assert np.array_equal(gpu.download(lens, np.uint32, 2), 100 - (np.diff(starts) - 1 - wn))
        lib.lv_graph_destroy(g)


@pytest.mark.parametrize("kind", [I8, E4M3], ids=pp.NAMES.get)
@pytest.mark.parametrize("out", [F32, BF16], ids=["to-f32", "to-bf16"])
@pytest.mark.parametrize("new", [3, 120])
@pytest.mark.parametrize("times", [12, 20])
def test_values_far_below_another_rows(gpu, kind, out, new, times):
    """The last position's values are 2^12 or 2^20 times the others', which all tokens before it do not see: weights are whole multiples of 2^-35 of the largest in units of the largest scale,
    which leaves 11 bits at 2^20 and 22 at 2^12."""
    rng = np.random.default_rng(times)
    c = pp.Cache(rng, [300], 1, 64, kind, 16).fill(rng)
    c.write(0, [299], 1, np.float32(2.0 ** times) * rng.standard_normal((1, 1, 64)).astype(np.float32))
    with Dev(gpu) as d:
        st = Step(d, c, [new], 1, out=out, behind=0)
        got = st.launch().result()
        u = 2.0 ** -22 if out == F32 else 2.0 ** -11
        want, bound = attend_tight(c, st.starts, st.q.reshape(new, 1, 64), 1, st.scale, out, u, u, 64)
        largest = np.abs(c.read(0, np.arange(300), 1)).max()
        assert (np.abs(got - want) <= bound + 300 * 2.0 ** -35 * largest).all()
