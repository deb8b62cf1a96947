"""The cache in pages, the attention over it, probabilities and the verification of drafts, through the C ABI against tests/paged_plain.py (float64)."""
import ctypes as C

import numpy as np
import pytest

import paged_plain as pp
from conftest import load_pkg
from device_data import Dev
from paged_plain import BF16, E4M3, F16, F32, I8

pytestmark = pytest.mark.gpu
pkg = load_pkg()
KINDS = [F16, BF16, I8, E4M3]


def ids(v):
    return pp.NAMES.get(v) if isinstance(v, int) and v in (24, 30, 259) else None


def error_word(gpu):
    """The pending device error, which is taken."""
    with pytest.raises(pkg.LvError) as e:
        gpu.sync()
    assert e.value.code == pkg.LV_ERR_DEVICE_WAIT
    gpu.sync()


def padded(x, ld, kind, fill=np.nan):
    """rows of x with junk behind them, as stored"""
    out = np.full((x.shape[0], ld), fill, np.float32)
    out[:, :x.shape[1]] = x
    return pp.bits(out, kind)


# ---- writing --------------------------------------------------------------------------------

@pytest.mark.parametrize("kind", KINDS, ids=pp.NAMES.get)
@pytest.mark.parametrize("lens,new,H,dim,page,given,pairs,extra", [([1], [1], 1, 16, 1, F32, 8, 0), ([700], [1], 8, 128, 16, F32, 64, 0), ([5, 40, 17, 9], [5, 1, 0, 7], 3, 80, 20, BF16, 13, 16),
                                                                   ([300, 64], [300, 33], 2, 256, 64, F16, 0, 8), ([33] * 40, [1] * 40, 2, 64, 32, F32, 32, 4)], ids=ids)
def test_new_rows_are_written_where_they_belong_and_nothing_else(gpu, kind, lens, new, H, dim, page, given, pairs, extra):
    rng = np.random.default_rng(dim + page)
    c = pp.Cache(rng, lens, H, dim, kind, page)
    starts, behind = np.cumsum([0] + new), 3
    tokens = starts[-1] + behind                                       # the last rows belong to no sequence
    k, v = (pp.rounded(rng.standard_normal((tokens, H * dim)) * rng.uniform(1e-3, 30, (tokens, 1)), given) for _ in range(2))
    k[0, :dim] = 0.0                                                   # a row of zeros, one below the smallest, one that is not finite
    v[0, :dim] *= 1e-37 if given == F32 else 0.0
    v[starts[-1] - 1, -1] = np.inf
    angles = pp.angles_of(rng, tokens, pairs) if pairs else None
    with Dev(gpu) as d:
        a = c.upload(d, starts)
        table = np.zeros((tokens, 2 * pairs + 2), np.float32)
        if pairs:
            table[:, :2 * pairs] = angles.reshape(tokens, -1)
        d.call("lv_paged_append", C.byref(a), d.up(padded(k, H * dim + extra, given)), d.up(padded(v, H * dim + extra, given)), given, H * dim + extra,
               d.up(table) if pairs else None, 2 * pairs + 2, pairs, tokens)
        data, scales = c.download(gpu)
    turned = pp.rotate(k.reshape(tokens, H, dim), angles)
    with np.errstate(invalid="ignore", over="ignore"):
        for s, n in enumerate(new):
            rows = slice(starts[s], starts[s] + n)
            c.write(s, np.arange(lens[s] - n, lens[s]), 0, turned[rows])
            c.write(s, np.arange(lens[s] - n, lens[s]), 1, v[rows].reshape(n, H, dim))
    for which in range(2):
        assert np.array_equal(data[which], c.data[which])
        if kind in pp.TOP:
            assert np.array_equal(scales[which].view(np.uint32) | 0x00000000, c.scales[which].view(np.uint32)) or \
                np.array_equal(np.nan_to_num(scales[which], nan=-1.0), np.nan_to_num(c.scales[which], nan=-1.0))


@pytest.mark.parametrize("kind", [I8, E4M3], ids=pp.NAMES.get)
def test_values_between_two_codes_go_to_the_even_one(gpu, kind):
    rng = np.random.default_rng(3)
    c = pp.Cache(rng, [1], 1, 64, kind, 4)
    codes = np.arange(-60, 60, 2)[:63] + 0.5 if kind == I8 else (pp.E4M3_VALUES[20:83] + pp.E4M3_VALUES[21:84]) / 2
    x = np.concatenate([[pp.TOP[kind]], codes, np.zeros(63)])[:64].astype(np.float32)[None]          # the scale is 1
    with Dev(gpu) as d:
        a = c.upload(d, [0, 1])
        d.call("lv_paged_append", C.byref(a), d.f32(x), d.f32(-x), F32, 64, None, 0, 0, 1)
        data, scales = c.download(gpu)
    c.write(0, [0], 0, x.reshape(1, 1, 64))
    c.write(0, [0], 1, -x.reshape(1, 1, 64))
    page = c.table[0, 0]
    assert scales[0][page, 0, 0] == 1.0 and np.array_equal(data[0], c.data[0]) and np.array_equal(data[1], c.data[1])


# ---- reading back ------------------------------------------------------------------------------

@pytest.mark.parametrize("kind", KINDS, ids=pp.NAMES.get)
@pytest.mark.parametrize("lens,H,dim,page,out,first,rows", [([1], 1, 16, 1, F32, 0, 1), ([700, 0, 33], 4, 128, 16, BF16, 0, 720), ([50, 21], 3, 80, 20, F16, 13, 20), ([300], 2, 256, 64, F32, 299, 5)], ids=ids)
def test_rows_come_back(gpu, kind, lens, H, dim, page, out, first, rows):
    rng = np.random.default_rng(dim)
    c = pp.Cache(rng, lens, H, dim, kind, page).fill(rng)
    pad = 16
    rs, hs = dim + pad, rows * (dim + pad) + pad                        # [seq][head][row][dim] with gaps
    ss = H * hs
    with Dev(gpu) as d:
        a = c.upload(d, [0] * (len(lens) + 1))
        blank = pp.bits(np.full((len(lens), ss), -7.0, np.float32), out)
        to = [d.up(blank) for _ in range(2)]
        d.call("lv_paged_read", C.byref(a), to[0], to[1], out, ss, hs, rs, first, rows)
        got = [gpu.download(t, blank.dtype, blank.size).reshape(blank.shape) for t in to]
    for which in range(2):
        want = np.full(blank.shape, -7.0, np.float32)
        for s, n in enumerate(lens):
            there = np.arange(first, max(first, min(n, first + rows)))
            if len(there):
                x = c.read(s, there, which, f32=True)
                for h in range(H):
                    for i in range(len(there)):
                        want[s, h * hs + i * rs:h * hs + i * rs + dim] = x[i, h]
        assert np.array_equal(got[which], pp.bits(want, out))


# ---- attention ----------------------------------------------------------------------------------

class Step:
    """A step's attention on the device."""

    def __init__(self, d, c, new, heads, seed=0, given=F32, out=BF16, window=0, sink=False, pairs=0, scale=None, behind=2, max_new=None, max_len=None, gap=8, size=1.0):
        rng = np.random.default_rng(seed + 100)
        self.d, self.c, self.heads, self.out, self.window = d, c, heads, out, window
        self.starts = np.cumsum([0] + list(new))
        self.tokens = int(self.starts[-1]) + behind
        self.scale = scale or c.dim ** -0.5
        self.q = pp.rounded(size * rng.standard_normal((self.tokens, heads * c.dim)), given)
        self.sink = (rng.standard_normal(heads) * 2).astype(np.float32) if sink else None
        self.angles = pp.angles_of(rng, self.tokens, pairs) if pairs else None
        q = self.q.copy()
        q[self.starts[-1]:] = np.nan
        self.ld = heads * c.dim + gap
        self.blank = pp.bits(np.full((self.tokens, self.ld), -7.0, np.float32), out)
        self.dout = d.up(self.blank)
        self.a = pkg.PagedAttentionArgs(cache=c.upload(d, self.starts), q=d.up(padded(q, self.ld, given)).value, q_type=given, q_ld=self.ld, heads=heads, tokens=self.tokens,
                                        max_new=max_new or max(new), max_len=max_len or max(c.lens), scale=self.scale, window=window,
                                        sink=d.f32(self.sink).value if sink else None, angles=d.f32(self.angles).value if pairs else None, angle_ld=2 * pairs, angle_pairs=pairs,
                                        out=self.dout.value, out_type=out, out_ld=self.ld)
        self.bytes = d.gpu.lib.lv_paged_attention_scratch_bytes(d.gpu.handle, C.byref(self.a))
        assert self.bytes > 0
        self.scratch = d.up(np.full(self.bytes, 0xFF, np.uint8))

    def launch(self):
        pkg.check(self.d.gpu.lib.lv_paged_attention(self.d.gpu.handle, C.byref(self.a), self.scratch, self.bytes))
        return self

    def result(self):
        self.d.gpu.sync()
        got = pp.values(self.d.gpu.download(self.dout, self.blank.dtype, self.blank.size), self.out).reshape(self.tokens, self.ld)
        width, last = self.heads * self.c.dim, self.starts[-1]
        assert (got[:, width:] == -7.0).all() and (got[last:] == -7.0).all()             # what is nobody's stays
        return got[:last, :width].reshape(last, self.heads, self.c.dim).astype(np.float64)

    def check(self, got=None):
        got = self.result() if got is None else got
        last = int(self.starts[-1])
        want, bound = pp.attend(self.c, self.starts, self.q[:last].reshape(last, self.heads, self.c.dim), self.heads, self.scale, self.window, self.sink,
                                None if self.angles is None else self.angles[:last], self.out)
        assert np.isfinite(got).all()
        worst = (np.abs(got - want) / bound).max() if last else 0.0
        assert worst <= 1.0, worst
        return got


SHAPES = [  # lens, new, heads, kv heads, dim, page
    ([1], [1], 1, 1, 16, 1), ([1, 2, 3], [1, 1, 1], 4, 4, 64, 16), ([521], [1], 8, 8, 128, 16), ([700, 3, 0, 64, 65], [1, 1, 0, 1, 1], 8, 2, 128, 64), ([1300, 77], [1, 1], 14, 2, 80, 20),
    ([130, 40, 9], [5, 3, 9], 8, 2, 128, 32), ([257, 64], [4, 7], 15, 3, 64, 128), ([90, 1], [17, 1], 4, 4, 256, 16), ([200, 31], [2, 2], 12, 1, 240, 8), ([48, 200, 33], [48, 100, 2], 4, 2, 128, 16),
    ([300], [300], 2, 1, 64, 32), ([150, 400], [129, 131], 5, 1, 80, 20), ([260], [257], 1, 1, 256, 64)]


@pytest.mark.parametrize("kind", KINDS, ids=pp.NAMES.get)
@pytest.mark.parametrize("out", [F32, BF16, F16], ids=["to-f32", "to-bf16", "to-f16"])
@pytest.mark.parametrize("lens,new,heads,H,dim,page", SHAPES, ids=[f"{max(s[0])}x{max(s[1])}-h{s[2]}k{s[3]}d{s[4]}p{s[5]}" for s in SHAPES])
def test_attention_of_new_tokens(gpu, kind, out, lens, new, heads, H, dim, page):
    rng = np.random.default_rng(max(lens) + dim)
    c = pp.Cache(rng, lens, H, dim, kind, page).fill(rng)              # (places behind a sequence hold NaN)
    with Dev(gpu) as d:
        Step(d, c, new, heads, out=out, given=BF16 if out == BF16 else F32).launch().check()


@pytest.mark.parametrize("kind", [BF16, I8], ids=pp.NAMES.get)
@pytest.mark.parametrize("window,lens,new", [(1, [40], [3]), (16, [100, 9], [1, 9]), (64, [300], [200]), (100, [128, 500], [1, 2]), (129, [400], [260]), (1000, [300], [150])])
@pytest.mark.parametrize("sink", [False, True], ids=["", "sinks"])
def test_windows_sinks_and_rotation(gpu, kind, window, lens, new, sink):
    rng = np.random.default_rng(window)
    c = pp.Cache(rng, lens, 2, 128, kind, 16).fill(rng)
    for s, (n, m) in enumerate(zip(lens, new)):                          # what has left all windows is not looked at, whatever it holds
        gone = np.arange(max(0, n - m + 1 - window))
        p, r = c.place(s, gone)
        for which in range(2):
            c.data[which][p, :, r] = 0x7F if kind == I8 else 0x7FC0
            c.scales[which][p, :, r] = np.nan
    c.table[0, :max(0, (lens[0] - new[0] + 1 - window)) // 16] = 0xFFFFFFFF       # and need no page
    with Dev(gpu) as d:
        for out, pairs in ((F32, 64), (BF16, 24)):
            Step(d, c, new, 8, out=out, window=window, sink=sink, pairs=pairs).launch().check()


@pytest.mark.parametrize("kind", KINDS, ids=pp.NAMES.get)
@pytest.mark.parametrize("new", [1, 3, 140])
def test_scores_of_every_size(gpu, kind, new):
    """One key far above all others, equal keys, tiny queries; scores up to several hundred."""
    rng = np.random.default_rng(new)
    lens = [600, 600, 200]
    c = pp.Cache(rng, lens, 1, 64, kind, 32).fill(rng)
    hot = np.zeros((1, 1, 64), np.float32)
    hot[..., :8] = 40.0
    c.write(0, [555 - new], 0, hot)
    c.write(1, np.arange(600), 0, np.repeat(rng.standard_normal((1, 1, 64)).astype(np.float32), 600, 0))
    with Dev(gpu) as d:
        for out in (F32, BF16):
            for size in (1.0, 1e-6, 6.0):
                Step(d, c, [new] * 3, 4, out=out, size=size).launch().check()


def test_long_contexts_are_split(gpu):
    rng = np.random.default_rng(8)
    lens = [9000, 12001, 17]
    with Dev(gpu) as d:
        for kind, new, out in ((BF16, [1, 1, 1], F32), (E4M3, [3, 2, 1], BF16), (F16, [70, 33, 17], F16)):
            c = pp.Cache(rng, lens, 1, 128, kind, 64).fill(rng)
            one = Step(d, c, new, 2, out=out, sink=True)
            first = one.launch().check()
            assert np.array_equal(one.launch().result(), first)                    # the same again, bit for bit, in a used workspace
            assert np.array_equal(Step(d, c, new, 2, out=out, sink=True, max_len=12001 + 20).launch().check().shape, first.shape)


def test_a_step_in_which_nobody_has_new_tokens(gpu):
    rng = np.random.default_rng(6)
    c = pp.Cache(rng, [40, 0], 2, 64, F16, 16).fill(rng)
    with Dev(gpu) as d:
        Step(d, c, [0, 0], 4, out=BF16).launch().check()                 # (two rows of nobody's: as they were)
        empty = pp.Cache(rng, [0, 0], 2, 64, I8, 16)
        st = Step(d, empty, [0, 0], 4, out=F32)
        st.a.tokens = st.a.max_new = st.a.max_len = 0
        assert gpu.lib.lv_paged_attention_scratch_bytes(gpu.handle, C.byref(st.a)) > 0
        st.launch().check()


@pytest.mark.parametrize("kind", KINDS, ids=pp.NAMES.get)
@pytest.mark.parametrize("page,dim,heads,H,lens,new", [(8, 16, 3, 1, [90], [31]), (24, 48, 2, 2, [200, 1, 60], [40, 1, 35]), (40, 112, 4, 1, [700], [33]), (128, 128, 1, 1, [129, 128], [129, 128]),
                                                       (256, 64, 5, 1, [600, 34], [60, 7]), (8, 128, 8, 2, [1, 300, 0, 257], [1, 64, 0, 65])])
def test_many_rows_of_every_page(gpu, kind, page, dim, heads, H, lens, new):
    """Boxes of 8 to 128 rows, head sizes that do not fill a block of columns, tiles of one row; windows that begin inside a box."""
    rng = np.random.default_rng(page + dim)
    c = pp.Cache(rng, lens, H, dim, kind, page).fill(rng)
    with Dev(gpu) as d:
        for window, out in ((0, BF16), (37, F16)):
            Step(d, c, new, heads, out=out, window=window, sink=bool(window), pairs=dim // 2 if window else 0).launch().check()


@pytest.mark.parametrize("new", [3, 100])
@pytest.mark.parametrize("kind", KINDS, ids=pp.NAMES.get)
def test_pages_that_are_not_there_to_16_bits(gpu, kind, new):
    """As above through the kernels of 16-bit outputs: a masked key is one with a score of -infinity."""
    rng = np.random.default_rng(new + 1)
    c = pp.Cache(rng, [320], 1, 64, kind, 16).fill(rng)
    with Dev(gpu) as d:
        st = Step(d, c, [new], 2, out=F16)
        table = c.table.copy()
        table[0, [0, 3, 4, 9]] = [c.pages, c.pages, 0xFFFFFFFF, c.pages + 5]
        st.a.cache.table = d.u32(table).value
        st.launch()
        error_word(gpu)
        got = st.result()
        gone = np.concatenate([np.arange(16), np.arange(48, 80), np.arange(144, 160)])
        k, v = c.read(0, np.arange(320), 0)[:, 0], c.read(0, np.arange(320), 1)[:, 0]
        z = st.scale * np.einsum("thd,jd->thj", st.q[:new].reshape(new, 2, 64).astype(np.float64), k)
        z[..., gone] = -np.inf
        z = np.where(np.arange(320) <= (320 - new + np.arange(new))[:, None, None], z, -np.inf)
        p = np.exp(z - z.max(-1, keepdims=True))
        # operands in 16 bits: scores off by 2^-8 (bf16) or 2^-11 times the largest sum |q| |k|, a weight by twice that and its rounding, results by f16's
        u = pp.HALF_STEP[BF16 if kind == BF16 else F16]
        most = st.scale * np.einsum("thd,jd->thj", np.abs(st.q[:new]).reshape(new, 2, 64).astype(np.float64), np.abs(k)).max()
        off = (np.expm1(2 * u * most) + 2 * u + 2.0 ** -15) * (p @ np.abs(v) / p.sum(-1, keepdims=True))
        want = p @ v / p.sum(-1, keepdims=True)
        assert (np.abs(got - want) <= off + 2.0 ** -11 * (np.abs(want) + off) + 2.0 ** -25 + 320 * 2.0 ** -35 * np.abs(v).max()).all()
        st.a.cache.table = d.u32(np.full_like(table, c.pages)).value
        st.launch()
        error_word(gpu)
        assert (st.result() == 0.0).all()


@pytest.mark.parametrize("new", [1, 60])
@pytest.mark.parametrize("kind", [BF16, I8], ids=pp.NAMES.get)
def test_a_query_that_is_no_number_keeps_to_its_row(gpu, kind, new):
    rng = np.random.default_rng(3)
    c = pp.Cache(rng, [300, 200], 1, 64, kind, 16).fill(rng)
    with Dev(gpu) as d:
        for out in (F32, BF16):
            st = Step(d, c, [new, new], 2, out=out)
            good = st.launch().check()
            q = padded(st.q, st.ld, F32, 0.0)
            q[new // 2, :64] = np.nan
            st.a.q = d.up(q).value
            got = st.launch().result()
            bad = np.zeros(got.shape, bool)
            bad[new // 2, 0] = True
            assert np.isnan(got[bad]).all() and np.array_equal(got[~bad], good[~bad])


def test_two_contexts_at_once(gpu):
    """Two streams, each with its own scratch, many rows and few, split and whole."""
    rng = np.random.default_rng(12)
    c = pp.Cache(rng, [3000, 700], 2, 128, BF16, 64).fill(rng)
    other = pkg.Context(0)
    try:
        with Dev(gpu) as d, Dev(other) as e:
            steps = [Step(x, c, new, 8, out=BF16, seed=i) for x in (d, e) for i, new in enumerate(([60, 33], [1, 2]))]
            gpu.sync()
            other.sync()
            for _ in range(8):
                for st in steps:
                    st.launch()
            for st in steps:
                st.check()
    finally:
        other.close()


def test_many_rows_in_a_recorded_step(gpu):
    rng = np.random.default_rng(13)
    c = pp.Cache(rng, [900, 260], 1, 128, E4M3, 32).fill(rng)
    with Dev(gpu) as d:
        st = Step(d, c, [70, 40], 4, out=BF16, window=500, sink=True)
        first = st.launch().check()
        pkg.check(gpu.lib.lv_graph_begin_capture(gpu.handle))
        st.launch()
        g = C.c_void_p()
        pkg.check(gpu.lib.lv_graph_end_capture(gpu.handle, C.byref(g)))
        for _ in range(3):
            pkg.check(gpu.lib.lv_graph_launch(gpu.handle, g))
            assert np.array_equal(st.result(), first)
        gpu.lib.lv_graph_destroy(g)


def test_two_sequences_share_a_page(gpu):
    rng = np.random.default_rng(5)
    c = pp.Cache(rng, [40, 45], 2, 64, F16, 16).fill(rng)
    c.table[1, :2] = c.table[0, :2]                                      # a common beginning
    with Dev(gpu) as d:
        Step(d, c, [1, 6], 4, out=F32).launch().check()


def test_a_recorded_step_serves_every_token(gpu):
    """append and attention in one graph, twice with shared scratch; lengths and starts move on the device."""
    rng = np.random.default_rng(11)
    H, dim, heads, page = 2, 128, 8, 16
    lens = [30, 500]
    c = pp.Cache(rng, [60, 560], H, dim, I8, page).fill(rng)
    c.lens = lens
    new = [1, 1]
    with Dev(gpu) as d:
        st = Step(d, c, new, heads, out=F32, behind=0, max_len=560)
        dk, dv = d.zeros(2 * H * dim * 4), d.zeros(2 * H * dim * 4)
        graphs = []
        for _ in range(2):
            pkg.check(gpu.lib.lv_graph_begin_capture(gpu.handle))
            pkg.check(gpu.lib.lv_paged_append(gpu.handle, C.byref(st.a.cache), dk, dv, F32, H * dim, None, 0, 0, 2))
            st.launch()
            g = C.c_void_p()
            pkg.check(gpu.lib.lv_graph_end_capture(gpu.handle, C.byref(g)))
            graphs.append(g)
        for step in range(4):
            k, v = rng.standard_normal((2, 2, H, dim)).astype(np.float32)
            c.lens = [n + 1 for n in c.lens]
            for b, x in ((dk, k), (dv, v), (c.dlens, np.array(c.lens, np.uint32))):
                pkg.check(gpu.lib.lv_upload(gpu.handle, b, np.ascontiguousarray(x).ctypes.data_as(C.c_void_p), x.nbytes))
            for s in range(2):
                c.write(s, [c.lens[s] - 1], 0, k[s:s + 1])
                c.write(s, [c.lens[s] - 1], 1, v[s:s + 1])
            pkg.check(gpu.lib.lv_graph_launch(gpu.handle, graphs[step % 2]))
            st.check()
        for g in graphs:
            gpu.lib.lv_graph_destroy(g)


@pytest.mark.parametrize("new", [[1, 1, 1], [40, 3, 150]], ids=["tokens", "prompts"])
def test_what_contradicts_itself_is_reported_and_left_out(gpu, new):
    rng = np.random.default_rng(2)
    lens = [200, 64, 300]
    c = pp.Cache(rng, lens, 1, 64, BF16, 32).fill(rng)

    def others(st, got, bad):
        want, bound = pp.attend(c, st.starts, st.q[:st.starts[-1]].reshape(-1, 2, 64), 2, st.scale, out_kind=BF16)
        for s in range(3):
            if s != bad:
                rows = slice(st.starts[s], st.starts[s + 1])
                assert (np.abs(got[rows] - want[rows]) <= bound[rows]).all()
            else:
                assert (got[st.starts[s]:st.starts[s + 1]] == -7.0).all()
    with Dev(gpu) as d:
        for change in ("too long", "before the beginning", "more than stated", "longer than stated"):
            st = Step(d, c, new, 2)
            bad = 2 if change == "longer than stated" else 0
            if change == "too long":
                st.a.cache.lens = d.u32([c.width * 32 + 1] + lens[1:]).value
            elif change == "before the beginning":
                st.a.cache.lens = d.u32([new[0] - 1] + lens[1:]).value
            elif change == "more than stated":
                if max(new) == 1:
                    continue
                st.a.max_new, bad = max(new) - 1, 2
            else:
                st.a.max_len = max(lens) - 1
            st.launch()
            error_word(gpu)
            others(st, st.result(), bad)


@pytest.mark.parametrize("new", [1, 3, 100])
@pytest.mark.parametrize("kind", [F16, I8], ids=pp.NAMES.get)
def test_pages_that_are_not_there_count_as_masked(gpu, kind, new):
    rng = np.random.default_rng(new)
    c = pp.Cache(rng, [320], 1, 64, kind, 16).fill(rng)
    with Dev(gpu) as d:
        st = Step(d, c, [new], 2, out=F32)
        table = c.table.copy()
        table[0, [3, 4, 9]] = [c.pages, 0xFFFFFFFF, c.pages + 5]
        st.a.cache.table = d.u32(table).value
        st.launch()
        error_word(gpu)
        got = st.result()
        # the same with these keys far below all others
        gone = np.concatenate([np.arange(48, 80), np.arange(144, 160)])
        k, v = c.read(0, np.arange(320), 0)[:, 0], c.read(0, np.arange(320), 1)[:, 0]
        q = st.q[:new].reshape(new, 2, 64).astype(np.float64)
        z = st.scale * np.einsum("thd,jd->thj", q, k)
        z[..., gone] = -np.inf
        z = np.where(np.arange(320) <= (320 - new + np.arange(new))[:, None, None], z, -np.inf)
        p = np.exp(z - z.max(-1, keepdims=True))
        want = p @ v / p.sum(-1, keepdims=True)
        assert np.abs(got - want).max() <= 1e-5 * np.abs(v).max()
        # nothing left: zeros
        st.a.cache.table = d.u32(np.full_like(table, c.pages)).value
        st.launch()
        error_word(gpu)
        assert (st.result() == 0.0).all()


def test_places_beyond_32_bits(gpu):
    """A cache of more than 2^32 values: its last page."""
    H, dim, page = 8, 256, 64
    pages = (1 << 32) // (H * dim * page) + 2
    rng = np.random.default_rng(4)
    with Dev(gpu) as d:
        k, v = d.zeros(pages * H * page * dim), d.zeros(pages * H * page * dim)
        ks, vs = d.zeros(pages * H * page * 4), d.zeros(pages * H * page * 4)
        c = pkg.PagedCache(k=k.value, v=v.value, k_scale=ks.value, v_scale=vs.value, type=I8, pages=pages, page_rows=page, kv_heads=H, dim=dim, table=d.u32([pages - 1]).value, table_ld=1,
                           lens=d.u32([page]).value, starts=d.u32([0, page]).value, seqs=1)
        x = rng.standard_normal((page, H * dim)).astype(np.float32)
        d.call("lv_paged_append", C.byref(c), d.f32(x), d.f32(-x), F32, H * dim, None, 0, 0, page)
        out = [d.zeros(page * H * dim * 4) for _ in range(2)]
        d.call("lv_paged_read", C.byref(c), out[0], out[1], F32, 0, dim, H * dim, 0, page)
        codes, scale = pp.quantise(x.reshape(page, H, dim), I8)
        want = codes.view(np.int8).astype(np.float32) * scale[..., None]
        assert np.array_equal(d.get(out[0], (page, H, dim)), want) and np.array_equal(d.get(out[1], (page, H, dim)), -want)
        got = d.zeros(page * H * dim * 4)
        q = rng.standard_normal((page, H * dim)).astype(np.float32)
        for first in (page - 1, 0):                                     # the last token alone, and all of them
            n = page - first
            a = pkg.PagedAttentionArgs(cache=c, q=d.f32(q[first:]).value, q_type=F32, q_ld=H * dim, heads=H, tokens=n, max_new=n, max_len=page, scale=dim ** -0.5, out=got.value, out_type=F32,
                                       out_ld=H * dim)
            a.cache.starts = d.u32([0, n]).value
            nbytes = gpu.lib.lv_paged_attention_scratch_bytes(gpu.handle, C.byref(a))
            d.call("lv_paged_attention", C.byref(a), d.zeros(nbytes), nbytes)
            z = np.einsum("thd,jhd->htj", q[first:].reshape(n, H, dim).astype(np.float64), want.astype(np.float64)) * dim ** -0.5
            z = np.where(np.arange(page) <= np.arange(first, page)[:, None], z, -np.inf)
            p = np.exp(z - z.max(-1, keepdims=True))
            ref = np.einsum("htj,jhd->thd", p / p.sum(-1, keepdims=True), -want.astype(np.float64))
            assert np.abs(d.get(got, (n, H, dim)) - ref).max() <= 1e-5 * np.abs(ref).max()


# ---- probabilities ----------------------------------------------------------------------------------

@pytest.mark.parametrize("rows,vocab,gap", [(1, 1, 0), (1, 32000, 0), (5, 32000, 0), (3, 1001, 3), (9, 50021, 7), (2, 262147, 1), (1, 1500000, 0), (300, 515, 1), (70000, 3, 0)])
@pytest.mark.parametrize("place", [False, True], ids=["", "in-place"])
def test_probabilities(gpu, rows, vocab, gap, place):
    rng = np.random.default_rng(vocab)
    x = (rng.standard_normal((rows, vocab + gap)) * 4).astype(np.float32)
    T = rng.uniform(0.3, 1.5, rows).astype(np.float32)
    T[::3] = 0.0
    x[0, vocab // 2], x[0, vocab - 1] = 50.0, 50.0                     # two maxima
    if rows > 1:
        x[1, :vocab:2] = -np.inf
    with Dev(gpu) as d:
        dx = d.f32(x)
        out = dx if place else d.up(np.full(x.shape, -7.0, np.float32))
        d.call("lv_probabilities", out, vocab + gap, dx, vocab + gap, vocab, rows, d.f32(T))
        got = d.get(out, x.shape)
    assert np.array_equal(got[:, vocab:], x[:, vocab:] if place else np.full((rows, gap), -7.0, np.float32))
    for r in range(min(rows, 400)):
        row = x[r, :vocab].astype(np.float64)
        if T[r] == 0:
            want = np.zeros(vocab)
            want[row.argmax()] = 1.0
            assert np.array_equal(got[r, :vocab], want)
            continue
        z = (row - row.max()) / np.float64(T[r])
        e = np.exp(z)
        # the argument of each exponential is off by 2^-22 of itself, the exponential by 2^-22, the sum by at most its longest chain of 64 + 32 + 10 additions
        tol = np.where(np.isfinite(z), np.abs(z), 0) * 2.0 ** -22 + 2.0 ** -22 + (np.where(e > 0, np.abs(np.maximum(z, -200)), 0) * e).sum() / e.sum() * 2.0 ** -22 + (128 + vocab / 1024) * 2.0 ** -24
        assert (np.abs(got[r, :vocab] - e / e.sum()) <= tol * e / e.sum() + 1e-37).all()


def test_probabilities_of_rows_without_a_choice(gpu):
    x = np.zeros((4, 700), np.float32)
    x[0] = -np.inf
    x[1] = -np.inf
    x[2, 5] = np.nan
    x[3, :] = np.nan
    x[3, 650] = -5.0
    with Dev(gpu) as d:
        out = d.zeros(x.nbytes)
        d.call("lv_probabilities", out, 700, d.f32(x), 700, 700, 4, d.f32([1.0, 0.0, 0.5, 0.0]))
        got = d.get(out, x.shape)
    assert (got[0] == 0).all() and got[1, 0] == 1.0 and got[1].sum() == 1.0 and np.isnan(got[2]).all() and got[3, 650] == 1.0 and got[3].sum() == 1.0
    with Dev(gpu) as d:                                                  # no temperatures: 1
        out = d.zeros(40)
        d.call("lv_probabilities", out, 10, d.f32(np.arange(10)), 10, 10, 1, None)
        e = np.exp(np.arange(10.0) - 9)
        assert np.abs(d.get(out, (10,)) - e / e.sum()).max() < 1e-6


@pytest.mark.parametrize("vocab", [50, 40001, 300000])
def test_probabilities_at_the_smallest_temperatures(gpu, vocab):
    x = np.random.default_rng(vocab).standard_normal((3, vocab)).astype(np.float32)
    x[:, 7], x[1, vocab - 2], x[2, ::3] = 50.0, 50.0, -np.inf
    want = np.zeros((3, vocab), np.float32)
    want[:, 7] = 1.0
    want[1, [7, vocab - 2]] = 0.5
    with Dev(gpu) as d:
        for T in (1e-45, 1e-42, 1e-38, 1e-30):
            out = d.zeros(3 * vocab * 4)
            d.call("lv_probabilities", out, vocab, d.f32(x), vocab, vocab, 3, d.f32(np.full(3, T, np.float32)))
            assert np.array_equal(d.get(out, (3, vocab)), want)


# ---- verification -------------------------------------------------------------------------------------

def run_verify(gpu, target, draft, drafted, starts, accept, pick, lens=None, gap=0):
    rows, vocab = target.shape
    with Dev(gpu) as d:
        tok, acc = d.u32(np.full(rows + 1, 77)), d.u32(np.full(len(starts), 77))
        wide = (lambda x: d.f32(np.pad(x, ((0, 0), (0, gap)), constant_values=9.0)).value)
        dl = d.u32(lens) if lens is not None else None
        a = pkg.VerifyArgs(target=wide(target), target_ld=vocab + gap, draft=None if draft is None else wide(draft), draft_ld=vocab + gap, vocab=vocab, drafted=d.u32(drafted).value,
                           starts=d.u32(starts).value, seqs=len(starts) - 1, rows=rows, accept=d.f32(accept).value, pick=d.f32(pick).value, tokens=tok.value, accepted=acc.value,
                           lens=dl.value if dl else None)
        pkg.check(gpu.lib.lv_verify_drafts(gpu.handle, C.byref(a)))
        failed = None
        try:
            gpu.sync()
        except pkg.LvError as e:
            failed = e.code
        t, n = gpu.download(tok, np.uint32, rows + 1), gpu.download(acc, np.uint32, len(starts))
        assert t[rows] == 77 and n[-1] == 77
        return n[:-1], t[:rows], None if dl is None else gpu.download(dl, np.uint32, len(lens)), failed


def distributions(rng, rows, vocab, sharp=3.0):
    x = rng.standard_normal((rows, vocab)) * sharp
    p, q = np.exp(x), np.exp(x + 0.7 * rng.standard_normal((rows, vocab)))
    return (p / p.sum(1, keepdims=True)).astype(np.float32), (q / q.sum(1, keepdims=True)).astype(np.float32)


@pytest.mark.parametrize("vocab,counts,gap", [(1, [0, 1], 0), (5, [3, 0, 4, 2] * 10, 0), (1000, [4, 4, 0, 9], 5), (32000, [4], 0), (32000, [40, 1], 0), (50021, [7, 2, 3], 2), (300001, [2, 0], 1)])
@pytest.mark.parametrize("certain", [False, True], ids=["", "certain"])
def test_drafts_are_accepted_and_tokens_drawn_by_the_definition(gpu, vocab, counts, gap, certain):
    rng = np.random.default_rng(vocab + len(counts))
    starts = np.cumsum([0] + [n + 1 for n in counts])
    starts[1:] += 0
    rows = int(starts[-1]) + 2                                           # two rows that are nobody's
    target, draft = distributions(rng, rows, vocab)
    drafted = np.array([rng.choice(vocab, p=q.astype(np.float64) / q.astype(np.float64).sum()) for q in draft], np.uint32)
    lens = rng.integers(100, 200, len(counts))
    for trial in range(4):
        accept, pick = rng.random(rows).astype(np.float32), rng.random(len(counts)).astype(np.float32)
        accept, pick = np.minimum(accept, np.float32(1 - 2 ** -24)), np.minimum(pick, np.float32(1 - 2 ** -24))
        if trial == 1:
            accept[:] = 0                                                # all accepted
        if trial == 2:
            pick[:] = np.float32(1 - 2 ** -24)
        if trial == 3:
            pick[:], accept[:] = 0, np.float32(1 - 2 ** -24)
        n, t, left, failed = run_verify(gpu, target, None if certain else draft, drafted, starts, accept, pick, lens, gap)
        wn, wt = pp.verify(target, None if certain else draft, drafted, starts, accept, pick)
        assert failed is None and np.array_equal(n, wn)
        assert np.array_equal(t[:starts[-1]], wt[:starts[-1]]) and (t[starts[-1]:] == 77).all()
        assert np.array_equal(left, lens - (np.array(counts) - wn))


def test_sequences_without_rows_and_drafts_that_are_no_tokens(gpu):
    rng = np.random.default_rng(0)
    target, draft = distributions(rng, 6, 100)
    starts = [0, 0, 3, 3, 6]
    drafted = np.array([1, 100, 0, 2, 0xFFFFFFFF, 0], np.uint32)
    accept, pick = np.zeros(6, np.float32), np.full(4, 0.5, np.float32)
    n, t, _, failed = run_verify(gpu, target, draft, drafted, starts, accept, pick)
    assert failed == pkg.LV_ERR_DEVICE_WAIT and list(n) == [0, 1, 0, 1]
    assert t[0] == 1 and t[3] == 2 and t[2] == t[5] == 0xFFFFFFFF
    for row, got in ((1, t[1]), (4, t[4])):                              # drawn as behind a rejected draft
        w = np.cumsum(np.maximum(target[row].astype(np.float64) - draft[row], 0))
        assert got == np.argmax(w > 0.5 * w[-1])
    # starts that run backwards or beyond the rows: the sequence is left out
    for bad in ([0, 3, 2, 6], [0, 3, 9]):
        n, t, _, failed = run_verify(gpu, target, draft, np.ones(6, np.uint32), bad, accept, pick[:len(bad) - 1])
        assert failed == pkg.LV_ERR_DEVICE_WAIT and n[1] == 77 and n[0] == 2


def test_rows_without_weight(gpu):
    target, draft = np.zeros((3, 64), np.float32), np.zeros((3, 64), np.float32)
    target[1, 7], draft[1, 9] = 0.25, 1.0
    target[2, 5], draft[2, 5] = 0.5, 0.5
    starts, drafted = [0, 1, 3], np.array([0, 9, 0], np.uint32)
    half = np.full(3, 0.5, np.float32)
    n, t, _, failed = run_verify(gpu, target, draft, drafted, starts, half, half[:2])
    assert failed == pkg.LV_ERR_DEVICE_WAIT and list(n) == [0, 0] and list(t) == [0xFFFFFFFF, 7, 0xFFFFFFFF]
    # a rejected draft that leaves nothing: from the target itself
    n, t, _, failed = run_verify(gpu, target[[2, 2]], np.concatenate([target[2:] * 2, target[2:]]), np.array([5, 0], np.uint32), [0, 2], half[:2] + 0.0, half[:1])
    assert failed is None and list(n) == [0] and t[0] == 5


def test_picks_and_weights_that_name_no_token(gpu):
    target = np.full((5, 64), 1 / 64, np.float32)
    target[4, 3] = np.inf
    pick = np.array([1.0, np.nan, -0.25, 0.5, 0.5], np.float32)
    n, t, _, failed = run_verify(gpu, target, None, np.zeros(5, np.uint32), [0, 1, 2, 3, 4, 5], np.zeros(5, np.float32), pick)
    assert failed == pkg.LV_ERR_DEVICE_WAIT and list(n) == [0] * 5 and list(t) == [0xFFFFFFFF] * 3 + [32, 0xFFFFFFFF]


# ---- a step of all of them together -------------------------------------------------------------------

def test_a_step_with_drafts(gpu):
    """Drafted tokens of two sequences through append, attention, a head, probabilities and verification; the next step overwrites what was rejected."""
    rng = np.random.default_rng(21)
    H, heads, dim, vocab, page = 2, 4, 64, 200, 16
    kept, new = [37, 90], [4, 3]
    full = pp.Cache(rng, [60, 120], H, dim, E4M3, page).fill(rng)
    width, starts = heads * dim, np.cumsum([0] + new)
    rows = int(starts[-1])
    head = (rng.standard_normal((vocab, width)) * 0.5).astype(np.float32)
    head = pp.rounded(head, BF16)
    with Dev(gpu) as d:
        dhead = d.bf16(head)
        lens = list(kept)
        full.lens = [n + m for n, m in zip(lens, new)]
        st = Step(d, full, new, heads, out=F32, behind=0, gap=0, max_len=120)
        logits, probs, temperature = d.zeros(rows * vocab * 4), d.zeros(rows * vocab * 4), np.full(rows, 0.9, np.float32)
        dt = d.f32(temperature)
        for step in range(3):
            full.lens = [n + m for n, m in zip(lens, new)]
            k, v = (rng.standard_normal((rows, H * dim)).astype(np.float32) for _ in range(2))
            drafted = rng.integers(0, vocab, rows).astype(np.uint32)
            accept, pick = rng.random(rows).astype(np.float32) * np.float32(0.02), rng.random(2).astype(np.float32)
            pkg.check(gpu.lib.lv_upload(gpu.handle, full.dlens, np.array(full.lens, np.uint32).ctypes.data_as(C.c_void_p), 8))
            lib, h = gpu.lib, gpu.handle
            tok, acc = d.zeros(rows * 4), d.zeros(8)
            va = pkg.VerifyArgs(target=probs.value, target_ld=vocab, vocab=vocab, drafted=d.u32(drafted).value, starts=st.a.cache.starts, seqs=2, rows=rows, accept=d.f32(accept).value,
                                pick=d.f32(pick).value, tokens=tok.value, accepted=acc.value, lens=full.dlens.value)
            pkg.check(lib.lv_paged_append(h, C.byref(st.a.cache), d.f32(k), d.f32(v), F32, H * dim, None, 0, 0, rows))
            st.launch()
            pkg.check(lib.lv_gemv_bf16(h, logits, vocab, dhead, vocab, width, width, st.dout, width, rows, 1.0, 0))
            pkg.check(lib.lv_probabilities(h, probs, vocab, logits, vocab, vocab, rows, dt))
            pkg.check(lib.lv_verify_drafts(h, C.byref(va)))
            gpu.sync()
            for s in range(2):
                at = np.arange(lens[s], lens[s] + new[s])
                full.write(s, at, 0, k[starts[s]:starts[s + 1]].reshape(-1, H, dim))
                full.write(s, at, 1, v[starts[s]:starts[s + 1]].reshape(-1, H, dim))
            got = st.check()
            z = (got.reshape(rows, width) @ head.T.astype(np.float64)) / 0.9
            e = np.exp(z - z.max(1, keepdims=True))
            p = d.get(probs, (rows, vocab))
            assert np.abs(p - e / e.sum(1, keepdims=True)).max() < 1e-5
            wn, wt = pp.verify(p, None, drafted, starts, accept, pick)
            n = gpu.download(acc, np.uint32, 2)
            assert np.array_equal(n, wn) and np.array_equal(gpu.download(tok, np.uint32, rows), wt)
            lens = [full.lens[s] - (new[s] - 1 - int(n[s])) for s in range(2)]
            assert np.array_equal(gpu.download(full.dlens, np.uint32, 2), lens)
            full.lens = lens
