"""A cache in pages and the operators over it in plain numpy and float64, for the tests."""
import numpy as np

import sonuzen_plain as sp
from conftest import load_pkg

pkg = load_pkg()
F32, F16, BF16, I8, E4M3 = pkg.TYPE_F32, pkg.TYPE_F16, pkg.TYPE_BF16, pkg.TYPE_I8, pkg.TYPE_E4M3
TOP = {I8: 127.0, E4M3: 448.0}
HALF_STEP = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8, E4M3: 2.0 ** -4}       # of a rounding, relative to the value
NAMES = {F32: "f32", F16: "f16", BF16: "bf16", I8: "i8", E4M3: "e4m3"}


def e4m3_values():
    """value of each of the 256 codes"""
    u = np.arange(256)
    e, f = (u >> 3) & 15, u & 7
    v = np.where(e > 0, (1 + f / 8) * 2.0 ** (e - 7.0), f / 8 * 2.0 ** -6)
    v[(u & 127) == 127] = np.nan
    return np.where(u >> 7, -v, v)


E4M3_VALUES = e4m3_values()


def to_e4m3(x):
    """codes of float32 values of at most 464 in magnitude, to the nearest, ties to the even code"""
    table = E4M3_VALUES[:127]
    a = np.abs(x.astype(np.float64))
    hi = np.clip(np.searchsorted(table, a), 0, 126)
    lo = np.maximum(hi - 1, 0)
    dl, dh = a - table[lo], table[hi] - a
    code = np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    return (code | np.where(np.signbit(x), 128, 0)).astype(np.uint8)


def bits(x, kind):
    """device representation of float32 values of a 16- or 32-bit type"""
    x = np.asarray(x, np.float32)
    return x if kind == F32 else x.astype(np.float16).view(np.uint16) if kind == F16 else sp.bf16_bits(x)


def values(u, kind):
    """the numbers (float32) that stored values stand for; 8-bit codes without their scale"""
    if kind == F32:
        return np.asarray(u, np.float32)
    if kind == F16:
        return np.asarray(u).view(np.float16).astype(np.float32)
    if kind == BF16:
        return (np.asarray(u).astype(np.uint32) << 16).view(np.float32)
    return np.asarray(u).view(np.int8).astype(np.float32) if kind == I8 else E4M3_VALUES[u].astype(np.float32)


def rounded(x, kind):
    return values(bits(x, kind), kind)


def quantise(x, kind):
    """(codes uint8, scales) of float32 rows, in float32 arithmetic"""
    a = np.abs(x).max(axis=-1, keepdims=True)
    fine = a < np.inf
    live = fine & (a >= np.float32(2.0 ** -100))
    top = np.float32(TOP[kind])
    safe = np.where(live, a, np.float32(1))
    scale = np.where(live, safe / top, np.where(fine, np.float32(0), np.float32(np.nan))).astype(np.float32)
    y = np.where(live, x * (top / safe).astype(np.float32), np.float32(0)).astype(np.float32)
    return (np.rint(y).astype(np.int8).view(np.uint8) if kind == I8 else to_e4m3(y)), scale[..., 0]


def rotate(x, angles):
    """x float32 [tokens][heads][dim], angles [tokens][pairs][2]: every product and sum rounded to float32"""
    if angles is None:
        return x
    y = x.copy()
    n = angles.shape[1]
    c, s = angles[:, None, :, 0], angles[:, None, :, 1]
    a, b = x[..., 0:2 * n:2], x[..., 1:2 * n:2]
    y[..., 0:2 * n:2] = a * c - b * s
    y[..., 1:2 * n:2] = b * c + a * s
    return y


class Cache:
    """Pages in a random order on the host; every place that no position uses holds `junk` bytes."""

    def __init__(self, rng, lens, H, dim, kind, page, junk=0xFF, spare=2, share=None):
        self.H, self.dim, self.kind, self.page, self.lens = H, dim, kind, page, list(lens)
        counts = [-(-n // page) for n in lens]
        self.pages, self.width = sum(counts) + spare, max(max(counts), 1)
        order = rng.permutation(self.pages)
        self.table, at = np.full((len(lens), self.width), 0xFFFFFFFF, np.uint32), 0
        for s, n in enumerate(counts):
            self.table[s, :n] = order[at:at + n]
            at += n
        dtype = np.uint8 if kind in TOP else np.uint16
        shape = (self.pages, H, page)
        self.data = [np.full(shape + (dim * dtype().itemsize,), junk, np.uint8).view(dtype) for _ in range(2)]
        self.scales = [np.full(shape, np.nan, np.float32) for _ in range(2)]

    def place(self, s, positions):
        positions = np.asarray(positions)
        return self.table[s, positions // self.page], positions % self.page

    def write(self, s, positions, which, x):
        """float32 [n][H][dim] at positions of sequence s"""
        p, r = self.place(s, positions)
        if self.kind in TOP:
            codes, scale = quantise(x, self.kind)
            self.data[which][p, :, r] = codes
            self.scales[which][p, :, r] = scale
        else:
            self.data[which][p, :, r] = bits(x, self.kind)

    def read(self, s, positions, which, f32=False):
        """[n][H][dim], float64; f32: the product with the scale rounded to float32"""
        p, r = self.place(s, positions)
        x = values(self.data[which][p, :, r], self.kind)
        if self.kind in TOP:
            scale = self.scales[which][p, :, r][..., None]
            return x * scale if f32 else x.astype(np.float64) * scale.astype(np.float64)
        return x if f32 else x.astype(np.float64)

    def fill(self, rng):
        for s, n in enumerate(self.lens):
            if n:
                for which in range(2):
                    self.write(s, np.arange(n), which, (rng.standard_normal((n, self.H, self.dim)) * rng.uniform(0.4, 2.0, (n, self.H, 1))).astype(np.float32))
        return self

    def upload(self, d, starts, lens=None):
        """argument block; d: device_data.Dev"""
        self.k, self.v, self.ks, self.vs = d.up(self.data[0]), d.up(self.data[1]), d.up(self.scales[0]), d.up(self.scales[1])
        self.dlens = d.u32(self.lens if lens is None else lens)
        eight = self.kind in TOP
        return pkg.PagedCache(k=self.k.value, v=self.v.value, k_scale=self.ks.value if eight else None, v_scale=self.vs.value if eight else None, type=self.kind,
                              pages=self.pages, page_rows=self.page, kv_heads=self.H, dim=self.dim, table=d.up(self.table).value, table_ld=self.width,
                              lens=self.dlens.value, starts=d.u32(starts).value, seqs=len(self.lens))

    def download(self, gpu):
        return [gpu.download(b, a.dtype, a.size).reshape(a.shape) for b, a in zip((self.k, self.v), self.data)], \
               [gpu.download(b, np.float32, a.size).reshape(a.shape) for b, a in zip((self.ks, self.vs), self.scales)]


def attend(cache, starts, q, heads, scale, window=0, sink=None, angles=None, out_kind=F32):
    """(out, bound) float64 [tokens][heads][dim] of the float32 queries q [tokens][heads][dim].

    bound: how far a result may be off.  With u the relative error of an operand of the products (queries, probabilities), a score is off by at most
    d = (u + (dim + 3) 2^-24 + 4 2^-24) scale sum |q| |k| (the rounding of q, f32 sums in any order, the factors), a weight by 2 d + 2 u relative to
    itself, its own and the normaliser's (plus 2^-22 |s| + 2^-20 for the exponentials), the sums over n keys by (log2-like chains of at most n) 2^-24 each; all
    together times sum p |v|, and the rounding of the output.  Weights in f16 (all caches but bf16) are whole multiples of 2^-24, while the largest of a row
    is at least 2^10: each is off by up to 2^-25, which is 2^-35 of the largest one and so of the normaliser; with |v| <= max |v| that is n 2^-35 max |v|
    at most over n keys (a value that the visible keys of large weight do not have at all is left to weights that small)."""
    u16 = HALF_STEP[BF16 if cache.kind == BF16 else F16]
    u = 2.0 * u16 * u16 if out_kind == F32 else u16
    tokens, dim, G = q.shape[0], cache.dim, heads // cache.H
    x = rotate(q, angles).astype(np.float64)
    out, bound = np.zeros((tokens, heads, dim)), np.zeros((tokens, heads, dim))
    for s, n in enumerate(cache.lens):
        m = int(starts[s + 1]) - int(starts[s])
        if not m:
            continue
        base = max(0, n - m + 1 - window) if window else 0                # (what lies before may have no page)
        k, v = (cache.read(s, np.arange(base, n), w) for w in range(2))
        for i in range(m):
            at, t = n - m + i, int(starts[s]) + i
            lo = max(0, at + 1 - window) if window else 0
            for h in range(heads):
                kk, vv = k[lo - base:at + 1 - base, h // G], v[lo - base:at + 1 - base, h // G]
                z = scale * (kk @ x[t, h])
                top = max(z.max(), -np.inf if sink is None else sink[h])
                w = np.exp(z - top)
                total = w.sum() + (0.0 if sink is None else np.exp(np.float64(sink[h]) - top))
                out[t, h] = w @ vv / total
                size = scale * (np.abs(kk) @ np.abs(x[t, h]))
                d = (u + (dim + 7) * 2.0 ** -24) * size.max()
                floor = 0.0 if cache.kind == BF16 else len(z) * 2.0 ** -35 * np.abs(vv).max()
                bound[t, h] = floor + (np.expm1(2 * d) + 2 * u + 2.0 ** -19 + 2.0 ** -22 * size.max() + len(z) * 2.0 ** -24) * (w @ np.abs(vv) / total)
    bound += HALF_STEP[out_kind] * (np.abs(out) + bound) + 1e-30 + (2.0 ** -25 if out_kind == F16 else 0)
    return out, bound


def angles_of(rng, tokens, pairs):
    a = rng.uniform(0, 2 * np.pi, (tokens, pairs))
    return np.stack([np.cos(a), np.sin(a)], -1).astype(np.float32)


def verify(target, draft, drafted, starts, accept, pick):
    """(accepted, tokens) by the definition, in float64"""
    accepted, tokens = [], np.full(len(drafted), 0xFFFFFFFF, np.uint32)
    for s in range(len(starts) - 1):
        a, b = starts[s], starts[s + 1]
        if a == b:
            accepted.append(0)
            continue
        n, got = b - a - 1, 0
        while got < n:
            d = drafted[a + got]
            if not float(accept[a + got]) * (1.0 if draft is None else float(draft[a + got, d])) < float(target[a + got, d]):
                break
            tokens[a + got] = d
            got += 1
        w = target[a + got].astype(np.float64)
        if got < n:
            q = draft[a + got].astype(np.float64) if draft is not None else np.eye(1, w.size, drafted[a + got])[0]
            rest = np.maximum(w - q, 0.0)
            w = rest if rest.sum() > 0 else w
        mass = np.cumsum(w)
        tokens[a + got] = np.argmax(mass > float(pick[s]) * mass[-1])
        accepted.append(got)
    return np.array(accepted, np.uint32), tokens
