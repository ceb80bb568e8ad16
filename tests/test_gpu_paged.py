"""A paged cache of keys and values in few bits and the attention over it on the GPU: bytes against the definition, attention against 64 bits on what the cache holds (kv_oracle.py;
bounds are those of attn_oracle.py)."""
import ctypes as C

import numpy as np
import pytest

from attn_oracle import U
from axiom_amd.hip import KvCache, KvRules
from kv_oracle import F16, I8, MX4, paged_attention, quantised, row_bytes

pytestmark = pytest.mark.gpu

TYPES = pytest.mark.parametrize("kind", [F16, I8, MX4], ids=["f16", "i8", "mx4"])


def say(*a):
    print(*a, flush=True)


class Cache:
    """Pages on the device, all bytes `fill` at first, and a table [B, cols] of host numbers"""

    def __init__(self, hip, kind, heads, dk, page_rows, table, pages, fill=0):
        self.hip, self.kind, self.heads, self.dk, self.page_rows, self.table, self.pages = hip, kind, heads, dk, page_rows, np.asarray(table, np.int32), pages
        shape = (pages, heads, page_rows, row_bytes(kind, dk))
        self.arrays = {n: hip.array(np.full(shape if "scale" not in n else shape[:3] + (4,), fill, np.uint8)) for n in ("k", "v", "k_scale", "v_scale")}
        self.d_table = hip.array(self.table)
        self.struct = KvCache(type=kind, page_rows=page_rows, pages=pages, heads=heads, dk=dk, table=self.d_table.ptr, table_ld=self.table.shape[1],
                              **{n: x.ptr for n, x in self.arrays.items()})

    def place(self, b, pos):
        """(page, row) or None"""
        page = int(self.table[b, pos // self.page_rows])
        return (page, pos % self.page_rows) if 0 <= page < self.pages else None

    def there(self, b, length):
        return np.array([self.place(b, j) is not None for j in range(length)], bool)


def table_of(rng, lens, page_rows, spare=1):
    """Pages in any order, as many as the lengths need, none behind them"""
    used = [-(-int(n) // page_rows) for n in lens]
    order = rng.permutation(sum(used) + 2)
    table = np.full((len(lens), max(used + [0]) + spare), -1, np.int32)
    at = 0
    for b, n in enumerate(used):
        table[b, :n] = order[at:at + n]
        at += n
    return table, sum(used) + 2


def rows_of(new):
    return np.concatenate([[0], np.cumsum(new)]).astype(np.int32)


def pitched(hip, x, ld, garbage=np.nan):
    """x [T, heads, dk] as rows of pitch ld"""
    full = np.full((len(x), ld), garbage, np.float32)
    full[:, :x.shape[1] * x.shape[2]] = x.reshape(len(x), -1)
    return hip.array(full)


def write(hip, cache, k, v, first, lens, Sq, pitch=0):
    ld = cache.heads * cache.dk + pitch
    dk, dv = pitched(hip, k, ld), pitched(hip, v, ld)
    f, n = None if first is None else hip.array(np.asarray(first, np.int32)), hip.array(np.asarray(lens, np.int32))
    hip.check(hip.L.axhip_kv_write(C.byref(cache.struct), dk.ptr, ld, dv.ptr, ld, f and f.ptr, n.ptr, len(lens), len(k), Sq))
    hip.sync()


def read(hip, cache, T, first, lens, Sq, pitch=0):
    ld = cache.heads * cache.dk + pitch
    out = [hip.array(np.full((T, ld), 7, np.float32)) for _ in range(2)]
    f, n = None if first is None else hip.array(np.asarray(first, np.int32)), hip.array(np.asarray(lens, np.int32))
    hip.check(hip.L.axhip_kv_read(C.byref(cache.struct), out[0].ptr, ld, out[1].ptr, ld, f and f.ptr, n.ptr, len(lens), T, Sq))
    got = [x.numpy() for x in out]
    assert all((x[:, cache.heads * cache.dk:] == 7).all() for x in got)
    return [x[:, :cache.heads * cache.dk].reshape(T, cache.heads, cache.dk) for x in got]


def fill(hip, cache, k, v, lens):
    """Whole sequences k[b], v[b] [lens[b], heads, dk] into the cache; gives back what it holds, in 64 bits"""
    T = sum(lens)
    if T:
        write(hip, cache, np.concatenate(k), np.concatenate(v), rows_of(lens), lens, max(lens))
    return [quantised(cache.kind, x)[2] for x in k], [quantised(cache.kind, x)[2] for x in v]


# ---- the cache -------------------------------------------------------------------------------------------------------

def values(rng, kind, rows, heads, dk):
    """Ordinary rows, and among them zeros, ties, subnormals, the largest floats, infinities and NaNs"""
    x = rng.normal(size=(rows, heads, dk)).astype(np.float32)
    x *= (2.0 ** rng.integers(-40, 40, (rows, heads, 1))).astype(np.float32)
    special = rng.integers(0, 12, (rows, heads))
    x[special == 0] = 0
    x[special == 1] *= np.float32(1e-38)
    x[special == 2] = (x[special == 2] * np.float32(2.0 ** -149))
    ties = np.concatenate([np.arange(-20, 21) / 4.0, [6, 7, 5, -5, 2.5, 3.5, -3.5, 127, -127, 126.5, 0.5, 64.5]]).astype(np.float32)
    tied = rng.choice(ties, size=x.shape).astype(np.float32)
    tied[..., 0] = 127 if kind == I8 else 7
    x[special == 3] = (tied * (2.0 ** rng.integers(-30, 30, (rows, heads, 1))).astype(np.float32))[special == 3]
    x[special == 4] = (rng.integers(-2 ** 12, 2 ** 12, x.shape) * 2.0 ** -11).astype(np.float32)[special == 4]
    big = special == 5
    x[big] = np.clip(rng.normal(size=x.shape) * 2e38, -3.4028234e38, 3.4028234e38).astype(np.float32)[big]
    for n, bad in ((6, np.inf), (7, -np.inf), (8, np.nan)):
        if (special == n).any():
            rows_, heads_ = np.nonzero(special == n)
            x[rows_, heads_, rng.integers(0, dk, len(rows_))] = bad
    return x


@TYPES
@pytest.mark.parametrize("dk,heads,page_rows", [(4, 3, 1), (12, 1, 2), (32, 4, 16), (36, 2, 8), (40, 5, 16), (64, 3, 64), (80, 2, 32), (96, 9, 16), (100, 1, 4), (128, 8, 16), (124, 2, 128)])
def test_bytes(hip, kind, dk, heads, page_rows):
    """What is written is the definition's bytes, in their places, and nothing else is touched; what is read is s n, and the rest of the caller's rows is left."""
    say("kv bytes", kind, dk, heads, page_rows)
    rng = np.random.default_rng(dk * 7 + heads + kind)
    new, lens = [5, 0, 1, 17, 3, 40], [5, 9, 30, 17, 2, 71]              # the fifth has padding: a row at position -1
    table, pages = table_of(rng, lens, page_rows)
    table[5, 35 // page_rows] = -1                                       # pages that are not there
    table[3, 0] = pages
    cache = Cache(hip, kind, heads, dk, page_rows, table, pages, fill=0xab)
    first, T = rows_of(new), sum(new)
    k, v = values(rng, kind, T, heads, dk), values(rng, kind, T, heads, dk)
    write(hip, cache, k, v, first, lens, 40, pitch=4 * (dk % 3))
    want = {n: np.full(cache.arrays[n].shape, 0xab, np.uint8) for n in cache.arrays}
    held, left = [np.full((T, heads, dk), 7.0) for _ in range(2)], np.ones(T, bool)
    for b in range(len(new)):
        for i in range(new[b]):
            t, pos = first[b] + i, lens[b] - new[b] + i
            at = cache.place(b, pos) if pos >= 0 else None
            if at is None:
                continue
            left[t] = False
            for n, x, out in (("k", k, held[0]), ("v", v, held[1])):
                payload, scales, value = quantised(kind, x[t:t + 1])
                want[n][at[0], :, at[1]], want[n + "_scale"][at[0], :, at[1]] = payload[0], scales[0]
                out[t] = value[0]
    assert left.any() and not left.all()
    for n in ("k_scale", "v_scale", "k", "v"):
        got, w = cache.arrays[n].numpy(), want[n]
        if kind != MX4 and "scale" in n:                                 # NaNs of any bits
            got, w = got.copy().view(np.float32), w.view(np.float32)
        assert np.array_equal(got, w, equal_nan=kind != MX4 and "scale" in n), (n, np.argwhere(got != w)[:5])
    for got, x in zip(read(hip, cache, T, first, lens, 40, pitch=8), held):
        with np.errstate(over="ignore"):
            x32 = x.astype(np.float32)
        other = np.argwhere(~((got == x32) | (np.isnan(got) & np.isnan(x32))))
        assert len(other) == 0, [(tuple(at), got[tuple(at)], x32[tuple(at)]) for at in other[:5]]


@TYPES
def test_rows_of_equal_counts(hip, kind):
    """Without `first`: Sq rows of each sequence, some of them padding; many sequences, so that their search takes several steps with it."""
    say("kv uniform", kind)
    rng = np.random.default_rng(3)
    B, Sq, heads, dk, page_rows = 150, 3, 2, 64, 16
    lens = rng.integers(0, 50, B)
    table, pages = table_of(rng, lens, page_rows)
    k, v = (rng.normal(size=(B * Sq, heads, dk)).astype(np.float32) for _ in range(2))
    got = []
    for first in (None, np.arange(B + 1) * Sq):
        cache = Cache(hip, kind, heads, dk, page_rows, table, pages)
        write(hip, cache, k, v, first, lens, Sq)
        got.append([cache.arrays[n].numpy() for n in ("k", "v", "k_scale", "v_scale")] + read(hip, cache, B * Sq, first, lens, Sq))
    for a, b in zip(*got):
        assert np.array_equal(a, b)
    pos = (lens[:, None] - Sq + np.arange(Sq)).reshape(-1)
    want = np.where((pos >= 0)[:, None, None], quantised(kind, k)[2].astype(np.float32), 7)
    assert np.array_equal(got[0][4], want)


@TYPES
@pytest.mark.parametrize("B", [64, 65, 4096, 5000])
def test_many_sequences(hip, kind, B):
    """Rows of unlike counts, none and one mostly, of so many sequences that the search for a row's takes one, two and three steps: written, read and attended to by both forms."""
    say("kv many", kind, B)
    rng = np.random.default_rng(B)
    heads, G, dk, page_rows = 1, 2, 32, 4
    new = rng.integers(0, 3, B)
    new[[0, B // 3, B - 1]] = [0, 70, 5]
    lens = new + rng.integers(0, 4, B)
    check(hip, kind, heads, G, dk, page_rows, new.tolist(), lens.tolist(), seed=B, behind=1)


def test_offsets_that_pass_32_bits(hip):
    """Pages past 4 GiB of a pool: written, read and attended to there."""
    say("kv far")
    rng = np.random.default_rng(4)
    heads, dk, page_rows, n = 8, 128, 256, 300
    pages = (5 << 30) // (heads * page_rows * row_bytes(F16, dk))
    size = pages * heads * page_rows
    L = hip.L
    at = {"k": L.axhip_malloc(size * row_bytes(F16, dk)), "v": L.axhip_malloc(size * row_bytes(F16, dk)), "k_scale": L.axhip_malloc(4 * size), "v_scale": L.axhip_malloc(4 * size)}
    try:
        assert all(at.values())
        table = hip.array(np.array([[pages - 1, pages - 3]], np.int32))
        struct = KvCache(type=F16, page_rows=page_rows, pages=pages, heads=heads, dk=dk, table=table.ptr, table_ld=2, **at)
        k, v, q = (rng.normal(size=(n, heads, dk)).astype(np.float32) for _ in range(3))
        ld = heads * dk
        dk_, dv, dq, lens, o, lse = hip.array(k), hip.array(v), hip.array(q), hip.array(np.array([n], np.int32)), hip.empty(q.shape), hip.empty((n, heads))
        back = [hip.empty(k.shape), hip.empty(k.shape)]
        hip.check(L.axhip_kv_write(C.byref(struct), dk_.ptr, ld, dv.ptr, ld, None, lens.ptr, 1, n, n))
        hip.check(L.axhip_kv_read(C.byref(struct), back[0].ptr, ld, back[1].ptr, ld, None, lens.ptr, 1, n, n))
        hip.check(L.axhip_attn_paged(dq.ptr, ld, C.byref(struct), o.ptr, ld, lse.ptr, None, lens.ptr, 1, n, heads, n, n, 0.1, None))
        kk, vv = quantised(F16, k)[2], quantised(F16, v)[2]
        assert np.array_equal(back[0].numpy(), kk.astype(np.float32)) and np.array_equal(back[1].numpy(), vv.astype(np.float32))
        w = paged_attention(q, kk, vv, np.ones(n, bool), 0.1)
        within(o.numpy(), w, "o")
        within(lse.numpy(), w, "lse")
        for b in range(3):                                               # a token of it, by the other form
            one = hip.array(q[n - 1 - b:n - b])
            hip.check(L.axhip_attn_paged(one.ptr, ld, C.byref(struct), o.ptr, ld, lse.ptr, None, hip.array(np.array([n - b], np.int32)).ptr, 1, 1, heads, 1, n, 0.1, None))
            assert (np.abs(o.numpy()[0] - w["o"][n - 1 - b]) <= w["tol_o"][n - 1 - b]).all()
    finally:
        hip.sync()
        for p in at.values():
            L.axhip_free(p)


# ---- attention -------------------------------------------------------------------------------------------------------

def within(got, want, n):
    same = np.isneginf(got) & np.isneginf(want[n])
    off, tol = np.abs(np.where(same, 0, got) - np.where(same, 0, want[n])), want["tol_" + n]
    bad = ~(off <= tol)
    if bad.any():
        at = np.unravel_index(np.argmax(np.where(bad, np.nan_to_num(off / np.maximum(tol, 1e-300), nan=np.inf), 0)), off.shape)
        pytest.fail("%s: %d of %d out of bounds, the worst at %s: %r, not %r +- %r" % (n, bad.sum(), bad.size, at, got[at], want[n][at], tol[at]))


def attend(hip, cache, q, new, lens, rules=None, scale=None, uniform=False, pitch=0, Sk=None, kernel=None, slopes=None, behind=0):
    """q [T, H, dk] -> (o [T, H, dk], lse [T, H]); `behind` rows of no sequence come after T and are checked to be left as they were"""
    T, H, dk = q.shape
    ld = H * dk + pitch
    dq = pitched(hip, np.concatenate([q, np.full((behind, H, dk), np.nan, np.float32)]), ld)
    o, lse = hip.array(np.full((T + behind, ld), 7, np.float32)), hip.array(np.full((T + behind, H), 7, np.float32))
    first, n = hip.array(rows_of(new)), hip.array(np.asarray(lens, np.int32))
    held = hip.array(np.asarray(slopes, np.float32)) if slopes is not None else None
    r = KvRules(slopes=held and held.ptr, **(rules or {}))
    hip.check(hip.L.axhip_attn_paged(dq.ptr, ld, C.byref(cache.struct), o.ptr, ld, lse.ptr, None if uniform else first.ptr, n.ptr, len(lens), T + behind if not uniform else T, H, max(new),
                                     max(max(lens), 0) if Sk is None else Sk, dk ** -0.5 if scale is None else scale, C.byref(r)))
    if kernel:
        assert hip.last_kernel() == kernel, hip.last_kernel()
    full, sums = o.numpy(), lse.numpy()
    assert (full[:, H * dk:] == 7).all() and (full[T:] == 7).all() and (sums[T:] == 7).all()
    return full[:T, :H * dk].reshape(T, H, dk), sums[:T]


def check(hip, kind, heads, G, dk, page_rows, new, lens, rules=None, slopes=False, holes=(), seed=0, want=None, pitch=0, **kw):
    """Sequences of these lengths in a cache, their last `new` rows as queries, against 64 bits; gives back what came out."""
    rng = np.random.default_rng(seed + 31 * dk + kind)
    H = heads * G
    stored = [max(n, 0) for n in lens]
    table, pages = table_of(rng, stored, page_rows)
    for b, col in holes:
        table[b, col] = -1 if col % 2 else pages + 5
    cache = Cache(hip, kind, heads, dk, page_rows, table, pages, fill=0xff)
    k, v = ([rng.normal(size=(n, heads, dk)).astype(np.float32) for n in stored] for _ in range(2))
    kk, vv = fill(hip, cache, k, v, stored)
    q = rng.normal(size=(sum(new), H, dk)).astype(np.float32)
    slope = (2.0 ** -np.arange(1, H + 1)).astype(np.float32) if slopes else None
    o, lse = attend(hip, cache, q, new, lens, rules, slopes=slope, pitch=pitch, **kw)
    first = rows_of(new)
    for b in range(len(new)):
        n = min(new[b], stored[b])
        at = slice(first[b + 1] - n, first[b + 1])
        pad = slice(first[b], first[b + 1] - n)
        assert (o[pad] == 0).all() and np.isneginf(lse[pad]).all()
        if n == 0:
            continue
        w = paged_attention(q[at], kk[b], vv[b], cache.there(b, stored[b]), dk ** -0.5, slopes=slope, **(rules or {}))
        within(o[at], w, "o")
        within(lse[at], w, "lse")
        empty = np.isneginf(w["lse"])
        assert (o[at][empty] == 0).all() and np.isneginf(lse[at][empty]).all()
    return o, lse


RULES = {"plain": {}, "window": dict(window=19), "sinks": dict(window=40, sinks=5), "wide": dict(window=1000, sinks=3), "one": dict(window=1), "late": dict(window=7, sinks=70),
         "cap": dict(cap=2.0), "slopes": {}, "all": dict(cap=20.0, window=50, sinks=33)}


@TYPES
@pytest.mark.parametrize("rules", RULES)
@pytest.mark.parametrize("dk,heads,G", [(64, 2, 4), (128, 1, 8), (80, 2, 1), (32, 1, 2), (20, 2, 3), (4, 3, 5), (104, 1, 16)])
def test_tokens(hip, kind, rules, dk, heads, G):
    """One token, a few, none, more than there are positions: the form for few rows."""
    say("tokens", kind, rules, dk, heads, G)
    new = [1, 1, 3, 0, 4, 1, 2, 1]
    check(hip, kind, heads, G, dk, 16, new, [1, 33, 150, 12, 70, 64, 1, 0], RULES[rules], rules in ("slopes", "all"), pitch=4 * (dk % 3), behind=2)


@TYPES
@pytest.mark.parametrize("rules", RULES)
@pytest.mark.parametrize("dk,heads,G,page_rows", [(64, 2, 4, 32), (128, 2, 2, 16), (96, 1, 3, 64), (40, 1, 40, 8), (112, 2, 1, 128), (32, 1, 8, 1), (4, 2, 3, 16)])
def test_chunks(hip, kind, rules, dk, heads, G, page_rows):
    """Chunks of unlike lengths, single tokens and nothing beside them: both forms in one call."""
    say("chunks", kind, rules, dk, heads, G, page_rows)
    new = [70, 1, 0, 33, 9, 2, 140]
    check(hip, kind, heads, G, dk, page_rows, new, [70, 200, 12, 100, 8, 1, 300], RULES[rules], rules in ("slopes", "all"), pitch=4 * (dk % 3), behind=3)


@TYPES
@pytest.mark.parametrize("dk", [64, 128, 72])
@pytest.mark.parametrize("new,lens,kernel", [([1], [2000], "paged_few_ranges"), ([1] * 600, [40] * 600, "paged_few"), ([70], [300], "paged_few"), ([30] * 30, [3000] * 30, "paged_tiles_128_ranges"),
                                             ([30] * 100, [40] * 99 + [3], "paged_tiles_128"), ([700] * 3, [1800, 700, 5], "paged_tiles_256_ranges"), ([257] * 12, [300] * 12, "paged_tiles_256")],
                         ids=lambda v: str(v)[:12])
def test_forms(hip, kind, dk, new, lens, kernel):
    """Each form, by the kernel that it says it is."""
    say("forms", kind, dk, kernel)
    heads, G = (23, 1) if kernel == "paged_tiles_256" else (2, 4) if len(new) <= 100 else (1, 2)
    check(hip, kind, heads, G, dk, 64, new, lens, dict(window=1500, sinks=70) if dk == 72 else {}, uniform=True, kernel=kernel)


@TYPES
def test_pages_that_are_not_there(hip, kind):
    """Keys on no page are not seen; a row that sees nothing but those is empty."""
    say("holes", kind)
    check(hip, kind, 2, 2, 64, 16, [1, 20, 90, 3], [40, 64, 130, 30], holes=[(0, 0), (1, 1), (1, 2), (2, 3), (2, 5), (3, 0), (3, 1)])
    check(hip, kind, 2, 2, 64, 16, [1, 20, 90, 3], [40, 64, 130, 30], dict(window=10, sinks=2), holes=[(0, 2), (1, 1), (2, 0), (2, 4), (3, 1)])
    check(hip, kind, 1, 8, 128, 8, [2], [400], holes=[(0, n) for n in range(50)])


@TYPES
@pytest.mark.parametrize("dk", [64, 128])
def test_same_bits(hip, kind, dk):
    """Ranges of keys are added in order: the same call gives the same bits, whoever arrives last, and leaves the counters for the next."""
    say("same bits", kind, dk)
    rng = np.random.default_rng(9)
    lens, heads, G = [3000, 1700], 2, 4
    table, pages = table_of(rng, lens, 32)
    cache = Cache(hip, kind, heads, dk, 32, table, pages)
    fill(hip, cache, *([rng.normal(size=(n, heads, dk)).astype(np.float32) for n in lens] for _ in range(2)), lens)
    for new in ([1, 1], [40, 90]):
        q = rng.normal(size=(sum(new), heads * G, dk)).astype(np.float32)
        outs = [attend(hip, cache, q, new, lens) for _ in range(5)]
        for o, lse in outs[1:]:
            assert np.array_equal(o, outs[0][0]) and np.array_equal(lse, outs[0][1])


@TYPES
@pytest.mark.parametrize("new", [[1, 1], [60, 70]])
def test_infinities_and_nans(hip, kind, new):
    """A NaN key, an infinite value: rows that do not see them, and other heads, are as if they were not there; those that do are NaN, and for MX4 values only in the group's columns."""
    say("nan rows", kind, new)
    rng = np.random.default_rng(10)
    heads, G, dk, lens = 2, 2, 64, [150, 180]
    table, pages = table_of(rng, lens, 16)
    cache = Cache(hip, kind, heads, dk, 16, table, pages)
    k, v = ([rng.normal(size=(n, heads, dk)).astype(np.float32) for n in lens] for _ in range(2))
    k[0][100, 0, 3] = np.nan
    v[1][130, 1, 5] = np.inf
    kk, vv = fill(hip, cache, k, v, lens)
    q = rng.normal(size=(sum(new), heads * G, dk)).astype(np.float32)
    for rules in ({}, dict(window=30, sinks=4)):
        o, lse = attend(hip, cache, q, new, lens, rules)
        first = rows_of(new)
        for b in range(2):
            at = slice(first[b], first[b + 1])
            p = lens[b] - new[b] + np.arange(new[b])
            bad_at, head = (100, 0) if b == 0 else (130, 1)
            sees = (p >= bad_at) & ((p - bad_at < rules["window"]) if rules else True)
            clean_k, clean_v = np.nan_to_num(kk[b]), np.nan_to_num(vv[b])
            w = paged_attention(q[at], clean_k, clean_v, np.ones(lens[b], bool), dk ** -0.5, **rules)
            hit = np.zeros((new[b], heads * G), bool)
            hit[:, head * G:(head + 1) * G] = sees[:, None]
            within(np.where(hit[..., None], w["o"], o[at]), w, "o")
            if b == 0:
                assert np.isnan(o[at][hit]).all() and np.isnan(lse[at][hit]).all()
                within(np.where(hit, w["lse"], lse[at]), w, "lse")
            else:
                within(lse[at], w, "lse")
                cols = np.arange(dk) < (32 if kind == MX4 else dk)
                assert np.isnan(o[at][hit][:, cols]).all()
                if kind == MX4:
                    good = np.broadcast_to(hit[..., None] & ~cols, o[at].shape)
                    within(np.where(good, o[at], w["o"]), w, "o")


@TYPES
@pytest.mark.parametrize("new", [1, 40, 130])
@pytest.mark.parametrize("garbage", [0xff, 0x7c])
def test_rows_that_were_never_written(hip, kind, new, garbage):
    """Positions behind a window that hold bytes of all kinds (NaNs and infinities as f16 and as scales), on pages that are there: as if they were not."""
    say("never written", kind, new, garbage)
    rng = np.random.default_rng(13)
    heads, G, dk, length, window = 2, 4, 64, 300, 30
    written = new + window
    table, pages = table_of(rng, [length], 16)
    cache = Cache(hip, kind, heads, dk, 16, table, pages, fill=garbage)
    k, v = (rng.normal(size=(written, heads, dk)).astype(np.float32) for _ in range(2))
    write(hip, cache, k, v, None, [length], written)
    q = rng.normal(size=(new, heads * G, dk)).astype(np.float32)
    o, lse = attend(hip, cache, q, [new], [length], dict(window=window))
    kk, vv = (np.concatenate([np.zeros((length - written, heads, dk)), quantised(kind, x)[2]]) for x in (k, v))
    w = paged_attention(q, kk, vv, np.ones(length, bool), dk ** -0.5, window=window)
    within(o, w, "o")
    within(lse, w, "lse")


@TYPES
@pytest.mark.parametrize("new", [[1, 2], [60, 70]])
def test_sizes_far_apart(hip, kind, new):
    """Huge values and keys that a window hides, rows of zeros, tiny rows, huge keys under tiny queries."""
    say("sizes", kind, new)
    rng = np.random.default_rng(11)
    heads, G, dk, lens = 2, 2, 64, [150, 180]
    table, pages = table_of(rng, lens, 16)
    first = rows_of(new)

    def hold(k, v, q, scale, rules):
        cache = Cache(hip, kind, heads, dk, 16, table, pages)
        kk, vv = fill(hip, cache, k, v, lens)
        o, lse = attend(hip, cache, q, new, lens, rules, scale=scale)
        for b in range(2):
            at = slice(first[b], first[b + 1])
            w = paged_attention(q[at], kk[b], vv[b], np.ones(lens[b], bool), scale, **rules)
            # A probability's reference is the largest of the scores and their values' scales: 2^(y), where y is by log2 of the scale, and the scales' own 34 bits, further from zero than the
            # score.  y is rounded by U |y| (a probability by that times ln 2, twice in o: itself and the sum), and so are the logarithm of the sum and what it is added to.
            top = np.abs(vv[b]).max(-1)
            apart = np.abs(np.log2(np.where(top > 0, top, 2.0 ** -100))).max() + 34
            w["tol_o"] = w["tol_o"] * (1 + 2 * U * apart) + 2 * U * np.log(2) * apart * mean_size(q[at], kk[b], vv[b], scale, rules)
            w["tol_lse"] = w["tol_lse"] + np.where(np.isfinite(w["lse"]), 3 * U * np.log(2) * apart, 0)
            within(o[at], w, "o")
            within(lse[at], w, "lse")

    def mean_size(q, k, v, scale, rules):
        return paged_attention(q, k, np.abs(v), np.ones(len(k), bool), scale, **rules)["o"]

    def draw():
        return ([rng.normal(size=(n, heads, dk)).astype(np.float32) for n in lens] for _ in range(2))

    q = rng.normal(size=(sum(new), heads * G, dk)).astype(np.float32)
    k, v = draw()
    for b in range(2):
        k[b][10] *= np.float32(1e30)
        v[b][12] *= np.float32(1e30)
        v[b][60] *= np.float32(1e20)                                     # some rows of the chunks see it
    hold(k, v, q, 0.125, dict(window=30, sinks=4))
    k, v = draw()
    for b in range(2):
        v[b][::3] = 0
        k[b][1::3] = 0
    hold(k, v, q, 0.125, {})
    hold([x * 0 for x in k], [x * 0 for x in v], q, 0.125, {})
    k, v = draw()
    hold([x * np.float32(1e25) for x in k], [x * np.float32(1e-25) for x in v], q * np.float32(1e-25), 0.125, {})
    hold([x * np.float32(1e-20) for x in k], [x * np.float32(1e20) for x in v], q * np.float32(1e20), 0.125, {})
    v[0] *= (10.0 ** rng.integers(-12, 12, (lens[0], 1, 1))).astype(np.float32)
    hold(k, v, q, 0.125, {})
    hold(k, [x * np.float32(2.0 ** 80) for x in draw().__next__()], q, 0.125, {})


@pytest.mark.parametrize("seed", range(48))
def test_drawn(hip, seed):
    """Any types, heads, pages, rules, counts and holes together."""
    rng = np.random.default_rng(1000 + seed)
    kind, heads, G, dk, page_rows = int(rng.integers(3)), int(rng.integers(1, 5)), int(rng.integers(1, 20)), 4 * int(rng.integers(1, 33)), 1 << int(rng.integers(0, 9))
    B, most = int(rng.integers(1, 9)), int(rng.choice([1, 2, 9, 40, 150, 400]))
    new = rng.integers(0, most + 1, B)
    new[0] = most
    lens = np.maximum(new + rng.integers(-2, 300, B) * rng.integers(0, 2, B), 0)
    if rng.random() < 0.3:
        new[:] = most
    rules = {}
    if rng.random() < 0.5:
        rules.update(window=int(rng.choice([1, 3, 31, 32, 33, 64, 100, 257])), sinks=int(rng.choice([0, 1, 4, 32, 33, 130])))
    if rng.random() < 0.3:
        rules.update(cap=float(rng.choice([0.5, 5.0, 50.0])))
    holes = [(b, int(rng.integers(0, max(1, -(-int(lens[b]) // page_rows))))) for b in range(B) if lens[b] and rng.random() < 0.3]
    say("drawn", seed, kind, heads, G, dk, page_rows, new.tolist(), lens.tolist(), rules, holes)
    check(hip, kind, heads, G, dk, page_rows, new.tolist(), lens.tolist(), rules, bool(rng.random() < 0.3), holes, seed, pitch=4 * int(rng.integers(0, 3)), behind=int(rng.integers(0, 3)),
          uniform=False)


# ---- together --------------------------------------------------------------------------------------------------------

@TYPES
@pytest.mark.parametrize("rules", [{}, dict(window=24, sinks=2)])
def test_a_layer_serving(hip, kind, rules):
    """A decoder layer between its projections, served: prompts in chunks, then single tokens, with a sequence that joins late, on rows of a fused projection: norm and rotation in place,
    write, attention; every step against the whole sequences in 64 bits, and the cache read back to contiguous rows for axhip_attn_fwd."""
    say("serving", kind, rules)
    rng = np.random.default_rng(12)
    heads, G, dk, page_rows, B = 2, 2, 64, 16, 3
    H, wide = heads * G, (heads * G + 2 * heads) * dk
    steps = [[40, 0, 17], [33, 0, 1], [1, 60, 1], [1, 1, 1], [0, 1, 1]]
    total = np.sum(steps, 0)
    order = rng.permutation(64)
    table, at = np.full((B, 8), -1, np.int32), 0
    cache = Cache(hip, kind, heads, dk, page_rows, table, 64)
    x = [rng.normal(size=(n, wide)).astype(np.float32) for n in total]
    gq, gk = ((1 + 0.2 * rng.normal(size=dk)).astype(np.float32) for _ in range(2))
    freq = hip.empty((dk // 2,))
    hip.check(hip.L.axhip_rope_frequencies(freq.ptr, dk, 10000.0, 0, 1.0, 0.0, 0.0, 0))
    d_gq, d_gk = hip.array(gq), hip.array(gk)
    done = np.zeros(B, int)
    seen = [[np.zeros((0, h, dk), np.float32) for _ in range(B)] for h in (H, heads, heads)]
    for new in steps:
        before, done = done, done + new
        for b in range(B):                                               # pages as they are needed
            while (table[b] >= 0).sum() * page_rows < done[b]:
                table[b, (table[b] >= 0).sum()] = order[at]
                at += 1
        cache.table = table
        cache.d_table.upload(table)
        rows = np.concatenate([x[b][before[b]:done[b]] for b in range(B)])
        pos = np.concatenate([np.arange(before[b], done[b]) for b in range(B)]).astype(np.int32)
        T, first, lens = len(rows), hip.array(rows_of(new)), hip.array(done.astype(np.int32))
        qkv, d_pos, o, lse = hip.array(rows), hip.array(pos), hip.empty((T, H * dk)), hip.empty((T, H))
        hip.check(hip.L.axhip_qk_norm_rope_fwd(qkv.ptr, wide, qkv.ptr, wide, None, d_gq.ptr, d_gk.ptr, 1e-6, d_pos.ptr, freq.ptr, T, H, heads, dk, dk, 1.0, 1))
        k, v = qkv.ptr + 4 * H * dk, qkv.ptr + 4 * (H + heads) * dk
        hip.check(hip.L.axhip_kv_write(C.byref(cache.struct), k, wide, v, wide, first.ptr, lens.ptr, B, T, max(new)))
        r = KvRules(**rules)
        hip.check(hip.L.axhip_attn_paged(qkv.ptr, wide, C.byref(cache.struct), o.ptr, H * dk, lse.ptr, first.ptr, lens.ptr, B, T, H, max(new), int(done.max()), dk ** -0.5, C.byref(r)))
        turned, got, sums, f = qkv.numpy(), o.numpy().reshape(T, H, dk), lse.numpy(), rows_of(new)
        for b in range(B):
            mine = slice(f[b], f[b + 1])
            parts = np.split(turned[mine], [H * dk, (H + heads) * dk], 1)
            for i, part in enumerate(parts):
                seen[i][b] = np.concatenate([seen[i][b], part.reshape(new[b], part.shape[1] // dk, dk)])
            if new[b]:
                w = paged_attention(seen[0][b][-new[b]:], quantised(kind, seen[1][b])[2], quantised(kind, seen[2][b])[2], np.ones(done[b], bool), dk ** -0.5, **rules)
                within(got[mine], w, "o")
                within(sums[mine], w, "lse")
    back = read(hip, cache, int(done.sum()), rows_of(done), done, int(done.max()))
    for i in range(2):
        assert np.array_equal(back[i], np.concatenate([quantised(kind, y)[2] for y in seen[i + 1]]).astype(np.float32))
    if not rules:                                                        # contiguous rows of one sequence, by the attention that reads those
        b = int(done.argmax())
        f = rows_of(done)
        kb, vb, qb = hip.array(back[0][f[b]:f[b + 1]]), hip.array(back[1][f[b]:f[b + 1]]), hip.array(seen[0][b])
        n = int(done[b])
        o1, o2, l1, l2 = hip.empty((n, H * dk)), hip.empty((n, H * dk)), hip.empty((1, H, n)), hip.empty((n, H))
        from axiom_amd.hip import AttnRules
        causal = AttnRules(causal=1)
        hip.check(hip.L.axhip_attn_fwd(qb.ptr, H * dk, kb.ptr, heads * dk, vb.ptr, heads * dk, n, o1.ptr, H * dk, l1.ptr, 1, H, heads, n, n, dk, dk ** -0.5, C.byref(causal)))
        one = KvCache.from_buffer_copy(cache.struct)
        one.table = cache.d_table.ptr + 4 * 8 * b
        hip.check(hip.L.axhip_attn_paged(qb.ptr, H * dk, C.byref(one), o2.ptr, H * dk, l2.ptr, None, hip.array(np.array([n], np.int32)).ptr, 1, n, H, n, n, dk ** -0.5, None))
        w = paged_attention(seen[0][b], quantised(kind, seen[1][b])[2], quantised(kind, seen[2][b])[2], np.ones(n, bool), dk ** -0.5)
        assert (np.abs(o1.numpy() - o2.numpy()).reshape(n, H, dk) <= 3 * w["tol_o"]).all()
        assert (np.abs(l1.numpy()[0].T - l2.numpy()) <= 3 * w["tol_lse"]).all()
