"""Attention over a paged cache by tiles of queries and by ranges of their keys, where it can go wrong: NaNs and infinities, garbage behind a window, sizes far apart, the same bits, a pool past 4 GiB.
Each call says which form it must be: sequences without new rows beside those with many make a batch that the form for few rows does not take as a whole (64-bit forms and bounds: kv_oracle.py)."""
import ctypes as C

import numpy as np
import pytest

from attn_oracle import U
from axiom_amd.hip import KvCache
from kv_oracle import F16, I8, MX4, paged_attention, quantised, row_bytes
from test_gpu_paged import Cache, TYPES, attend, check, fill, rows_of, say, table_of, within, write

pytestmark = pytest.mark.gpu

NONE = [0] * 4                       # sequences that are there and have no new rows
NEW = [60, 70] + NONE
# (query heads to a head of keys, lengths, a window that hides some keys, the kernel): 32 or 16 rows of tokens a wave, keys in one range and in several, which a second launch adds
FORMS = [(1, [150, 180], 30, "paged_tiles_128"), (2, [150, 180], 30, "paged_tiles_256"), (1, [1500, 1700], 900, "paged_tiles_128_ranges"), (2, [1500, 1700], 900, "paged_tiles_256_ranges")]
forms = pytest.mark.parametrize("G,lens,window,kernel", FORMS, ids=[f[-1] for f in FORMS])


def normal(rng, n, heads, dk):
    return rng.normal(size=(n, heads, dk)).astype(np.float32)


@TYPES
@pytest.mark.parametrize("dk", [64, 128, 32, 96])
@pytest.mark.parametrize("G,kernel", [(1, "paged_tiles_128_ranges"), (2, "paged_tiles_256_ranges")])
def test_same_bits(hip, kind, dk, G, kernel):
    """Ranges of keys are added in order: the same call gives the same bits."""
    say("tiles same bits", kind, dk, kernel)
    rng = np.random.default_rng(29)
    lens, heads, new = [3000, 1700] + NONE, 2, [70, 60] + NONE
    table, pages = table_of(rng, lens, 32)
    cache = Cache(hip, kind, heads, dk, 32, table, pages)
    fill(hip, cache, *([normal(rng, n, heads, dk) for n in lens] for _ in range(2)), lens)
    q = normal(rng, sum(new), heads * G, dk)
    outs = [attend(hip, cache, q, new, lens, kernel=kernel) for _ in range(5)]
    for o, lse in outs[1:]:
        assert np.array_equal(o, outs[0][0]) and np.array_equal(lse, outs[0][1])


@TYPES
@forms
@pytest.mark.parametrize("dk", [64, 128, 80])
@pytest.mark.parametrize("narrow", [False, True], ids=["all", "window"])
def test_infinities_and_nans(hip, kind, G, lens, window, kernel, dk, narrow):
    """A NaN key, an infinite value: rows that do not see them, and other heads, are as if they were not there; those that do are NaN, and for 4-bit values only in the group's columns."""
    say("tiles nan rows", kind, kernel, dk, narrow)
    rng = np.random.default_rng(30)
    heads, lens = 2, lens + NONE
    rules = dict(window=window, sinks=4) if narrow else {}
    table, pages = table_of(rng, lens, 16)
    cache = Cache(hip, kind, heads, dk, 16, table, pages)
    k, v = ([normal(rng, n, heads, dk) for n in lens] for _ in range(2))
    bad_key, bad_value = lens[0] - 50, lens[1] - 50                      # behind the first of the new rows, so that those do not see them
    k[0][bad_key, 0, 3] = np.nan
    v[1][bad_value, 1, 5] = np.inf
    k[0][lens[0] - 60 - window - 20, 1] = np.inf                         # and before every row's window
    kk, vv = fill(hip, cache, k, v, lens)
    q = normal(rng, sum(NEW), heads * G, dk)
    o, lse = attend(hip, cache, q, NEW, lens, rules, kernel=kernel)
    first = rows_of(NEW)
    for b in range(2):
        at = slice(first[b], first[b + 1])
        p = lens[b] - NEW[b] + np.arange(NEW[b])
        bad_at, head = (bad_key, 0) if b == 0 else (bad_value, 1)
        hit = np.zeros((NEW[b], heads * G), bool)
        hit[:, head * G:(head + 1) * G] = ((p >= bad_at) & ((p - bad_at < window) if narrow else True))[:, None]
        if b == 0 and not narrow:
            hit[:, G:] = True
        assert hit.any() and not hit.all()
        w = paged_attention(q[at], np.nan_to_num(kk[b]), np.nan_to_num(vv[b]), np.ones(lens[b], bool), dk ** -0.5, **rules)
        within(np.where(hit[..., None], w["o"], o[at]), w, "o")
        if b == 0:
            assert np.isnan(o[at][hit]).all() and np.isnan(lse[at][hit]).all()
            within(np.where(hit, w["lse"], lse[at]), w, "lse")
        else:
            within(lse[at], w, "lse")
            cols = np.arange(dk) < (32 if kind == MX4 else dk)
            assert np.isnan(o[at][hit][:, cols]).all()
            if kind == MX4:
                within(np.where(hit[..., None] & ~cols, o[at], w["o"]), w, "o")


@TYPES
@forms
@pytest.mark.parametrize("dk", [64, 128])
@pytest.mark.parametrize("garbage", [0xff, 0x7c])
def test_rows_that_were_never_written(hip, kind, G, lens, window, kernel, dk, garbage):
    """Positions behind a window that hold bytes of all kinds (NaNs and infinities as f16 and as scales), on pages that are there: as if they were not."""
    say("tiles never written", kind, kernel, dk, garbage)
    rng = np.random.default_rng(31)
    heads, new, length = 2, [70] + NONE, lens[1]
    written = 70 + window
    table, pages = table_of(rng, [length] + NONE, 16)
    cache = Cache(hip, kind, heads, dk, 16, table, pages, fill=garbage)
    k, v = (normal(rng, written, heads, dk) for _ in range(2))
    write(hip, cache, k, v, None, [length], written)
    q = normal(rng, 70, heads * G, dk)
    o, lse = attend(hip, cache, q, new, [length] + NONE, dict(window=window), kernel=kernel)
    kk, vv = (np.concatenate([np.zeros((length - written, heads, dk)), quantised(kind, x)[2]]) for x in (k, v))
    w = paged_attention(q, kk, vv, np.ones(length, bool), dk ** -0.5, window=window)
    within(o, w, "o")
    within(lse, w, "lse")


def held(hip, kind, G, dk, lens, kernel, k, v, q, scale, rules, new=NEW):
    """Sequences k[b], v[b] in a cache, queries q, against 64 bits with what values' sizes cost"""
    rng = np.random.default_rng(32)
    heads, first = k[0].shape[1], rows_of(new)
    table, pages = table_of(rng, lens, 16)
    cache = Cache(hip, kind, heads, dk, 16, table, pages)
    kk, vv = fill(hip, cache, k, v, lens)
    o, lse = attend(hip, cache, q, new, lens, rules, scale=scale, kernel=kernel)
    for b in range(2):
        at, there = slice(first[b], first[b + 1]), np.ones(lens[b], bool)
        w = paged_attention(q[at], kk[b], vv[b], there, scale, **rules)
        # A probability's reference is the largest of the scores and their values' scales: 2^(y), where y is by log2 of the scale, and the scales' own 34 bits, further from zero than the
        # score.  y is rounded by U |y| (a probability by that times ln 2, twice in o: itself and the sum), and so are the logarithm of the sum and what it is added to.
        top = np.abs(vv[b]).max(-1)
        apart = np.abs(np.log2(np.where(top > 0, top, 2.0 ** -100))).max() + 34
        size = paged_attention(q[at], kk[b], np.abs(vv[b]), there, scale, **rules)["o"]
        w["tol_o"] = w["tol_o"] * (1 + 2 * U * apart) + 2 * U * np.log(2) * apart * size
        w["tol_lse"] = w["tol_lse"] + np.where(np.isfinite(w["lse"]), 3 * U * np.log(2) * apart, 0)
        within(o[at], w, "o")
        within(lse[at], w, "lse")


@TYPES
@forms
def test_sizes_far_apart(hip, kind, G, lens, window, kernel):
    """Huge values and keys that a window hides, rows of zeros, tiny rows, huge keys under tiny queries, values whose rows are formed again."""
    say("tiles sizes", kind, kernel)
    rng = np.random.default_rng(33)
    heads, dk, lens = 2, 64, lens + NONE

    def draw():
        return ([normal(rng, n, heads, dk) for n in lens] for _ in range(2))

    def hold(k, v, q, scale, rules):
        held(hip, kind, G, dk, lens, kernel, k, v, q, scale, rules)

    q = normal(rng, sum(NEW), heads * G, dk)
    k, v = draw()
    for b in range(2):
        k[b][10] *= np.float32(1e30)
        v[b][12] *= np.float32(1e30)
        v[b][lens[b] - NEW[b] - window + 30] *= np.float32(1e20)         # some rows of the chunks see it
    hold(k, v, q, 0.125, dict(window=window, sinks=4))
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


@TYPES
@forms
@pytest.mark.parametrize("rules", [{}, dict(sinks=40), dict(cap=5.0)], ids=["plain", "window", "cap"])
def test_pages_that_are_not_there(hip, kind, G, lens, window, kernel, rules):
    """Keys on no page are not seen, also where whole blocks have none, and a row that sees nothing but those is empty."""
    say("tiles holes", kind, kernel, rules)
    if "sinks" in rules:
        rules = dict(rules, window=window)
    holes = [(0, 0), (0, 3), (1, 1), (1, (lens[1] - 1) // 16)] + [(0, n) for n in range(5, 9)]
    check(hip, kind, 2, G, 64, 16, NEW, lens + NONE, rules, holes=holes, kernel=kernel)
    check(hip, kind, 2, G, 72, 16, NEW, lens + NONE, rules, holes=[(1, n) for n in range(-(-lens[1] // 16))], kernel=kernel)


@pytest.mark.parametrize("kind,dk", [(F16, 128), (I8, 128), (MX4, 64)])
def test_offsets_that_pass_32_bits(hip, kind, dk):
    """Pages past 4 GiB of a pool, and their scales, attended to by tiles, in one range of keys and in several, and by single tokens."""
    say("tiles far", kind, dk)
    rng = np.random.default_rng(34)
    L, heads, page_rows, n = hip.L, 8, 256, 1400
    pages = (5 << 30) // (heads * page_rows * row_bytes(kind, dk))
    size = pages * heads * page_rows
    at = {"k": L.axhip_malloc(size * row_bytes(kind, dk)), "v": L.axhip_malloc(size * row_bytes(kind, dk)), "k_scale": L.axhip_malloc(4 * size), "v_scale": L.axhip_malloc(4 * size)}
    try:
        assert all(at.values())
        own = np.full((5, 6), -1, np.int32)
        own[0] = pages - 1 - rng.permutation(6)
        table = hip.array(own)
        struct = KvCache(type=kind, page_rows=page_rows, pages=pages, heads=heads, dk=dk, table=table.ptr, table_ld=6, **at)
        k, v, q = normal(rng, n, heads, dk), normal(rng, n, heads, dk), normal(rng, 80, heads, dk)
        ld = heads * dk
        d_k, d_v, d_q, lens, o, lse = hip.array(k), hip.array(v), hip.array(q), hip.array(np.array([n] + NONE, np.int32)), hip.empty(q.shape), hip.empty((80, heads))
        hip.check(L.axhip_kv_write(C.byref(struct), d_k.ptr, ld, d_v.ptr, ld, None, lens.ptr, 1, n, n))
        kk, vv = quantised(kind, k)[2], quantised(kind, v)[2]
        first = hip.array(rows_of([80] + NONE))
        for length, kernel in ((n, "paged_tiles_128_ranges"), (300, "paged_tiles_128")):
            lengths = hip.array(np.array([length] + NONE, np.int32))
            hip.check(L.axhip_attn_paged(d_q.ptr, ld, C.byref(struct), o.ptr, ld, lse.ptr, first.ptr, lengths.ptr, 5, 80, heads, 80, length, 0.1, None))
            assert hip.last_kernel() == kernel, hip.last_kernel()
            w = paged_attention(q, kk[:length], vv[:length], np.ones(length, bool), 0.1)
            within(o.numpy(), w, "o")
            within(lse.numpy(), w, "lse")
        hip.check(L.axhip_attn_paged(d_q.ptr, ld, C.byref(struct), o.ptr, ld, lse.ptr, None, lens.ptr, 1, 1, heads, 1, n, 0.1, None))
        assert hip.last_kernel() == "paged_few_ranges", hip.last_kernel()
        w = paged_attention(q[:1], kk, vv, np.ones(n, bool), 0.1)
        within(o.numpy()[:1], w, "o")
    finally:
        hip.sync()
        for p in at.values():
            L.axhip_free(p)


@pytest.mark.parametrize("seed", range(48))
def test_drawn(hip, seed):
    """Any types, heads, pages, rules, counts and holes together, where tiles take the long sequences."""
    rng = np.random.default_rng(3000 + seed)
    kind, heads, G, dk, page_rows = int(rng.integers(3)), int(rng.integers(1, 5)), int(rng.integers(1, 20)), 4 * int(rng.integers(1, 33)), 1 << int(rng.integers(0, 9))
    most = int(rng.choice([33, 70, 150, 400]))
    most = max(most, 64 // G + 1, 33 // G + 1)
    new = np.concatenate([[most], rng.integers(0, most // 2 + 1, int(rng.integers(1, 4)))])
    new = np.concatenate([new, np.zeros(2 * (new.sum() // most) + 1, int)])       # 2 T < B Sq
    rng.shuffle(new)
    lens = np.where(new > 0, np.maximum(new + rng.integers(-2, int(rng.choice([40, 300, 1500])), len(new)), 0), 0)
    rules = {}
    if rng.random() < 0.5:
        rules.update(window=int(rng.choice([1, 3, 31, 32, 33, 64, 100, 257, 1100])), sinks=int(rng.choice([0, 1, 4, 32, 33, 130])))
    if rng.random() < 0.3:
        rules.update(cap=float(rng.choice([0.5, 5.0, 50.0])))
    holes = [(b, int(rng.integers(0, max(1, -(-int(lens[b]) // page_rows))))) for b in range(len(new)) if lens[b] and rng.random() < 0.3]
    say("tiles drawn", seed, kind, heads, G, dk, page_rows, new.tolist(), lens.tolist(), rules, holes)
    check(hip, kind, heads, G, dk, page_rows, new.tolist(), lens.tolist(), rules, bool(rng.random() < 0.3), holes, seed, pitch=4 * int(rng.integers(0, 3)), behind=int(rng.integers(0, 3)))
    assert hip.last_kernel().startswith("paged_tiles"), hip.last_kernel()
