"""What the entry points of the paged cache and the attention over it refuse and what they launch, on the host, without a GPU."""
import pytest

from test_host_runtime import run, stub  # noqa: F401  (stub is a fixture)

PAGED = """
from axiom_amd.hip import KvCache, KvRules
hip.check(L.axhip_init())
P = [1 << n for n in range(45, 57)]
def cache(type=1, page_rows=16, pages=100, heads=2, dk=64, k=P[0], v=P[1], k_scale=P[2], v_scale=P[3], table=P[4], table_ld=8):
    return C.byref(KvCache(type=type, page_rows=page_rows, pages=pages, heads=heads, dk=dk, k=k, v=v, k_scale=k_scale, v_scale=v_scale, table=table, table_ld=table_ld))
def rows(f, c=None, K=P[5], ldk=128, V=P[6], ldv=128, first=P[7], lens=P[8], B=3, T=20, Sq=10, **more):
    return f(cache(**more) if c is None else c, K, ldk, V, ldv, first, lens, B, T, Sq)
def write(*a, **more): return rows(L.axhip_kv_write, *a, **more)
def read(*a, **more): return rows(L.axhip_kv_read, *a, **more)
def attend(c=None, Q=P[5], ldq=256, O=P[6], ldo=256, lse=P[9], first=P[7], lens=P[8], B=3, T=20, H=4, Sq=10, Sk=128, scale=0.125, rules=None, **more):
    return L.axhip_attn_paged(Q, ldq, cache(**more) if c is None else c, O, ldo, lse, first, lens, B, T, H, Sq, Sk, scale, C.byref(rules) if rules else None)
"""


def test_refusals(stub):  # noqa: F811
    run(stub, PAGED + """
nan, inf = float("nan"), float("inf")
for f in (write, read, attend):
    for dk in (0, 2, 6, 132, 63, -4, 1 << 62):
        assert f(dk=dk) == 10, dk
    for bad in (dict(type=-1), dict(type=3), dict(page_rows=0), dict(page_rows=3), dict(page_rows=-16), dict(page_rows=1 << 17), dict(heads=0), dict(heads=-2), dict(heads=(1 << 20) + 1),
                dict(pages=-1), dict(pages=1 << 31), dict(pages=1 << 30, heads=1 << 10), dict(table_ld=-1), dict(table_ld=1 << 41), dict(B=-1), dict(B=1 << 23), dict(T=-1), dict(T=(1 << 24) + 1), dict(Sq=-1),
                dict(Sq=(1 << 24) + 1), dict(first=None), dict(k=P[0] + 8), dict(v=P[1] + 4), dict(k_scale=P[2] + 4), dict(v_scale=P[3] + 12)):
        assert f(**bad) == 3, bad
    for bad in (dict(k=None), dict(v=None), dict(k_scale=None), dict(v_scale=None), dict(table=None), dict(lens=None), dict(c=C.POINTER(KvCache)())):
        assert f(**bad) == 1, bad
for f in (write, read):
    for bad in (dict(ldk=127), dict(ldv=124), dict(ldk=130), dict(ldv=(1 << 22) + 4), dict(K=P[5] + 4), dict(V=P[6] + 8)):
        assert f(**bad) == 3, bad
    assert f(K=None) == 1 and f(V=None) == 1
for bad in (dict(ldq=255), dict(ldq=258), dict(ldo=252), dict(ldo=(1 << 22) + 4), dict(Q=P[5] + 4), dict(O=P[6] + 8), dict(H=0), dict(H=3), dict(H=-2), dict(H=(1 << 20) + 2), dict(H=1 << 62),
            dict(Sk=-1), dict(Sk=(1 << 24) + 1), dict(B=1 << 22, H=1 << 10, ldq=1 << 16, ldo=1 << 16), dict(rules=KvRules(cap=-1.0)), dict(rules=KvRules(cap=nan)), dict(rules=KvRules(cap=inf)),
            dict(rules=KvRules(cap=1e-40)), dict(scale=2.4e38), dict(rules=KvRules(window=-1)), dict(rules=KvRules(sinks=-1))):
    assert attend(**bad) == 3, bad
assert attend(Q=None) == 1 and attend(O=None) == 1
assert len(launched()) == 0
for f in (write, read, attend):
    assert f(B=0) == 0 and f(T=0) == 0 and f(Sq=0) == 0 and f(first=None, B=2, T=0, Sq=0) == 0
    assert f(B=0, T=0, lens=None, table=None, k=None) == 0
assert len(launched()) == 0
assert write() == 0 and read() == 0 and attend() == 0 and attend(lse=None, rules=KvRules(window=(1 << 31) - 1, sinks=(1 << 31) - 1)) == 0 and attend(first=None, B=2) == 0
assert len(launched()) > 0
""")


def test_row_bytes(stub):  # noqa: F811
    run(stub, """
f = L.axhip_kv_row_bytes
assert [f(t, 128) for t in (0, 1, 2)] == [256, 128, 64] and [f(t, 80) for t in (0, 1, 2)] == [160, 80, 48] and [f(t, 4) for t in (0, 1, 2)] == [16, 16, 16]
assert all(f(t, dk) == 0 for t, dk in ((-1, 64), (3, 64), (0, 0), (0, 132), (1, 30), (2, -4)))
""")


def test_which_launches(stub):  # noqa: F811
    """Few rows of every sequence, or not many in all: one launch; many of every one: tiles alone; unlike ones: both."""
    run(stub, PAGED + """
def names(**more):
    before = stub.stub_launches()
    assert attend(**more) == 0
    return [("few" if b"paged_few" in x.kernel else "tiles" if b"paged_tiles" in x.kernel else "join" if b"paged_join" in x.kernel else "?") for x in launched()[before:]]
assert names(Sq=1, T=3, first=None) == ["few"] and names(Sq=4, T=9) == ["few"] and names(Sq=16, T=9) == ["few"]
assert names(Sq=100, T=300, first=None, Sk=100) == ["few"] and names(Sq=100, T=100, B=1) == ["few"]
assert names(Sq=4000, T=12000, first=None) == ["tiles"] and names(Sq=8000, T=8000, B=1) == ["tiles"]
assert names(Sq=100, T=120) == ["few", "tiles"] and names(Sq=100, T=150) == ["few"]
assert names(Sq=4000, T=12000) == ["tiles"] and names(Sq=4000, T=11999) == ["few", "tiles"]
assert names(Sq=2000, T=2000, B=1, Sk=100000, table_ld=10000) == ["tiles", "join"]
""")


@pytest.mark.parametrize("B,T,H,heads,Sq,Sk,dk,kind,uniform", [(1, 1, 1, 1, 1, 0, 4, 0, False), (8388607, 1 << 24, 1, 1, 1 << 24, 1 << 24, 128, 1, False), (1, 1 << 24, 8, 1, 1 << 24, 1 << 24, 128, 2, True),
                                                               (2047, 2047, 1 << 20, 1 << 20, 1, 100, 4, 1, True), (1 << 20, 1 << 20, 8, 8, 1, 1 << 20, 64, 2, True),
                                                               (1, 3, 1 << 15, 1, 3, 1 << 24, 128, 1, True), (100, 1 << 20, 64, 1, 1 << 20, 1 << 20, 32, 0, False)])
def test_launches(stub, B, T, H, heads, Sq, Sk, dk, kind, uniform):  # noqa: F811
    """Any extent is made of launches that the runtime takes, or refused."""
    run(stub, PAGED + """
B, T, H, heads, Sq, Sk, dk, kind, uniform = %r
stub.stub_set_free(C.c_size_t(200 << 30))
first = None if uniform else P[7]
more = dict(type=kind, heads=heads, dk=dk, pages=1 << 12, table_ld=1 << 20, B=B, T=T, Sq=Sq, first=first)
hip.check(write(ldk=heads * dk, ldv=heads * dk, **more))
hip.check(read(ldk=heads * dk, ldv=heads * dk, **more))
for rules in (None, KvRules(window=1000, sinks=4, cap=10.0)):
    hip.check(attend(ldq=H * dk, ldo=H * dk, H=H, Sk=Sk, rules=rules, **more))
for x in launched():
    assert 0 < x.grid[0] < 1 << 31 and x.grid[0] * x.block[0] < 1 << 32 and x.block[0] <= 1024 and x.shared <= 160 * 1024, (x.kernel, list(x.grid), list(x.block))
""" % ((B, T, H, heads, Sq, Sk, dk, kind, uniform),))


@pytest.mark.parametrize("B,T,H,heads,Sq,Sk,dk", [(2000, 6000, 8, 8, 2000, 4000, 128), (300, 3000, 32, 8, 1000, 100000, 128), (24, 2217, 16, 4, 600, 3000, 80), (1, 64, 32, 8, 64, 1 << 20, 128),
                                                  (128, 128, 8, 1, 1, 1 << 20, 128), (8388607, 1 << 20, 8, 1, 1000, 100000, 64)])
def test_what_ranges_keep(stub, B, T, H, heads, Sq, Sk, dk):  # noqa: F811
    """The shared workspace holds what ranges of keys leave, and stays at 256 MiB or what it started with, however many sequences a call has."""
    run(stub, PAGED + """
B, T, H, heads, Sq, Sk, dk = %r
hip.check(attend(ldq=H * dk, ldo=H * dk, H=H, Sk=Sk, heads=heads, dk=dk, pages=1 << 12, table_ld=1 << 20, B=B, T=T, Sq=Sq))
have = C.c_size_t()
hip.check(L.axhip_workspace_reserve(0, C.byref(have)))
assert have.value <= 256 * MIB, have.value
""" % ((B, T, H, heads, Sq, Sk, dk),))


def test_a_bound_on_rows_is_no_count_of_them(stub):  # noqa: F811
    """Sq is the most rows that a sequence may have, and none has more than there are: callers with a bound of their own launch for the rows that come."""
    run(stub, PAGED + """
def shapes(**more):
    before = stub.stub_launches()
    assert attend(**more) == 0
    return [(x.kernel, list(x.grid), list(x.block)) for x in launched()[before:]]
for B, T in ((1, 1), (1, 3), (8, 8), (3, 10), (1, 40), (1, 300)):
    for heads, H, dk in ((2, 4, 64), (8, 64, 128), (1, 1, 32)):
        for rules in (None, KvRules(window=30, sinks=4)):
            more = dict(B=B, T=T, heads=heads, H=H, dk=dk, ldq=H * dk, ldo=H * dk, rules=rules)
            want = shapes(Sq=T, **more)
            for Sq in (T + 1, 4096, 1 << 24):
                assert shapes(Sq=Sq, **more) == want, (B, T, heads, Sq)
assert all(b"paged_few" in x[0] for T in (1, 8) for x in shapes(B=T, T=T, Sq=4096, heads=8, H=64, dk=128, ldq=8192, ldo=8192)[:1])
assert len(shapes(B=1, T=1, Sq=4096, heads=8, H=64, dk=128, ldq=8192, ldo=8192)) == 1
# eight single tokens with room for eight each: as many ranges of keys, a workgroup for each of the four sets of rows that each could have
one, more = (shapes(B=8, T=8, Sq=Sq, heads=8, H=64, dk=128, ldq=8192, ldo=8192, Sk=4096, table_ld=256)[0] for Sq in (1, 4096))
assert one[1][0] > 8 * 8 and more[1][0] == 4 * one[1][0] and one[2] == more[2], (one, more)
""")


@pytest.mark.parametrize("B,T,H,heads,dk", [(1000, 64, 1, 1, 128), (8, 8, 64, 8, 128), (100000, 16, 4, 1, 128), (3, 60, 8, 8, 64), (2, 500, 8, 8, 128), (300, 3, 64, 4, 64)])
@pytest.mark.parametrize("Sq", [0, 1 << 24])
def test_what_ranges_of_few_rows_keep(stub, B, T, H, heads, dk, Sq):  # noqa: F811
    """... and where any sequence may have all of the rows, ranges are counted by the rows that there are, within what the workspace and the counters start with."""
    run(stub, PAGED + """
B, T, H, heads, dk, Sq = %r
hip.check(attend(ldq=H * dk, ldo=H * dk, H=H, Sk=100000, heads=heads, dk=dk, pages=1 << 12, table_ld=1 << 20, B=B, T=T, Sq=Sq or T))
have = C.c_size_t()
hip.check(L.axhip_workspace_reserve(0, C.byref(have)))
assert have.value == 160 * MIB and all(x.grid[0] < 1 << 22 for x in launched()), have.value
""" % ((B, T, H, heads, dk, Sq),))


def test_as_many_workgroups_a_sequence_as_a_launch_holds(stub):  # noqa: F811
    """2^20 heads of four sets of rows each: a launch a sequence."""
    run(stub, PAGED + """
hip.check(attend(ldq=1 << 22, ldo=1 << 22, H=1 << 20, heads=1 << 20, dk=4, pages=1 << 12, table_ld=1 << 20, Sk=100, B=3, T=192, Sq=64, first=None))
assert [x.grid[0] for x in launched()] == [1 << 22] * 3 and all(b"paged_few" in x.kernel for x in launched())
""")


@pytest.mark.parametrize("B,n,H,heads,dk,Sk", [(1, 64, 32, 8, 128, 8192), (2, 150, 16, 4, 64, 30000), (1, 300, 8, 8, 80, 20000), (3, 257, 4, 1, 128, 50000)])
def test_ranges_of_equal_counts_however_they_are_given(stub, B, n, H, heads, dk, Sk):  # noqa: F811
    """Sequences of n rows each, with `first` and without: tiles have as many ranges of keys."""
    run(stub, PAGED + """
B, n, H, heads, dk, Sk = %r
G = H // heads
BQ = 256 if G * n > 128 else 128
def splits(first, slots, Sq=n):
    before = stub.stub_launches()
    hip.check(attend(ldq=H * dk, ldo=H * dk, H=H, Sk=Sk, heads=heads, dk=dk, pages=1 << 12, table_ld=1 << 12, B=B, T=B * n, Sq=Sq, first=first))
    tiles, join = launched()[before:]
    assert b"paged_tiles" in tiles.kernel and b"paged_join" in join.kernel and tiles.grid[0] %% (slots * heads) == 0
    return tiles.grid[0] // (slots * heads)
want = splits(None, B * -(-G * n // BQ))
assert want > 1 and splits(P[7], G * B * n // BQ + B) == want, want
if B == 1:
    assert splits(P[7], G * n // BQ + 1, Sq=4096) == want
""" % ((B, n, H, heads, dk, Sk),))
