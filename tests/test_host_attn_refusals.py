"""What the entry points of rotation, head norms and attention under score rules refuse and what they launch, on the host, without a GPU."""
import pytest

from test_host_runtime import run, stub  # noqa: F401  (stub is a fixture)

ROPE = """
hip.check(L.axhip_init())
def rope(rows=8, H=2, dk=64, rot=32, x=A, y=D, ldx=128, ldy=128, pos=B, freq=1 << 48, layout=0, back=0):
    return L.axhip_rope_rows(x, ldx, y, ldy, pos, freq, rows, H, dk, rot, 1.0, layout, back)
def norm(rows=8, H=2, Hk=1, dk=64, rot=32, x=A, y=D, ldx=256, ldy=192, eps=1e-6, pos=B, freq=1 << 48, layout=0):
    return L.axhip_qk_norm_rope_fwd(x, ldx, y, ldy, None, None, None, eps, pos, freq, rows, H, Hk, dk, rot, 1.0, layout)
def grad(rows=8, H=2, Hk=1, dk=64, rot=32, dy=1 << 49, x=A, inv=1 << 50, dx=D, ld=192, ldx=256, lddx=192, dgq=1 << 51, dgk=1 << 52, pos=B, freq=1 << 48, layout=0):
    return L.axhip_qk_norm_rope_bwd(dy, ld, x, ldx, inv, dx, lddx, None, None, dgq, dgk, pos, freq, rows, H, Hk, dk, rot, 1.0, layout)
"""


def test_rows_of_heads_refuse(stub):  # noqa: F811
    run(stub, ROPE + """
for f in (rope, norm, grad):
    assert f(rot=31) == 3 and f(rot=66) == 3 and f(rot=-2) == 3 and f(dk=0, rot=0) == 3 and f(dk=4098, rot=0) == 3 and f(layout=2) == 3 and f(rows=-1) == 3
    assert f(H=-1) == 3 and f(pos=None) == 1 and f(freq=None) == 1 and f(x=None) == 1 and f(ldx=100) == 3
    assert f(rows=1 << 41) == 3
assert rope(y=None) == 1 and rope(ldy=127) == 3 and rope(y=A, ldy=132) == 3
assert norm(y=None) == 1 and norm(ldy=191) == 3 and norm(eps=-1.0) == 3 and norm(eps=float("nan")) == 3 and norm(y=A) == 3
assert grad(dy=None) == 1 and grad(inv=None) == 1 and grad(dx=None) == 1 and grad(lddx=191) == 3 and grad(ld=191) == 3 and grad(dx=1 << 49, lddx=196) == 3
assert len(launched()) == 0
assert rope(rows=0) == 0 and rope(H=0) == 0 and norm(rows=0) == 0 and norm(H=0, Hk=0) == 0 and len(launched()) == 0
assert rope(rot=0, pos=None, freq=None) == 0 and len(launched()) == 1
assert grad(rows=0) == 0 and [b"fill" in x.kernel for x in launched()[1:]] == [True, True]
""")


def test_frequencies_refuse(stub):  # noqa: F811
    run(stub, ROPE + """
f = lambda freq=A, rot=64, theta=1e4, scaling=0, factor=1.0, slow=1.0, fast=32.0, trained=2048: L.axhip_rope_frequencies(freq, rot, theta, scaling, factor, slow, fast, trained)
nan, inf = float("nan"), float("inf")
assert f() == 0 and f(rot=0) == 0 and f(rot=4096) == 0
assert f(freq=None) == 1
for bad in (dict(rot=63), dict(rot=-2), dict(rot=4098), dict(theta=0.0), dict(theta=nan), dict(theta=inf), dict(scaling=4), dict(scaling=-1), dict(scaling=1, factor=0.5),
            dict(scaling=2, factor=nan), dict(scaling=3, slow=-1.0), dict(scaling=3, slow=32.0), dict(scaling=3, fast=inf), dict(scaling=3, trained=0)):
    assert f(**bad) == 3, bad
""")


@pytest.mark.parametrize("rows,H,dk,rot", [(1, 1, 8, 8), (1 << 24, 2, 64, 64), (1 << 26, 3, 12, 6), (3, 1 << 18, 64, 64), (1 << 39, 1, 4, 2)])
def test_rows_of_heads_launch(stub, rows, H, dk, rot):  # noqa: F811
    """Any count of rows and heads is a grid that a launch may have."""
    run(stub, ROPE + """
rows, H, dk, rot = %r
assert rope(rows, H, dk, rot, ldx=H * dk, ldy=H * dk) == 0 and norm(rows, H, 1, dk, rot, ldx=(H + 1) * dk, ldy=(H + 1) * dk) == 0
assert grad(rows, H, 1, dk, rot, ld=(H + 1) * dk, ldx=(H + 1) * dk, lddx=(H + 1) * dk) == 0
assert len(launched()) == 4 and b"gamma_sums" in launched()[3].kernel
""" % ((rows, H, dk, rot),))


ATTN = """
from axiom_amd.hip import AttnRules
hip.check(L.axhip_init())
P = [1 << n for n in range(45, 57)]
def fwd(t=None, B=2, H=4, Hkv=2, Sq=16, Sk=32, dk=64, ldq=256, ldk=128, ldv=128, ldo=256, kv_rows=32, rules=None):
    q, k, v, o = t or P[:4]
    return L.axhip_attn_fwd(q, ldq, k, ldk, v, ldv, kv_rows, o, ldo, P[4], B, H, Hkv, Sq, Sk, dk, 0.125, C.byref(rules) if rules else None)
def bwd(t=None, B=2, H=4, Hkv=2, Sq=16, Sk=32, dk=64, ldq=256, ldk=128, ldv=128, ldo=256, kv_rows=32, rules=None, lse=P[4], do=P[5], d=P[6:9], ldd=(256, 256, 128, 128)):
    q, k, v, o = t or P[:4]
    return L.axhip_attn_bwd(q, ldq, k, ldk, v, ldv, kv_rows, o, ldo, lse, do, ldd[0], d[0], ldd[1], d[1], ldd[2], d[2], ldd[3], B, H, Hkv, Sq, Sk, dk, 0.125,
                            C.byref(rules) if rules else None)
"""


def test_attention_refuses(stub):  # noqa: F811
    run(stub, ATTN + """
nan, inf = float("nan"), float("inf")
for f in (fwd, bwd):
    for i in range(4):
        for bad, code in ((None, 1), (P[i] + 4, 3)):
            t = P[:4]
            t[i] = bad
            assert f(t) == code
    for dk in (0, 2, 6, 132, 63):
        assert f(dk=dk, ldq=1024, ldk=1024, ldv=1024, ldo=1024) == 10, dk
    for bad in (dict(B=-1), dict(H=0), dict(Hkv=0), dict(H=3), dict(Sq=-1), dict(Sk=-1), dict(Sq=(1 << 24) + 1), dict(Sk=(1 << 24) + 1, kv_rows=1 << 25), dict(kv_rows=31),
                dict(ldq=255), dict(ldq=258), dict(ldk=124), dict(ldv=124), dict(ldo=252), dict(ldk=(1 << 22) + 4), dict(B=1 << 23), dict(kv_rows=1 << 41),
                dict(rules=AttnRules(cap=-1.0)), dict(rules=AttnRules(cap=nan)), dict(rules=AttnRules(cap=inf)), dict(rules=AttnRules(cap=1e-40)), dict(rules=AttnRules(prefix=P[9]))):
        assert f(**bad) == 3, bad
    assert f(rules=AttnRules(doc_q=P[9])) == 1 and f(rules=AttnRules(doc_k=P[9])) == 1
assert bwd(lse=None) == 1 and bwd(do=None) == 1 and bwd(do=P[5] + 8) == 3
for i in range(3):
    assert bwd(d=[None if n == i else P[6 + n] for n in range(3)]) == 1 and bwd(d=[P[6 + n] + 4 * (n == i) for n in range(3)]) == 3
    assert bwd(ldd=[124 if n == i + 1 else 256 for n in range(4)]) == 3
assert len(launched()) == 0
assert fwd(B=0) == 0 and fwd(Sq=0) == 0 and bwd(B=0) == 0 and len(launched()) == 0
assert fwd() == 0 and len(launched()) > 0
""")


@pytest.mark.parametrize("B,H,Hkv,Sq,Sk,dk", [(1, 1, 1, 1, 1, 4), (1, 1, 1, 1 << 24, 1 << 24, 128), (8388607, 8, 8, 1, 3, 64), (3, 65536, 1, 100, 1000, 32), (64, 64, 8, 1, 1 << 20, 128),
                                              (2, 8, 2, 1, 0, 64), (1 << 16, 1 << 10, 1 << 10, 129, 65, 96)])
def test_attention_launches(stub, B, H, Hkv, Sq, Sk, dk):  # noqa: F811
    """Any extent is made of launches that the runtime takes."""
    run(stub, ATTN + """
B, H, Hkv, Sq, Sk, dk = %r
ld = dict(ldq=min(H * dk, 1 << 22), ldk=Hkv * dk, ldv=Hkv * dk, ldo=min(H * dk, 1 << 22))
if H * dk <= 1 << 22:
    for rules in (None, AttnRules(cap=30.0, causal=1), AttnRules(doc_q=P[9], doc_k=P[10])):
        hip.check(fwd(None, B, H, Hkv, Sq, Sk, dk, kv_rows=Sk, rules=rules, **ld))
        hip.check(bwd(None, B, H, Hkv, Sq, Sk, dk, kv_rows=Sk, rules=rules, ldd=(H * dk, H * dk, Hkv * dk, Hkv * dk), **ld))
    assert len(launched()) >= (9 if Sk else 6)
""" % ((B, H, Hkv, Sq, Sk, dk),))


def test_which_caps_and_scales_are_taken(stub):  # noqa: F811
    """Any cap whose reciprocal is a float, the largest ones too, whatever the scale; and scales that are floats in log2 units."""
    run(stub, ATTN + """
def with_scale(scale, cap):
    rules = AttnRules(cap=cap)
    shape = (2, 4, 2, 16, 32, 64, scale, C.byref(rules))
    a = L.axhip_attn_fwd(P[0], 256, P[1], 128, P[2], 128, 32, P[3], 256, P[4], *shape)
    b = L.axhip_attn_bwd(P[0], 256, P[1], 128, P[2], 128, 32, P[3], 256, P[4], P[5], 256, P[6], 256, P[7], 128, P[8], 128, *shape)
    assert a == b
    return a
biggest = 3.4028234663852886e38
for cap in (0.0, 2.2e-39, 1e-20, 1.0, 1e33, 1e38, biggest):
    for scale in (1e-30, 0.125, 1e30):
        assert with_scale(scale, cap) == 0, (scale, cap)
for cap in (1e-45, 2e-39, float("inf"), float("nan"), -1.0):
    for scale in (1e-30, 0.125):
        assert with_scale(scale, cap) == 3, (scale, cap)
assert with_scale(2.3e38, 0.0) == 0 and with_scale(2.4e38, 0.0) == 3 and with_scale(-biggest, 30.0) == 3
""")


@pytest.mark.parametrize("B,H,Hkv", [(4, 1 << 62, 1 << 62), (4, 1 << 62, 1), (1, (1 << 62) + 4, 1), (2, 1 << 61, 1 << 61), (1, (1 << 20) + 1, 1)])
def test_head_counts_past_64_bits(stub, B, H, Hkv):  # noqa: F811
    """Heads times their size, or times sequences, that come out small in 64 bits."""
    run(stub, ATTN + """
B, H, Hkv = %r
ld = dict(ldq=1 << 22, ldk=1 << 22, ldv=1 << 22, ldo=1 << 22)
assert fwd(None, B, H, Hkv, 1, 3, 4, kv_rows=3, **ld) == 3
assert bwd(None, B, H, Hkv, 1, 3, 4, kv_rows=3, ldd=(1 << 22,) * 4, **ld) == 3
assert len(launched()) == 0
""" % ((B, H, Hkv),))
