"""Attention under score rules on the GPU, forward and backward, against 64 bits (attn_oracle.py, which derives the bounds)."""
import ctypes as C

import numpy as np
import pytest

from attn_oracle import Rules, attention
from axiom_amd.hip import AttnRules

pytestmark = pytest.mark.gpu


def say(*a):
    print(*a, flush=True)


def device_rules(hip, rules):
    """(the struct, the arrays that it points to)"""
    held = {n: hip.array(np.asarray(getattr(rules, n), np.float32 if n == "slopes" else np.int32)) for n in Rules.ARRAYS if getattr(rules, n) is not None}
    return AttnRules(cap=rules.cap, causal=rules.causal, **{n: x.ptr for n, x in held.items()}), held


def padded(hip, x, ld, rows, garbage):
    """x [B, S, heads, dk] as rows of pitch ld, `rows` of them for each sequence, garbage around"""
    B, S = x.shape[:2]
    full = np.full((B, rows, ld), garbage, np.float32)
    full[:, :S, :x.shape[2] * x.shape[3]] = x.reshape(B, S, x.shape[2] * x.shape[3])
    return hip.array(full)


def taken(d, like):
    """The values of `like`'s shape out of padded rows, and the rest"""
    B, S, h, dk = like.shape
    full = d.numpy()
    out = full[:, :S, :h * dk].reshape(like.shape)
    rest = full.copy()
    rest[:, :S, :h * dk] = 7.0
    return out, rest


def check(hip, q, k, v, scale, rules, d_o=None, pitch=0, more_rows=0, want=None, kernel=None):
    """Runs forward (and backward where d_o is given) on padded rows and holds both to the oracle; returns what came out."""
    B, Sq, H, dk = q.shape
    Sk, Hkv = k.shape[1], k.shape[2]
    r, held = device_rules(hip, rules)
    want = want or attention(q, k, v, scale, rules, d_o)
    ld, ldk, rows = H * dk + pitch, Hkv * dk + pitch, Sk + more_rows
    dq, dk_, dv = padded(hip, q, ld, Sq, np.nan), padded(hip, k, ldk, rows, np.nan), padded(hip, v, ldk, rows, np.nan)
    o, lse = hip.array(np.full((B, Sq, ld), 7, np.float32)), hip.array(np.full((B, H, Sq), 7, np.float32))
    hip.check(hip.L.axhip_attn_fwd(dq.ptr, ld, dk_.ptr, ldk, dv.ptr, ldk, rows, o.ptr, ld, lse.ptr, B, H, Hkv, Sq, Sk, dk, scale, C.byref(r)))
    if kernel:
        assert kernel in hip.last_kernel(), hip.last_kernel()
    got, rest = taken(o, q)
    out = {"o": got, "lse": lse.numpy()}
    assert (rest == 7).all()
    empty = np.isneginf(want["lse"])
    assert np.array_equal(np.isneginf(out["lse"]), empty)
    within(got, want, "o")
    within(np.where(empty, 0, out["lse"]), dict(want, lse=np.where(empty, 0, want["lse"])), "lse")
    if d_o is None:
        return out
    # the gradient from the exact forward pass, rounded
    oin, lin, do = padded(hip, want["o"].astype(np.float32), ld, Sq, np.nan), hip.array(want["lse"].astype(np.float32)), padded(hip, d_o, ld, Sq, np.nan)
    grads = {"dq": hip.array(np.full((B, Sq, ld), 7, np.float32)), "dk": hip.array(np.full((B, rows, ldk), 7, np.float32)), "dv": hip.array(np.full((B, rows, ldk), 7, np.float32))}
    hip.check(hip.L.axhip_attn_bwd(dq.ptr, ld, dk_.ptr, ldk, dv.ptr, ldk, rows, oin.ptr, ld, lin.ptr, do.ptr, ld, grads["dq"].ptr, ld, grads["dk"].ptr, ldk, grads["dv"].ptr, ldk,
                                   B, H, Hkv, Sq, Sk, dk, scale, C.byref(r)))
    for n, x in (("dq", q), ("dk", k), ("dv", v)):
        out[n], rest = taken(grads[n], x)
        assert (rest == 7).all(), n
        within(out[n], want, n)
    return out


def within(got, want, n):
    off, tol = np.abs(got - want[n]), want["tol_" + n]
    bad = ~(off <= tol)
    if bad.any():
        at = np.unravel_index(np.argmax(np.where(bad, np.nan_to_num(off / np.maximum(tol, 1e-300), nan=np.inf), 0)), off.shape)
        pytest.fail("%s: %d of %d out of bounds, the worst at %s: %r, not %r +- %r" % (n, bad.sum(), bad.size, at, got[at], want[n][at], tol[at]))


def draw(seed, B, Sq, Sk, H, Hkv, dk):
    rng = np.random.default_rng(seed)
    q, d_o = (rng.normal(size=(B, Sq, H, dk)).astype(np.float32) for _ in range(2))
    k, v = (rng.normal(size=(B, Sk, Hkv, dk)).astype(np.float32) for _ in range(2))
    return rng, q, k, v, d_o


def documents(rng, B, S, n, pad):
    """n pieces of unlike lengths in any order of ids, then `pad` rows of none"""
    out = np.full((B, S), -1, np.int32)
    for b in range(B):
        cuts = np.sort(rng.integers(0, max(S - pad, 1), n - 1))
        ids = rng.permutation(n)
        out[b, :S - pad] = ids[np.searchsorted(cuts, np.arange(S - pad), side="right")]
    return out


KINDS = ["plain", "causal", "capped", "distance", "prefix", "lens", "documents", "scattered", "everything"]


def rules_of(kind, rng, B, Sq, Sk, H):
    same = Sq == Sk
    lens = rng.integers(0, Sk + 1, B)
    slopes = (2.0 ** -np.arange(1, H + 1)).astype(np.float32)
    if kind == "plain":
        return Rules()
    if kind == "causal":
        return Rules(causal=1)
    if kind == "capped":
        return Rules(causal=1, cap=3.0)
    if kind == "distance":
        return Rules(slopes=slopes, lens=lens)
    if kind == "prefix":
        return Rules(causal=1, prefix=rng.integers(-1, Sk + 2, B), start=None if same else rng.integers(-3, Sk, B))
    if kind == "lens":
        return Rules(causal=1, lens=lens, start=np.maximum(lens - Sq, 0))
    if kind == "documents":
        ids = documents(rng, B, max(Sq, Sk), 3, max(Sq, Sk) // 6)
        return Rules(causal=int(same), doc_q=ids[:, :Sq].copy(), doc_k=ids[:, :Sk].copy())
    if kind == "scattered":                      # ids in no order, some negative
        return Rules(doc_q=rng.integers(-1, 3, (B, Sq)).astype(np.int32), doc_k=rng.integers(-1, 3, (B, Sk)).astype(np.int32))
    ids = documents(rng, B, max(Sq, Sk), 2, 1 if min(Sq, Sk) > 1 else 0)
    return Rules(cap=20.0, causal=1, slopes=slopes, prefix=rng.integers(0, Sk // 2 + 1, B), lens=lens, start=np.maximum(lens - Sq, 0), doc_q=ids[:, :Sq].copy(), doc_k=ids[:, :Sk].copy())


SHAPES = [(1, 1, 1, 1, 1, 4), (2, 1, 7, 4, 2, 64), (1, 33, 33, 2, 1, 32), (2, 64, 64, 2, 2, 64), (1, 65, 65, 3, 3, 20), (1, 130, 130, 4, 2, 128), (2, 97, 97, 2, 1, 80), (1, 5, 200, 4, 1, 96),
          (1, 200, 70, 2, 2, 48), (1, 257, 257, 2, 1, 64), (1, 31, 32, 1, 1, 124), (3, 2, 129, 8, 2, 36), (1, 160, 352, 2, 2, 112)]


@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "x".join(map(str, s)))
@pytest.mark.parametrize("kind", KINDS)
def test_against_64_bits(hip, shape, kind):
    say("attn", shape, kind)
    B, Sq, Sk, H, Hkv, dk = shape
    rng, q, k, v, d_o = draw(sum(shape) + KINDS.index(kind), *shape)
    check(hip, q, k, v, dk ** -0.5, rules_of(kind, rng, B, Sq, Sk, H), d_o, pitch=4 * (dk % 3), more_rows=Sq % 3)


@pytest.mark.parametrize("kind", ["causal", "documents", "everything", "lens"])
@pytest.mark.parametrize("dk", [64, 128])
def test_garbage_where_nobody_looks(hip, kind, dk):
    """NaN, infinities and the largest floats in rows that no query sees, and in queries that see nothing: what zeros there give."""
    say("attn garbage", kind, dk)
    B, S, H, Hkv = 2, 150, 4, 2
    rng, q, k, v, d_o = draw(7, B, S, S, H, Hkv, dk)
    rules = rules_of(kind, rng, B, S, S, H)
    if kind == "causal":
        rules.lens = np.array([100, 0])
    seen = [rules.sees(b, S, S)[0] for b in range(B)]
    outs = []
    for garbage in (0.0, np.nan, np.inf, -3e38):
        for b in range(B):
            k[b, ~seen[b].any(0)] = v[b, ~seen[b].any(0)] = garbage
            q[b, ~seen[b].any(1)] = d_o[b, ~seen[b].any(1)] = garbage
        outs.append(check(hip, q, k, v, 0.1, rules, d_o, want=outs[0]["want"] if outs else None))
        if len(outs) == 1:
            outs[0] = dict(outs[0], want=attention(q, k, v, 0.1, rules, d_o))
    for out in outs[1:]:
        for n in ("o", "lse", "dq", "dk", "dv"):
            scale = np.abs(outs[0][n][np.isfinite(outs[0][n])]).max()
            fine = np.isfinite(outs[0][n])
            assert np.array_equal(fine, np.isfinite(out[n])) and np.abs(out[n][fine] - outs[0][n][fine]).max() <= 1e-4 * scale


@pytest.mark.parametrize("dk", [32, 64, 128])
def test_a_value_that_only_some_see(hip, dk):
    """A NaN key at position 100 and an infinite value at 120 under the causal mask, and in a document of its own: rows before them and other documents
    are as without them, rows that see them are not finite; so for gradients."""
    say("attn nan", dk)
    B, S, H = 2, 200, 2
    rng, q, k, v, d_o = draw(8, B, S, S, H, H, dk)
    ids = np.zeros((B, S), np.int32)
    ids[1, 60:130] = 1
    rules = Rules(causal=1, doc_q=ids, doc_k=ids)
    clean = check(hip, q, k, v, 0.1, rules, d_o)
    k[0, 100, 0, 3] = np.nan
    v[1, 120, 1, 5] = np.inf
    r, held = device_rules(hip, rules)
    dq, dk_, dv, do, o, lse = hip.array(q), hip.array(k), hip.array(v), hip.array(d_o), hip.empty(q.shape), hip.empty((B, H, S))
    grads = [hip.empty(x.shape) for x in (q, k, v)]
    ld = H * dk
    hip.check(hip.L.axhip_attn_fwd(dq.ptr, ld, dk_.ptr, ld, dv.ptr, ld, S, o.ptr, ld, lse.ptr, B, H, H, S, S, dk, 0.1, C.byref(r)))
    hip.check(hip.L.axhip_attn_bwd(dq.ptr, ld, dk_.ptr, ld, dv.ptr, ld, S, o.ptr, ld, lse.ptr, do.ptr, ld, *sum(([g.ptr, ld] for g in grads), []), B, H, H, S, S, dk, 0.1, C.byref(r)))
    got = dict(zip(("o", "dq", "dk", "dv"), [o.numpy()] + [g.numpy() for g in grads]))
    hit = np.zeros((B, S, H), bool)
    hit[0, 100:, 0] = True
    hit[1, 120:130, 1] = True
    for n in ("o", "dq"):
        near = np.abs(got[n] - clean[n]) <= 1e-4 * np.abs(clean[n]).max()
        assert near[~hit].all(), n
        assert (~np.isfinite(got[n][hit])).any(-1).all(), n
    # keys before a hit row share it: their gradients are not finite; those after it, of other heads and of other documents are as before
    for n in ("dk", "dv"):
        clear = np.ones((B, S, H), bool)
        clear[0, :, 0] = False
        clear[1, 60:130, 1] = False
        assert (np.abs(got[n] - clean[n]) <= 1e-4 * np.abs(clean[n]).max())[clear].all(), n


@pytest.mark.parametrize("dk", [64, 128])
@pytest.mark.parametrize("size", [1e-30, 1e-12, 1e6, 1e15])
def test_large_and_small_values(hip, dk, size):
    """Values and gradients of any size, scores of ordinary size from large queries and small keys."""
    say("attn sizes", dk, size)
    rng, q, k, v, d_o = draw(9, 1, 100, 100, 2, 1, dk)
    v[0, 40:60] *= np.float32(1e-3)
    check(hip, q * np.float32(size), k / np.float32(size), v * np.float32(size), dk ** -0.5, Rules(causal=1, cap=10.0), d_o * np.float32(1 / size))


def test_scores_far_apart(hip):
    """Scores of hundreds: probabilities of one and of nothing."""
    rng, q, k, v, d_o = draw(10, 1, 150, 150, 2, 2, 64)
    check(hip, q * np.float32(30), k, v, 1.0, Rules(causal=1), d_o)
    check(hip, q * np.float32(30), k, v, 1.0, Rules(causal=1, cap=50.0), d_o)


@pytest.mark.parametrize("B,new,Sk,H,Hkv,dk", [(1, 1, 1, 4, 1, 64), (1, 1, 500, 16, 4, 64), (3, 1, 1000, 8, 8, 128), (2, 5, 777, 8, 2, 80), (1, 3, 5000, 2, 1, 32), (5, 2, 64, 32, 1, 96),
                                               (2, 1, 3000, 64, 1, 128), (70, 1, 130, 8, 2, 64), (1, 1, 20000, 4, 4, 64)])
@pytest.mark.parametrize("kind", ["lens", "plain", "bias", "documents"])
def test_tokens_over_a_cache(hip, B, new, Sk, H, Hkv, dk, kind):
    say("attn cache", B, new, Sk, H, Hkv, dk, kind)
    rng, q, k, v, _ = draw(B + Sk + dk, B, new, Sk, H, Hkv, dk)
    lens = rng.integers(min(new, Sk), Sk + 1, B)
    lens[0] = Sk
    slopes = (2.0 ** -rng.uniform(1, 8, H)).astype(np.float32)
    rules = {"plain": Rules(), "lens": Rules(causal=1, lens=lens, start=lens - new, cap=30.0), "bias": Rules(causal=1, lens=lens, start=lens - new, slopes=slopes)}.get(kind)
    if kind == "documents":
        ids = documents(rng, B, Sk, 3, 0)
        rules = Rules(doc_q=ids[:, -1:].repeat(new, 1).copy(), doc_k=ids, causal=1, lens=lens, start=lens - new)
    check(hip, q, k, v, dk ** -0.5, rules, pitch=8, more_rows=3)


def test_the_same_bits_twice(hip):
    """Forward, backward and over a cache, with another call between."""
    rng, q, k, v, d_o = draw(11, 2, 300, 300, 4, 2, 64)
    rules = rules_of("everything", rng, 2, 300, 300, 4)
    rules.lens = np.array([300, 170])
    want = attention(q, k, v, 0.125, rules, d_o)
    a = check(hip, q, k, v, 0.125, rules, d_o, want=want)
    c1 = check(hip, q[:, :1], k, v, 0.125, Rules())
    b = check(hip, q, k, v, 0.125, rules, d_o, want=want)
    c2 = check(hip, q[:, :1], k, v, 0.125, Rules())
    assert all(np.array_equal(a[n], b[n]) for n in ("o", "lse", "dq", "dk", "dv")) and all(np.array_equal(c1[n], c2[n]) for n in ("o", "lse"))


def test_no_keys_and_no_log_sum_exp(hip):
    rng, q, k, v, d_o = draw(12, 2, 3, 5, 2, 1, 8)
    out = check(hip, q, k[:, :0], v[:, :0], 0.5, Rules(), d_o, more_rows=1)
    assert (out["o"] == 0).all() and (out["dq"] == 0).all()
    dq, dk_, dv, o = hip.array(q), hip.array(k), hip.array(v), hip.empty(q.shape)
    hip.check(hip.L.axhip_attn_fwd(dq.ptr, 16, dk_.ptr, 8, dv.ptr, 8, 5, o.ptr, 16, None, 2, 2, 1, 3, 5, 8, 0.5, None))
    want = attention(q, k, v, 0.5, Rules())
    assert (np.abs(o.numpy() - want["o"]) <= want["tol_o"]).all()
    # no queries: zero gradients of keys
    g = [hip.array(np.full(x.shape, 9, np.float32)) for x in (k, v)]
    hip.check(hip.L.axhip_attn_bwd(dq.ptr, 16, dk_.ptr, 8, dv.ptr, 8, 5, o.ptr, 16, o.ptr, dq.ptr, 16, o.ptr, 16, g[0].ptr, 8, g[1].ptr, 8, 2, 2, 1, 0, 5, 8, 0.5, None))
    assert all((x.numpy() == 0).all() for x in g)


def test_layer_between_its_projections(hip):
    """A run of them together on the fused projection of a batch with a short sequence: norm and rotation, attention, and back to the projection's gradient,
    against 64 bits all the way; then the last token again over the keys as a cache, which gives the last row of the prompt."""
    from attn_oracle import inv_rms, norm_grad, rotate
    B, S, H, Hkv, dk, rot = 2, 150, 4, 2, 64, 32
    rng = np.random.default_rng(13)
    n, ld, ldn = H + 2 * Hkv, (H + 2 * Hkv) * dk, (H + Hkv) * dk
    qkv, d_o = rng.normal(size=(B * S, n, dk)).astype(np.float32), rng.normal(size=(B, S, H, dk)).astype(np.float32)
    pos, gq, gk = np.tile(np.arange(S), B).astype(np.int32), rng.normal(1, 0.2, dk).astype(np.float32), rng.normal(1, 0.2, dk).astype(np.float32)
    lens = np.array([S, 90], np.int32)
    rules = Rules(cap=30.0, causal=1, lens=lens)
    r, held = device_rules(hip, rules)
    x, dpos, dgq, dgk, freq = hip.array(qkv), hip.array(pos), hip.array(gq), hip.array(gk), hip.empty((rot // 2,))
    y, inv, o, lse = hip.empty((B * S, ldn)), hip.empty((B * S, H + Hkv)), hip.empty((B * S, H * dk)), hip.empty((B, H, S))
    L, at, vat = hip.L, H * dk * 4, (H + Hkv) * dk * 4
    hip.check(L.axhip_rope_frequencies(freq.ptr, rot, 10000.0, 0, 1.0, 0.0, 0.0, 0))
    hip.check(L.axhip_qk_norm_rope_fwd(x.ptr, ld, y.ptr, ldn, inv.ptr, dgq.ptr, dgk.ptr, 1e-6, dpos.ptr, freq.ptr, B * S, H, Hkv, dk, rot, 1.0, 1))
    hip.check(L.axhip_attn_fwd(y.ptr, ldn, y.ptr + at, ldn, x.ptr + vat, ld, S, o.ptr, H * dk, lse.ptr, B, H, Hkv, S, S, dk, 0.125, C.byref(r)))
    do, dy, dqkv, sq, sk = hip.array(d_o), hip.empty((B * S, ldn)), hip.empty((B * S, ld)), hip.empty((dk,)), hip.empty((dk,))
    hip.check(L.axhip_attn_bwd(y.ptr, ldn, y.ptr + at, ldn, x.ptr + vat, ld, S, o.ptr, H * dk, lse.ptr, do.ptr, H * dk, dy.ptr, ldn, dy.ptr + at, ldn, dqkv.ptr + vat, ld,
                               B, H, Hkv, S, S, dk, 0.125, C.byref(r)))
    hip.check(L.axhip_qk_norm_rope_bwd(dy.ptr, ldn, x.ptr, ld, inv.ptr, dqkv.ptr, ld, dgq.ptr, dgk.ptr, sq.ptr, sk.ptr, dpos.ptr, freq.ptr, B * S, H, Hkv, dk, rot, 1.0, 1))

    f = freq.numpy()
    x64 = qkv[:, :H + Hkv].astype(np.float64)
    gamma = np.concatenate([np.tile(gq, (H, 1)), np.tile(gk, (Hkv, 1))]).astype(np.float64)
    r64 = inv_rms(x64, 1e-6)
    normed = rotate(x64 * r64[..., None] * gamma, pos, f, rot, 1.0, 1).reshape(B, S, H + Hkv, dk)
    v64 = qkv[:, H + Hkv:].reshape(B, S, Hkv, dk)
    want = attention(normed[:, :, :H], normed[:, :, H:], v64, 0.125, rules, d_o)
    dn = rotate(np.concatenate([want["dq"], want["dk"]], 2).reshape(B * S, H + Hkv, dk), pos, f, rot, 1.0, 1, back=True)
    dx, dg = norm_grad(dn, x64, r64, gamma)
    full = np.concatenate([dx, want["dv"].reshape(B * S, Hkv, dk)], 1)
    got = dqkv.numpy().reshape(full.shape)
    # each of the four passes adds some 1e-6 of its outputs' size (a hundred half steps of fp32, a few times what any of them was measured at)
    def near(a, b):
        return np.linalg.norm(a - b) <= 100 * 2.0 ** -24 * 2 * np.linalg.norm(b)
    assert near(o.numpy().reshape(want["o"].shape), want["o"]) and near(got, full)
    assert near(sq.numpy(), dg[:, :H].sum((0, 1))) and near(sk.numpy(), dg[:, H:].sum((0, 1)))

    last = np.stack([y.numpy().reshape(B, S, -1)[b, lens[b] - 1, :H * dk] for b in range(B)])
    step, held2 = device_rules(hip, Rules(cap=30.0, causal=1, lens=lens, start=lens - 1))
    dl, o1 = hip.array(last), hip.empty((B, H * dk))
    hip.check(L.axhip_attn_fwd(dl.ptr, H * dk, y.ptr + at, ldn, x.ptr + vat, ld, S, o1.ptr, H * dk, None, B, H, Hkv, 1, S, dk, 0.125, C.byref(step)))
    prompt = o.numpy().reshape(B, S, H * dk)
    assert near(o1.numpy(), np.stack([prompt[b, lens[b] - 1] for b in range(B)]))


@pytest.mark.parametrize("dk", [32, 64, 96, 128])
def test_large_rows_beside_ordinary_ones(hip, dk):
    """Keys, values, queries and gradients whose rows differ by 10^15 and more, next to each other: what does not see the large ones, and what sees them with a probability
    of nothing, is held to its own size."""
    say("attn large rows", dk)
    B, S, H = 1, 130, 2
    rng, q, k, v, d_o = draw(14, B, S, S, H, 1, dk)
    v[0, 70] *= np.float32(1e20)                          # rows 0 .. 69 do not see it
    k[0, 75, 0, 0], q[0, :, :, 0] = 1e18, -1e-3           # seen with a score of -1e15 scale
    q[0, 20:22] *= np.float32(1e-15)
    d_o[0, 90] *= np.float32(1e-12)
    d_o[0, 33] *= np.float32(1e12)
    rules = Rules(causal=1)
    want = attention(q, k, v, dk ** -0.5, rules, d_o)
    # what the large value and gradient add to others is in their bounds, as in any fp32 sum
    check(hip, q, k, v, dk ** -0.5, rules, d_o, want=want)


def some_heads(rules, b, heads):
    """The rules of one sequence and some query heads"""
    cut = {n: None if getattr(rules, n) is None else np.asarray(getattr(rules, n))[heads if n == "slopes" else slice(b, b + 1)] for n in Rules.ARRAYS}
    return Rules(cap=rules.cap, causal=rules.causal, **cut)


@pytest.mark.parametrize("kind", ["plain", "causal", "documents", "everything"])
@pytest.mark.parametrize("B,Sq,Sk,H,Hkv,dk", [(1, 500, 500, 8, 2, 64), (1, 700, 40, 4, 4, 128), (1, 40, 1500, 2, 1, 96), (1, 1100, 1100, 1, 1, 32), (1, 333, 333, 4, 1, 80), (1, 1, 700, 2, 2, 64),
                                               (1, 600, 600, 16, 4, 128), (1, 128, 520, 64, 16, 128)])
def test_gradients_of_few_tiles(hip, B, Sq, Sk, H, Hkv, dk, kind):
    """Few tiles of rows or keys: workgroups share what each runs over and meet in memory; the same bits whoever comes last."""
    rng, q, k, v, d_o = draw(29, B, Sq, Sk, H, Hkv, dk)
    rules = rules_of(kind, rng, B, Sq, Sk, H)
    want = attention(q, k, v, 1 / dk ** 0.5, rules, d_o)
    first, second = (check(hip, q, k, v, 1 / dk ** 0.5, rules, d_o, want=want) for _ in range(2))
    for n in ("dq", "dk", "dv"):
        assert first[n].tobytes() == second[n].tobytes(), n


@pytest.mark.parametrize("dk", [32, 64, 100, 128])
def test_few_tiles_with_garbage_between(hip, dk):
    """NaN in keys that no query sees, beside others in their tiles: rows formed again by the last of several workgroups, the same bits each time."""
    S, H, Hkv = 420, 2, 1
    rng, q, k, v, d_o = draw(31, 1, S, S, H, Hkv, dk)
    ids = rng.integers(0, 2, (1, S)).astype(np.int32)
    ids[0, ::37] = -1
    rules = Rules(doc_q=ids, doc_k=ids)
    hidden = ids[0] < 0
    k[0, hidden] = v[0, hidden] = q[0, hidden] = d_o[0, hidden] = 0
    want = attention(q, k, v, 1 / dk ** 0.5, rules, d_o)
    k[0, hidden] = v[0, hidden] = q[0, hidden] = d_o[0, hidden] = np.nan
    first, second = (check(hip, q, k, v, 1 / dk ** 0.5, rules, d_o, want=want) for _ in range(2))
    for n in ("dq", "dk", "dv"):
        assert first[n].tobytes() == second[n].tobytes(), n


@pytest.mark.parametrize("dk", [20, 32, 48, 64, 80, 96, 100, 128])
@pytest.mark.parametrize("kind", ["plain", "capped", "documents", "everything"])
def test_many_heads(hip, dk, kind):
    """Enough tiles for the wide ones, forward and backward; a few heads of the first and last sequence are compared, keys shared by two heads."""
    say("attn many", dk, kind)
    B, S, H, Hkv = 8, 500, 64, 32
    rng, q, k, v, d_o = draw(dk, B, S, S, H, Hkv, dk)
    rules = rules_of(kind, rng, B, S, S, H)
    if rules.lens is not None:
        rules.lens[[0, -1]] = [S, 170]
        rules.start = None
    if kind == "documents":
        rules.causal = 0
    r, held = device_rules(hip, rules)
    ld, ldk = H * dk, Hkv * dk
    dq, dk_, dv, do, o, lse = hip.array(q), hip.array(k), hip.array(v), hip.array(d_o), hip.empty(q.shape), hip.empty((B, H, S))
    grads = [hip.empty(x.shape) for x in (q, k, v)]
    hip.check(hip.L.axhip_attn_fwd(dq.ptr, ld, dk_.ptr, ldk, dv.ptr, ldk, S, o.ptr, ld, lse.ptr, B, H, Hkv, S, S, dk, 0.1, C.byref(r)))
    assert hip.last_kernel() == "attn_tiles_256"
    hip.check(hip.L.axhip_attn_bwd(dq.ptr, ld, dk_.ptr, ldk, dv.ptr, ldk, S, o.ptr, ld, lse.ptr, do.ptr, ld, grads[0].ptr, ld, grads[1].ptr, ldk, grads[2].ptr, ldk,
                                   B, H, Hkv, S, S, dk, 0.1, C.byref(r)))
    assert hip.last_kernel() == "attn_grad_tiles"
    o, lse, grads = o.numpy(), lse.numpy(), [g.numpy() for g in grads]
    for b, h in ((0, 0), (0, 62), (B - 1, 34)):
        heads, kv = slice(h, h + 2), slice(h // 2, h // 2 + 1)
        part = some_heads(rules, b, heads)
        want = attention(q[b:b + 1, :, heads], k[b:b + 1, :, kv], v[b:b + 1, :, kv], 0.1, part, d_o[b:b + 1, :, heads])
        empty = np.isneginf(want["lse"])
        assert np.array_equal(np.isneginf(lse[b:b + 1, heads]), empty)
        within(o[b:b + 1, :, heads], want, "o")
        within(np.where(empty, 0, lse[b:b + 1, heads]), dict(want, lse=np.where(empty, 0, want["lse"])), "lse")
        for n, g, hh in (("dq", grads[0], heads), ("dk", grads[1], kv), ("dv", grads[2], kv)):
            # the gradient from the kernel's own O and log-sum-exp, off by their bounds: twice each bound holds both
            within(g[b:b + 1, :, hh], {n: want[n], "tol_" + n: 2 * want["tol_" + n]}, n)


@pytest.mark.parametrize("B,H,Hkv,Sq,Sk,dk,form", [(1, 8, 1, 4, 4000, 64, "attn_few_ranges"), (1, 8, 1, 5, 4000, 64, "attn_few_ranges"), (4, 4, 4, 512, 512, 64, "attn_few"),
                                                   (4, 16, 16, 400, 400, 64, "attn_tiles_128"), (32, 16, 2, 40, 200, 96, "attn_tiles_128"), (1, 64, 1, 1, 3000, 128, "attn_few_ranges"),
                                                   (2, 2, 2, 33, 100, 36, "attn_few")])
@pytest.mark.parametrize("kind", ["plain", "distance"])
def test_which_form_takes_it(hip, B, H, Hkv, Sq, Sk, dk, form, kind):
    """Both sides of the rules, several tiles of rows in the form for few rows among them (256 CUs)."""
    say("attn forms", B, H, Hkv, Sq, Sk, dk)
    rng, q, k, v, _ = draw(Sq + Sk, B, Sq, Sk, H, Hkv, dk)
    r = Rules() if kind == "plain" else Rules(slopes=(2.0 ** -rng.uniform(1, 6, H)).astype(np.float32))
    rules, held = device_rules(hip, r)
    dq, dk_, dv, o, lse = hip.array(q), hip.array(k), hip.array(v), hip.empty(q.shape), hip.empty((B, H, Sq))
    hip.check(hip.L.axhip_attn_fwd(dq.ptr, H * dk, dk_.ptr, Hkv * dk, dv.ptr, Hkv * dk, Sk, o.ptr, H * dk, lse.ptr, B, H, Hkv, Sq, Sk, dk, 0.2, C.byref(rules)))
    assert hip.last_kernel().startswith(form), hip.last_kernel()
    o, lse = o.numpy(), lse.numpy()
    for b, h in ((0, 0), (B - 1, H - 1)):
        want = attention(q[b:b + 1, :, h:h + 1], k[b:b + 1, :, h * Hkv // H][:, :, None], v[b:b + 1, :, h * Hkv // H][:, :, None], 0.2, some_heads(r, b, slice(h, h + 1)))
        within(o[b:b + 1, :, h:h + 1], want, "o")
        within(lse[b:b + 1, h:h + 1], want, "lse")


@pytest.mark.parametrize("causal", [False, True])
def test_backward_with_the_extension_signature(hip, causal):
    """ax_hip_sdpa_fwd and ax_hip_sdpa_bwd, one after the other, on device memory"""
    from axiom_amd.axiom import Axiom
    ax = Axiom()
    assert ax.L.ax_init() == 0, ax.err()
    BH, S, dk = 6, 150, 64
    rng, q, k, v, d_o = draw(41, BH, S, S, 1, 1, dk)
    want = attention(q, k, v, 0.125, Rules(causal=int(causal)), d_o)
    dq, dk_, dv, do = (hip.array(x.reshape(BH, S, dk)) for x in (q, k, v, d_o))
    o, lse, *grads = (hip.array(np.full(s, 7, np.float32)) for s in ((BH, S, dk), (BH, S)) + ((BH, S, dk),) * 3)
    assert ax.L.ax_hip_sdpa_fwd(dq.ptr, dk_.ptr, dv.ptr, o.ptr, lse.ptr, BH, S, dk, 0.125, causal, None) == 0
    # the gradient's bounds hold for an O and L that are rounded once
    o, lse = hip.array(want["o"].astype(np.float32).reshape(BH, S, dk)), hip.array(want["lse"].astype(np.float32).reshape(BH, S))
    args = [dq.ptr, dk_.ptr, dv.ptr, o.ptr, do.ptr, lse.ptr, *(g.ptr for g in grads), BH, S, dk, 0.125, causal, None]
    assert ax.L.ax_hip_sdpa_bwd(*args) == 0
    for n, g, x in zip(("dq", "dk", "dv"), grads, (q, k, v)):
        within(g.numpy().reshape(x.shape), want, n)
    args[5] = None
    assert ax.L.ax_hip_sdpa_bwd(*args) == 1


def test_caches_past_32_bits(hip):
    """Rows of a sequence, and sequences, that lie more than 2^32 bytes behind the pointer: 2 sequences of 1.2 million rows of 8 heads of 128, 4.9 GB each.  Keys are zero,
    so every probability is one over their number."""
    B, rows, Hkv, G, dk = 2, 1200000, 8, 2, 128
    ld, H = Hkv * dk, Hkv * G
    k, v = hip.empty((B * rows, ld)), hip.empty((B * rows, ld))      # zeroes
    rng = np.random.default_rng(15)
    tail = rng.normal(size=(B, 7, Hkv, dk)).astype(np.float32) * np.float32(rows)
    for b in range(B):
        piece = np.ascontiguousarray(tail[b])
        hip.check(hip.L.axhip_memcpy_h2d(v.ptr + 4 * ld * (b * rows + rows - 7), piece.ctypes.data, piece.nbytes))
    q, d_o = (rng.normal(size=(B, 3, H, dk)).astype(np.float32) for _ in range(2))
    dq, o, lse = hip.array(q), hip.empty(q.shape), hip.empty((B, H, 3))
    for Sq in (1, 3):
        hip.check(hip.L.axhip_attn_fwd(dq.ptr, H * dk, k.ptr, ld, v.ptr, ld, rows, o.ptr, H * dk, lse.ptr, B, H, Hkv, Sq, rows, dk, 0.1, None))
        want = tail.astype(np.float64).sum(1) / rows                 # [B, Hkv, dk]
        got = o.numpy().reshape(-1)[:B * Sq * H * dk].reshape(B, Sq, Hkv, G, dk)
        # seven terms of a size of one, each probability off by the sums' roundings over 37500 tiles at most
        assert np.abs(got - want[:, None, :, None]).max() <= 1e-5 * np.abs(want).max() + 1e-5
    k_grad, v_grad = hip.empty((B * rows, ld)), hip.empty((B * rows, ld))
    do, dqg = hip.array(d_o), hip.empty(q.shape)
    hip.check(hip.L.axhip_attn_bwd(dq.ptr, H * dk, k.ptr, ld, v.ptr, ld, rows, o.ptr, H * dk, lse.ptr, do.ptr, H * dk, dqg.ptr, H * dk, k_grad.ptr, ld, v_grad.ptr, ld,
                                   B, H, Hkv, 3, rows, dk, 0.1, None))
    want = d_o.astype(np.float64).reshape(B, 3, Hkv, G, dk).sum((1, 3)) / rows
    for b in range(B):
        for at in (0, 40000, rows - 1):
            row = np.empty((Hkv, dk), np.float32)
            hip.check(hip.L.axhip_memcpy_d2h(row.ctypes.data, v_grad.ptr + 4 * ld * (b * rows + at), row.nbytes))
            assert np.abs(row - want[b]).max() <= 1e-5 * np.abs(want).max()
    assert (dqg.numpy() == 0).all()                                  # keys of zero
