"""Rotary positions and norms of heads on the GPU against 64 bits: both layouts, part of a head, sizes on and off the 16-byte grid, pitches, in place, gradients."""
import numpy as np
import pytest

from attn_oracle import U, inv_rms, norm_grad, pair_size, rotate

pytestmark = pytest.mark.gpu

# A value of a rotation: sine and cosine 3 U and the amplitude 1 U, two products and a sum 3 U, of the size of its pair.
TURN = 8 * U
# 1 / rms of up to 512 values: the sum of squares at most 16 + 6 steps, mean, eps, square root and reciprocal 4 more, half of the sum's for the root.
INV = 16 * U
NORM = TURN + INV + 3 * U


def say(*a):
    print(*a, flush=True)


def rows_of(hip, x, ld, garbage=np.nan):
    """x [rows, n] on the device with row pitch ld, garbage between"""
    full = np.full((x.shape[0], ld), garbage, np.float32)
    full[:, :x.shape[1]] = x
    return hip.array(full)


SHAPES = [(1, 1, 8, 8), (8, 20, 64, 64), (3, 5, 80, 40), (37, 2, 128, 128), (130, 3, 96, 32), (5, 1, 512, 512), (300, 7, 32, 16), (2, 3, 48, 0), (4, 2, 256, 64), (2, 70, 16, 16),
          # off the grid of units: by head size, by rotated part, by more than 512 columns
          (7, 3, 12, 6), (5, 2, 63, 10), (9, 2, 64, 60), (3, 2, 1000, 500), (2, 1, 2, 2)]


@pytest.mark.parametrize("rows,H,dk,rot", SHAPES)
@pytest.mark.parametrize("layout", [0, 1])
@pytest.mark.parametrize("pitch", [0, 4, 3])
def test_rotation(hip, rows, H, dk, rot, layout, pitch):
    say("rope", rows, H, dk, rot, layout, pitch)
    rng = np.random.default_rng(rows + dk + rot)
    x = rng.normal(size=(rows, H * dk)).astype(np.float32)
    pos = rng.integers(-5, 1 << 20, rows).astype(np.int32)
    pos[0] = (1 << 24) - 1
    freq = (10000.0 ** (-2.0 * np.arange(max(rot // 2, 1)) / max(rot, 1))).astype(np.float32)
    ld, dpos, dfreq = H * dk + pitch, hip.array(pos), hip.array(freq)
    for amplitude, back in ((1.0, 0), (1.3, 1)):
        dx, dy = rows_of(hip, x, ld), rows_of(hip, np.zeros_like(x), ld, 7.0)
        hip.check(hip.L.axhip_rope_rows(dx.ptr, ld, dy.ptr, ld, dpos.ptr, dfreq.ptr, rows, H, dk, rot, amplitude, layout, back))
        got = dy.numpy()
        assert (got[:, H * dk:] == 7.0).all()
        got = got[:, :H * dk].reshape(rows, H, dk)
        x3 = x.reshape(rows, H, dk)
        want = rotate(x3.astype(np.float64), pos, freq[:rot // 2], rot, np.float32(amplitude), layout, back)
        assert (np.abs(got - want) <= TURN * pair_size(x3, rot, amplitude, layout)).all()
        assert np.array_equal(got[..., rot:], x3[..., rot:])
        hip.check(hip.L.axhip_rope_rows(dx.ptr, ld, dx.ptr, ld, dpos.ptr, dfreq.ptr, rows, H, dk, rot, amplitude, layout, back))
        assert np.array_equal(dx.numpy()[:, :H * dk].reshape(rows, H, dk), got)


def test_positions_at_the_ends_of_32_bits(hip):
    """The angle is exact to 2^-53 of its turns: 2^31 / 2 pi of them, off by 2 pi 2^28.4 2^-53 = 2^-22 at most."""
    pos, freq = np.array([2 ** 31 - 1, -2 ** 31, 123456789, -1], np.int32), np.array([1.0, 0.1, 3e-5, 0.9999], np.float32)
    x = np.ones((4, 8), np.float32)
    y = hip.empty((4, 8))
    dx, dp, df = hip.array(x), hip.array(pos), hip.array(freq)
    hip.check(hip.L.axhip_rope_rows(dx.ptr, 8, y.ptr, 8, dp.ptr, df.ptr, 4, 1, 8, 8, 1.0, 1, 0))
    a = np.array([[np.longdouble(int(p)) * np.longdouble(float(f)) for f in freq] for p in pos])
    want = np.concatenate([np.cos(a) - np.sin(a), np.cos(a) + np.sin(a)], 1).astype(np.float64)
    assert np.abs(y.numpy() - want).max() <= 2 * TURN + 2 * 2.0 ** -22


@pytest.mark.parametrize("scaling,args", [(0, (1.0, 0, 0, 0)), (1, (4.0, 0, 0, 0)), (2, (8.0, 0, 0, 0)), (3, (16.0, 1.0, 32.0, 2048))])
@pytest.mark.parametrize("rot", [2, 64, 128])
def test_frequencies(hip, scaling, args, rot):
    factor, slow, fast, trained = args
    out = hip.array(np.full(rot // 2 + 1, 7, np.float32))
    hip.check(hip.L.axhip_rope_frequencies(out.ptr, rot, 10000.0, scaling, factor, slow, fast, trained))
    i = np.arange(rot // 2)
    theta = 10000.0 * factor ** (rot / (rot - 2)) if scaling == 2 and rot > 2 else 10000.0
    f = theta ** (-2 * i / rot)
    if scaling == 1:
        f = f / factor
    if scaling == 3:
        keep = np.clip((trained * f / (2 * np.pi) - slow) / (fast - slow), 0, 1)
        f = f * keep + f / factor * (1 - keep)
    got = out.numpy()
    assert got[-1] == 7 and (np.abs(got[:-1] - f) <= 1.01 * U * f).all()
    if scaling == 2 and rot > 2:
        assert abs(got[rot // 2 - 1] * factor / 10000.0 ** (-(rot - 2) / rot) - 1) < 1e-6


@pytest.mark.parametrize("rows,H,dk,rot", SHAPES)
@pytest.mark.parametrize("layout", [0, 1])
@pytest.mark.parametrize("Hk", [0, 1, 3])
def test_norm(hip, rows, H, dk, rot, layout, Hk):
    """Forward and gradient; a row holds values behind the keys, which stay as they are in place."""
    say("qk norm", rows, H, dk, rot, layout, Hk)
    rng = np.random.default_rng(rows + dk + rot + Hk)
    n, tail = H + Hk, 4
    ld = n * dk + tail + (-n * dk) % 4
    x = (rng.normal(size=(rows, n, dk)) * np.exp(rng.uniform(-3, 3, (rows, n, 1)))).astype(np.float32)
    dy = rng.normal(size=(rows, n, dk)).astype(np.float32)
    pos = rng.integers(0, 100000, rows).astype(np.int32)
    freq = (10000.0 ** (-2.0 * np.arange(max(rot // 2, 1)) / max(rot, 1))).astype(np.float32)
    gq, gk = (rng.normal(1, 0.3, dk).astype(np.float32) for _ in range(2))
    gamma = np.concatenate([np.tile(gq, (H, 1)), np.tile(gk, (Hk, 1))]).astype(np.float64)
    amplitude, eps = np.float32(1.2), np.float32(1e-5)
    dx, dpos, dfreq, dgq, dgk = rows_of(hip, x.reshape(rows, -1), ld, 7.0), hip.array(pos), hip.array(freq), hip.array(gq), hip.array(gk)
    y, inv = rows_of(hip, np.zeros((rows, n * dk), np.float32), ld, 7.0), hip.empty((rows, n))
    hip.check(hip.L.axhip_qk_norm_rope_fwd(dx.ptr, ld, y.ptr, ld, inv.ptr, dgq.ptr, dgk.ptr, eps, dpos.ptr, dfreq.ptr, rows, H, Hk, dk, rot, amplitude, layout))
    r = inv_rms(x, float(eps))
    ginv, gy = inv.numpy(), y.numpy()
    assert (np.abs(ginv - r) <= INV * r).all() and (gy[:, n * dk:] == 7).all()
    normed = x * r[..., None] * gamma
    want = rotate(normed, pos, freq[:rot // 2], rot, amplitude, layout)
    assert (np.abs(gy[:, :n * dk].reshape(rows, n, dk) - want) <= NORM * pair_size(normed, rot, amplitude, layout)).all()

    out, sq, sk = rows_of(hip, np.zeros((rows, n * dk), np.float32), ld, 7.0), hip.array(np.full(dk, 9, np.float32)), hip.array(np.full(dk, 9, np.float32))
    ddy = rows_of(hip, dy.reshape(rows, -1), ld)
    args = (dgq.ptr, dgk.ptr, sq.ptr, sk.ptr, dpos.ptr, dfreq.ptr, rows, H, Hk, dk, rot, amplitude, layout)
    hip.check(hip.L.axhip_qk_norm_rope_bwd(ddy.ptr, ld, dx.ptr, ld, inv.ptr, out.ptr, ld, *args))
    r = ginv.astype(np.float64)
    dn = rotate(dy.astype(np.float64), pos, freq[:rot // 2], rot, amplitude, layout, back=True)
    size = pair_size(dy, rot, amplitude, layout)
    want, dg = norm_grad(dn, x.astype(np.float64), r, gamma)
    hat = np.abs(x * r[..., None])
    g_size = size * np.abs(gamma)
    tol = r[..., None] * ((TURN + 4 * U) * g_size + (TURN + 32 * U) * hat * (g_size * hat).mean(-1, keepdims=True))
    got = out.numpy()
    assert (got[:, n * dk:] == 7).all() and (np.abs(got[:, :n * dk].reshape(rows, n, dk) - want) <= tol).all()
    # at most as many additions one after the other as there are terms, and no more than 256
    for mine, part in ((sq.numpy(), slice(0, H)), (sk.numpy(), slice(H, n))):
        terms = (size * hat)[:, part].sum((0, 1))
        assert (np.abs(mine - dg[:, part].sum((0, 1))) <= (TURN + (8 + min(rows * n, 256)) * U) * terms + 1e-30).all()
    # in place: dx over dy, y over x
    hip.check(hip.L.axhip_qk_norm_rope_bwd(ddy.ptr, ld, dx.ptr, ld, inv.ptr, ddy.ptr, ld, *args[:2], None, None, *args[4:]))
    assert np.array_equal(ddy.numpy()[:, :n * dk], got[:, :n * dk])
    hip.check(hip.L.axhip_qk_norm_rope_fwd(dx.ptr, ld, dx.ptr, ld, None, dgq.ptr, dgk.ptr, eps, dpos.ptr, dfreq.ptr, rows, H, Hk, dk, rot, amplitude, layout))
    assert np.array_equal(dx.numpy(), gy)


def test_many_rows(hip):
    """More rows than groups of lanes, sums over all of them, the same bits from two calls; no gammas."""
    rows, H, Hk, dk, rot = 40001, 2, 1, 64, 32
    rng = np.random.default_rng(1)
    x, dy = (rng.normal(size=(rows, H + Hk, dk)).astype(np.float32) for _ in range(2))
    pos, freq = np.arange(rows, dtype=np.int32), (10000.0 ** (-np.arange(16) / 16)).astype(np.float32)
    ld = (H + Hk) * dk
    dx, ddy, dpos, dfreq, y, inv = hip.array(x), hip.array(dy), hip.array(pos), hip.array(freq), hip.empty(x.shape), hip.empty((rows, H + Hk))
    hip.check(hip.L.axhip_qk_norm_rope_fwd(dx.ptr, ld, y.ptr, ld, inv.ptr, None, None, 1e-6, dpos.ptr, dfreq.ptr, rows, H, Hk, dk, rot, 1.0, 1))
    r = inv_rms(x, 1e-6)
    normed = x * r[..., None]
    assert (np.abs(y.numpy() - rotate(normed, pos, freq, rot, 1, 1)) <= NORM * pair_size(normed, rot, 1, 1)).all()
    seen = []
    for _ in range(2):
        out, sq, sk = hip.empty(x.shape), hip.empty((dk,)), hip.empty((dk,))
        hip.check(hip.L.axhip_qk_norm_rope_bwd(ddy.ptr, ld, dx.ptr, ld, inv.ptr, out.ptr, ld, None, None, sq.ptr, sk.ptr, dpos.ptr, dfreq.ptr, rows, H, Hk, dk, rot, 1.0, 1))
        seen.append((out.numpy(), sq.numpy(), sk.numpy()))
    assert all(np.array_equal(a, b) for a, b in zip(*seen))
    _, dg = norm_grad(rotate(dy.astype(np.float64), pos, freq, rot, 1, 1, back=True), x.astype(np.float64), inv.numpy().astype(np.float64), 1.0)
    terms = (pair_size(dy, rot, 1, 1) * np.abs(normed))
    for mine, part in ((seen[0][1], slice(0, H)), (seen[0][2], slice(H, None))):
        assert (np.abs(mine - dg[:, part].sum((0, 1))) <= (TURN + 264 * U) * terms[:, part].sum((0, 1))).all()


def test_what_is_not_finite_stays_in_its_head(hip):
    x = np.ones((2, 3 * 64), np.float32)
    x[0, 5], x[1, 64 + 7] = np.nan, np.inf
    dx, pos, freq, y = hip.array(x), hip.array(np.array([3, 4], np.int32)), hip.array(np.ones(32, np.float32)), hip.empty(x.shape)
    hip.check(hip.L.axhip_qk_norm_rope_fwd(dx.ptr, 192, y.ptr, 192, None, None, None, 1e-6, pos.ptr, freq.ptr, 2, 2, 1, 64, 64, 1.0, 1))
    bad = ~np.isfinite(y.numpy()).reshape(2, 3, 64)
    assert bad[0, 0].all() and not bad[0, 1:].any() and bad[1, 1].any() and not bad[1, [0, 2]].any()
