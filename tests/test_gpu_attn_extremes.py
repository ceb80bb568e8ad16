"""Attention under score rules on the GPU at the ends of what fp32 holds, against 64 bits (attn_oracle.py, whose bounds these tests use as they are): every form of the
forward pass and the gradient."""
import numpy as np
import pytest

from attn_oracle import Rules, attention
from test_gpu_attn import check, draw

pytestmark = pytest.mark.gpu

# (B, Sq, Sk, H, Hkv, dk) and the forward form that takes it: few rows in ranges of keys, tiles whose keys two waves share, tiles of 256 rows
FORMS = [((1, 20, 300, 4, 2, 64), "attn_few_ranges"), ((1, 1, 100, 2, 2, 128), "attn_few"), ((1, 40, 150, 300, 300, 32), "attn_tiles_128"), ((1, 70, 140, 260, 260, 128), "attn_tiles_128"),
         ((1, 200, 200, 260, 260, 32), "attn_tiles_256")]
FORM_IDS = [form + "_%d" % shape[-1] for shape, form in FORMS]


def say(*a):
    print(*a, flush=True)


@pytest.mark.parametrize("shape,form", FORMS, ids=FORM_IDS)
@pytest.mark.parametrize("cap", [1e-37, 1e-20, 1e20, 1e33, 1e36, 1e38, 3.4028234663852886e38])
def test_caps_of_any_size(hip, shape, form, cap):
    """A cap far above the scores leaves them as they are, one far below makes them signs."""
    say("attn cap", shape, cap)
    rng, q, k, v, d_o = draw(51, *shape)
    check(hip, q, k, v, 3 / shape[-1] ** 0.5, Rules(cap=cap), d_o, kernel=form)
    check(hip, q, k, v, 3 / shape[-1] ** 0.5, Rules(cap=cap, slopes=np.full(shape[3], 0.01, np.float32)), d_o)


def low_scores(shape, q_size):
    """Queries of a size of q_size and keys of its inverse; the scores lie around -14, between -4 and -24."""
    rng, _, _, v, d_o = draw(52, *shape)
    B, Sq, Sk, H, Hkv, dk = shape
    q = rng.normal(1, 0.1, size=(B, Sq, H, dk))
    k = rng.normal(-14 / dk, 3 / dk ** 0.5, size=(B, Sk, Hkv, dk))
    return (q * q_size).astype(np.float32), (k / q_size).astype(np.float32), v, d_o


@pytest.mark.parametrize("shape,form", FORMS, ids=FORM_IDS)
@pytest.mark.parametrize("q_size", [1e-27, 1e-18, 1e27])
def test_low_scores_from_small_and_large_factors(hip, shape, form, q_size):
    """A visible key counts whatever powers of two its score is formed from."""
    say("attn low scores", shape, q_size)
    q, k, v, d_o = low_scores(shape, q_size)
    d_o = d_o * np.float32(1e-3)
    check(hip, q, k, v, 1.0, Rules(), d_o, kernel=form)
    check(hip, q, k, v, 1.0, Rules(slopes=np.full(shape[3], 0.01, np.float32)), d_o)
    check(hip, q, k, v, 1.0, Rules(cap=100.0), d_o)


# ... over 1000 keys, so that few keys weigh little
LONG = [((1, 3, 1000, 4, 2, 64), "attn_few_ranges"), ((1, 1, 1000, 600, 600, 32), "attn_few"), ((1, 40, 1000, 300, 300, 32), "attn_tiles_128"), ((1, 200, 1000, 260, 260, 32), "attn_tiles_256")]
LONG_IDS = [form for _, form in LONG]


@pytest.mark.parametrize("shape,form", LONG, ids=LONG_IDS)
@pytest.mark.parametrize("size", [1e23, 1e25, 1e32, 1e35])
def test_a_very_large_value_leaves_the_others_their_weight(hip, shape, form, size):
    """One value row of any size, seen with a probability of two thirds: the other keys, each 2^-11 of it, keep theirs."""
    say("attn large value", shape, size)
    B, Sq, Sk, H, Hkv, dk = shape
    rng, q, k, v, _ = draw(53, *shape)
    q[..., 0], k[..., 0] = 1, -11 * np.log(2)
    for at in (0, 500, 999):
        kk, vv = k * np.float32(0.01), v.copy()
        kk[..., 0] = k[..., 0]
        kk[:, at, :, 0] = 0
        vv[:, at] *= np.float32(size)
        check(hip, q, kk, vv, 1.0, Rules(), kernel=form)


@pytest.mark.parametrize("shape,form", LONG, ids=LONG_IDS)
@pytest.mark.parametrize("low,high", [(0.0, 1e13), (1e-20, 1e20), (1e-30, 1e22), (0.0, 1e23)])
def test_values_of_nothing_and_a_large_one_share_their_weight(hip, shape, form, low, high):
    """Rows of values of zeros, or small ones, before and behind a large one: as many keys share the probability as there are."""
    say("attn uneven values", shape, low, high)
    rng, q, k, v, _ = draw(54, *shape)
    for at in (10, 500, 999):
        vv = v * np.float32(low)
        vv[:, at] = v[:, at] * np.float32(high)
        check(hip, q, k, vv, 0.05, Rules(), kernel=form)


@pytest.mark.parametrize("dk", [32, 64, 96, 128])
@pytest.mark.parametrize("k_size,v_size", [(1e15, 1.0), (1e20, 1.0), (1e30, 1.0), (1e16, 1e13), (100.0, 1e4), (1e-20, 1.0), (1e25, 1e-25)])
def test_gradients_that_grow_along_the_keys(hip, dk, k_size, v_size):
    """Keys and values of any size, values a thousand times larger behind the first 64 keys and again behind 200: the gradient of the queries takes its scale anew, from
    wherever it was."""
    say("attn growing", dk, k_size, v_size)
    rng, q, k, v, d_o = draw(55, 1, 90, 300, 2, 1, dk)
    v[:, 64:] *= np.float32(1e3)
    v[:, 200:] *= np.float32(1e3)
    check(hip, q / np.float32(k_size), k * np.float32(k_size), v * np.float32(v_size), dk ** -0.5, Rules(), d_o)
    check(hip, q / np.float32(k_size), k * np.float32(k_size), v * np.float32(v_size), dk ** -0.5, Rules(cap=5.0), d_o)


@pytest.mark.parametrize("shape,form", FORMS, ids=FORM_IDS)
def test_small_values_beside_large_ones(hip, shape, form):
    """Columns of values and of output gradients down to 2^-38 of their row: off by 2^-39 of the row's largest more than others, at most."""
    say("attn small beside large", shape)
    rng, q, k, v, d_o = draw(56, *shape)
    B, Sq, Sk, H, Hkv, dk = shape
    small = (2.0 ** -rng.integers(0, 39, dk)).astype(np.float32)
    small[0] = 1
    v, d_o = v * small, d_o * small
    plain = Rules()
    want = attention(q, k, v, dk ** -0.5, plain, d_o)
    # probabilities over the largest of each row: attention of values that are it in every column, and the gradient of values with such output gradients
    of_v = attention(q, k, np.broadcast_to(np.abs(v).max(-1, keepdims=True), v.shape), dk ** -0.5, plain)["o"]
    of_o = attention(q, k, v, dk ** -0.5, plain, np.broadcast_to(np.abs(d_o).max(-1, keepdims=True), d_o.shape))["dv"]
    want["tol_o"] += 2.0 ** -39 * of_v
    want["tol_dv"] += 2.0 ** -39 * of_o
    out = check(hip, q, k, v, dk ** -0.5, plain, want=want, kernel=form)
    # scores' gradients are sums over a row, whose largest decides
    check(hip, q, k, v, dk ** -0.5, plain, d_o, want=want)
    assert np.isfinite(out["o"]).all()
