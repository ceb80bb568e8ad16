"""The 64-bit definitions that the kernels of attention under score rules and of rotated, normed heads are held to: their gradients against differences, and what
no query sees against garbage."""
import numpy as np
import pytest

from attn_oracle import Rules, attention, inv_rms, norm_grad, rotate

RULES = {
    "plain": dict(),
    "capped": dict(cap=2.0, causal=1),
    "distance": dict(causal=1, slopes=np.array([0.5, 0.1])),
    "prefix": dict(causal=1, prefix=np.array([3, 0]), lens=np.array([5, 6])),
    "documents": dict(cap=5.0, doc_q=np.array([[0, 0, 1, 1, -1], [2, 2, 2, 0, 0]]), doc_k=np.array([[0, 1, 1, 0, -1, 1], [0, 2, 0, 2, 2, -1]])),
}


@pytest.mark.parametrize("name", RULES)
def test_gradients_against_differences(name):
    rng = np.random.default_rng(3)
    rules = Rules(**RULES[name])
    q, k, v = rng.normal(size=(2, 5, 2, 4)), rng.normal(size=(2, 6, 1, 4)), rng.normal(size=(2, 6, 1, 4))
    d_o = rng.normal(size=q.shape)
    got = attention(q, k, v, 0.7, rules, d_o)
    for which, x, g in ((0, q, got["dq"]), (1, k, got["dk"]), (2, v, got["dv"])):
        num = np.zeros_like(x)
        for at in np.ndindex(x.shape):
            sides = []
            for sign in (1, -1):
                y = [q, k, v]
                y[which] = x.copy()
                y[which][at] += sign * 1e-5
                sides.append((attention(*y, 0.7, rules)["o"] * d_o).sum())
            num[at] = (sides[0] - sides[1]) / 2e-5
        assert np.abs(num - g).max() < 1e-8


@pytest.mark.parametrize("layout", [0, 1])
def test_norm_and_rotation_against_differences(layout):
    rng = np.random.default_rng(4)
    x, dy, gamma = rng.normal(size=(3, 2, 8)), rng.normal(size=(3, 2, 8)), rng.normal(size=8)
    pos, freq = np.array([0, 5, 1000000]), np.array([1.0, 0.3])
    f = lambda x, gamma: rotate(gamma * x * inv_rms(x, 1e-3)[..., None], pos, freq, 4, 1.2, layout)
    dx, dn = norm_grad(rotate(dy, pos, freq, 4, 1.2, layout, back=True), x, inv_rms(x, 1e-3), gamma)
    for at in np.ndindex(x.shape):
        a, b = x.copy(), x.copy()
        a[at] += 1e-5
        b[at] -= 1e-5
        assert abs(((f(a, gamma) - f(b, gamma)) * dy).sum() / 2e-5 - dx[at]) < 1e-8
    for c in range(8):
        a, b = gamma.copy(), gamma.copy()
        a[c] += 1e-5
        b[c] -= 1e-5
        assert abs(((f(x, a) - f(x, b)) * dy).sum() / 2e-5 - dn.sum((0, 1))[c]) < 1e-8


def test_what_nobody_sees_is_left_out():
    rng = np.random.default_rng(5)
    q, k, v, d_o = (rng.normal(size=(1, 4, 1, 4)) for _ in range(4))
    rules = Rules(causal=1, lens=np.array([2]))
    clean = attention(q, k, v, 0.5, rules, d_o)
    for x in (q, k, v, d_o):
        x[0, 2:] = np.nan
    dirty = attention(q, k, v, 0.5, rules, d_o)
    for n in ("o", "lse", "dq", "dk", "dv"):
        assert np.array_equal(clean[n], dirty[n])
    assert (clean["o"][0, 2:] == 0).all() and (clean["lse"][0, 0, 2:] == -np.inf).all() and (clean["dk"][0, 2:] == 0).all()
