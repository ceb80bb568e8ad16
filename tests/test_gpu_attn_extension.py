"""ax_hip_sdpa_fwd and ax_hip_sdpa_bwd as a caller uses them: the gradient from the O and the log-sum-exp that the forward pass left."""
import numpy as np
import pytest

from attn_oracle import Rules, attention
from test_gpu_attn import draw, within

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("BH,S,dk", [(6, 150, 64), (2, 1, 4), (3, 77, 128), (1, 300, 36)])
def test_forward_then_backward(hip, BH, S, dk, causal):
    from axiom_amd.axiom import Axiom
    ax = Axiom()
    assert ax.L.ax_init() == 0, ax.err()
    rng, q, k, v, d_o = draw(61, BH, S, S, 1, 1, dk)
    want = attention(q, k, v, dk ** -0.5, Rules(causal=int(causal)), d_o)
    dq, dk_, dv, do = (hip.array(x.reshape(BH, S, dk)) for x in (q, k, v, d_o))
    o, lse, *grads = (hip.array(np.full(s, 7, np.float32)) for s in ((BH, S, dk), (BH, S)) + ((BH, S, dk),) * 3)
    assert ax.L.ax_hip_sdpa_fwd(dq.ptr, dk_.ptr, dv.ptr, o.ptr, lse.ptr, BH, S, dk, dk ** -0.5, causal, None) == 0
    # the bounds of the kernels under rules hold for products of two terms; plain attention has three, of more bits
    within(o.numpy().reshape(q.shape), want, "o")
    within(lse.numpy().reshape(BH, 1, S), want, "lse")
    assert ax.L.ax_hip_sdpa_bwd(dq.ptr, dk_.ptr, dv.ptr, o.ptr, do.ptr, lse.ptr, *(g.ptr for g in grads), BH, S, dk, dk ** -0.5, causal, None) == 0
    for n, g, x in zip(("dq", "dk", "dv"), grads, (q, k, v)):
        # from the kernel's own O and log-sum-exp, off by their bounds: twice each bound holds both
        within(g.numpy().reshape(x.shape), {n: want[n], "tol_" + n: 2 * want["tol_" + n]}, n)
