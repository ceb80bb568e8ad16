"""The gammas' gradients of the head norms over many rows: what the workgroups leave is joined in 64 bits."""
import numpy as np
import pytest

from attn_oracle import U

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dk", [64, 128, 12])                        # 12: a wave per head
def test_sums_over_many_rows_are_rounded_once(hip, dk):
    """Terms are whole multiples of 2^-11 up to 2, few enough for a workgroup that its sums are exact in fp32; their sum over all rows is not, and is rounded once."""
    print("gamma sums", dk, flush=True)
    rows, H, Hk = (1 << 17) + 5, 1, 1
    rng = np.random.default_rng(dk)
    dy = (rng.integers(2048, 4096, (rows, H + Hk, dk)) / 2048).astype(np.float32)
    x = rng.choice(np.array([-1, 1], np.float32), (rows, 1, 1)) * np.ones_like(dy)
    dy *= x                                                           # all terms positive
    ld = (H + Hk) * dk
    dx, ddy, inv = hip.array(x), hip.array(dy), hip.array(np.ones((rows, H + Hk), np.float32))
    out, sq, sk = hip.empty(x.shape), hip.empty((dk,)), hip.empty((dk,))
    hip.check(hip.L.axhip_qk_norm_rope_bwd(ddy.ptr, ld, dx.ptr, ld, inv.ptr, out.ptr, ld, None, None, sq.ptr, sk.ptr, None, None, rows, H, Hk, dk, 0, 1.0, 0))
    want = (dy.astype(np.float64) * x).sum(0)
    for mine, exact in ((sq.numpy(), want[0]), (sk.numpy(), want[1])):
        assert (np.abs(mine - exact) <= U * exact).all(), np.abs(mine / exact - 1).max() / U
