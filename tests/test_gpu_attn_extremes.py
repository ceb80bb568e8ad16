"""Attention under score rules on the GPU at the ends of what fp32 holds, against 64 bits (attn_oracle.py, whose bounds these tests use as they are): every form of the
forward pass and the gradient."""
import numpy as np
import pytest

from attn_oracle import Rules
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
