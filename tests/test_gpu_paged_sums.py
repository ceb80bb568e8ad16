"""Attention over a paged cache where sums of values pass the largest float though their mean, which is the result, does not: every form, against 64 bits."""
import numpy as np
import pytest

from test_gpu_paged import TYPES, say
from test_gpu_paged_tiles import FORMS, NEW, NONE, held, normal

pytestmark = pytest.mark.gpu

FEW = [1, 2] + NONE
ALL = [(FEW, 2, [150, 180], "paged_few"), (FEW, 2, [1500, 1700], "paged_few_ranges")] + [(NEW, G, lens, kernel) for G, lens, _, kernel in FORMS]


@TYPES
@pytest.mark.parametrize("new,G,lens,kernel", ALL, ids=[f[-1] for f in ALL])
@pytest.mark.parametrize("signs", [False, True], ids=["positive", "mixed"])
def test_values_near_the_largest_float(hip, kind, new, G, lens, kernel, signs):
    """Rows of values of 1e38 to 3e38 (off by rounding of the 64-bit ones; the mean of such is a float), and one tiny column group, whose sums stay what they are."""
    say("paged sums", kind, kernel, signs)
    rng = np.random.default_rng(40)
    heads, dk, lens = 2, 64, lens + NONE
    k = [normal(rng, n, heads, dk) for n in lens]
    v = [rng.uniform(1e38, 3e38, (n, heads, dk)).astype(np.float32) for n in lens]
    if signs:
        v = [x * rng.choice([-1, 1], x.shape).astype(np.float32) for x in v]
    for x in v:
        x[:, 1, 32:] *= np.float32(1e-37)
    held(hip, kind, G, dk, lens, kernel, k, v, normal(rng, sum(new), heads * G, dk), 0.125, {}, new)
