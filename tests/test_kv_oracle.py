"""The oracle of the paged cache at hand-made values."""
import numpy as np

from kv_oracle import F16, I8, MX4, ladder_code, paged_attention, quantised, row_bytes


def test_ladder():
    y = np.array([0, 0.25, 0.26, 0.75, 0.7499, 1.25, 1.75, 2.5, 3.5, 5, 5.01, 6, 7, 7.99])
    assert ladder_code(y).tolist() == [0, 0, 1, 2, 1, 2, 4, 4, 6, 6, 7, 7, 7, 7]


def test_rows():
    assert [row_bytes(t, 4) for t in (F16, I8, MX4)] == [16, 16, 16] and [row_bytes(t, 80) for t in (F16, I8, MX4)] == [160, 80, 48]
    x = np.zeros((1, 1, 36), np.float32)
    x[0, 0, :4] = [127, 0.5, 1.5, -126.5]
    x[0, 0, 32:] = [3, -7.5, 0.3, np.nan]
    payload, scales, value = quantised(I8, x[..., :32])
    assert payload[0, 0].view(np.int8)[:4].tolist() == [127, 0, 2, -126] and scales.view(np.float32)[0, 0, 0] == 1
    payload, scales, value = quantised(MX4, x)
    # 127 = 1.98 * 2^6: s = 16, 7.94 -> 6
    assert scales[0, 0].tolist() == [127 + 4, 255, 0, 0] and payload[0, 0, :2].tolist() == [0x07, 0xf0] and np.isnan(value[0, 0, 32:]).all() and value[0, 0, 0] == 96
    payload, scales, value = quantised(F16, x[..., :32])
    assert scales.view(np.float32)[0, 0, 0] == 2.0 ** -8 and (value == x[..., :32]).all()
    for kind in (F16, I8):
        assert quantised(kind, np.zeros((1, 1, 4), np.float32))[1].view(np.float32)[0, 0, 0] == np.float32(2.0 ** -100)
        assert np.isnan(quantised(kind, x)[2]).all()
    assert quantised(MX4, np.zeros((1, 1, 4), np.float32))[1][0, 0].tolist() == [0, 0, 0, 0]


def test_attention_of_a_window():
    rng = np.random.default_rng(0)
    q, k, v = rng.normal(size=(3, 2, 8)), rng.normal(size=(9, 1, 8)), rng.normal(size=(9, 1, 8))
    there = np.ones(9, bool)
    there[1] = False
    w = paged_attention(q, k, v, there, 0.5, window=3, sinks=2)
    for i in range(3):
        p = 6 + i
        keys = [0] + list(range(p - 2, p + 1))
        for h in range(2):
            e = np.exp(k[keys, 0] @ q[i, h] * 0.5)
            assert np.allclose(w["o"][i, h], e @ v[keys, 0] / e.sum()) and np.allclose(w["lse"][i, h], np.log(e.sum()))
