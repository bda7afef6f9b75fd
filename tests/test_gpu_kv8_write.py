"""Quantising writes at the borders between codes, built from the scale that a row really has."""
from fractions import Fraction

import numpy as np
import pytest

import kv8_ref
from test_gpu_kv8 import Cache, dev

pytestmark = pytest.mark.gpu


def peaks_with_exact_borders(rs, n):
    """Peaks in [1, 2) whose scale, fl32(peak * fl32(1 / 127)), has its lowest 8 bits zero: (i + 1/2) * scale is then an
    fp32 value for every code i, and a tie."""
    p = (1 + rs.rand(400 * n)).astype(np.float32)
    s = p * np.float32(1 / 127)
    return p[(s.view(np.uint32) & 255) == 0][:n]


@pytest.mark.parametrize("n_kv,hd", [(1, 128), (2, 64), (3, 64), (8, 128)])
@pytest.mark.parametrize("exponent", [-120, -100, -99, -20, 0, 3, 120])
def test_borders_of_the_scale_that_is_used(ctx, n_kv, hd, exponent):
    import torch
    rs = np.random.RandomState(n_kv * 128 + exponent)
    n = 24
    peak = peaks_with_exact_borders(rs, n * n_kv).reshape(n, n_kv) * np.float32(2.0) ** np.float32(exponent)
    scale = peak * np.float32(1 / 127)
    i = rs.randint(-127, 127, (n, n_kv, hd))
    tie = (i + 0.5) * scale[..., None].astype(np.float64)
    x = tie.astype(np.float32)
    assert np.array_equal(x.astype(np.float64), tie)
    side = rs.randint(-1, 2, x.shape)  # below, on and above the border
    x = np.where(side < 0, np.nextafter(x, np.float32(-np.inf)), np.where(side > 0, np.nextafter(x, np.float32(np.inf)), x))
    even = i + (i & 1)  # a tie goes to the even one of i and i + 1
    want = np.where(side < 0, i, np.where(side > 0, i + 1, even))
    x[..., 5], want[..., 5] = peak, 127
    c = Cache(ctx, 1, n, n_kv, hd)
    d, ds, dp = dev(x), dev(np.zeros(n, np.int32)), dev(np.arange(n, dtype=np.int32))
    torch.cuda.synchronize()
    c.h.write_device(d.data_ptr(), d.data_ptr(), ds.data_ptr(), dp.data_ptr(), n)
    ctx.sync()
    k, ks, v, vs = c.arrays()
    for codes, scales in ((k, ks), (v, vs)):
        assert np.array_equal(scales[0].T, scale)
        assert np.array_equal(codes[0].transpose(1, 0, 2), want)
    # the oracle, and rational arithmetic, agree
    assert np.array_equal(kv8_ref.quantize(x)[0], want)
    assert all(round(Fraction(float(x[0, 0, j])) / Fraction(float(scale[0, 0]))) == want[0, 0, j] for j in range(hd))
