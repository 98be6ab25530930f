"""The e4m3 oracle on the CPU: its quantiser against torch's own e4m3 conversion, and its scales at the borders."""
import numpy as np
import torch

from oracle import fp8


def test_codes_match_torch():
    rng = np.random.default_rng(0)
    x = (rng.standard_normal((5, 300)) * np.exp(rng.standard_normal((5, 1)))).astype(np.float32)
    s = fp8.group_scales(x.astype(np.float64))
    want = torch.from_numpy(x / fp8.spread(s, 300).astype(np.float32)).to(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(fp8.codes(x.astype(np.float64), s), want)
    assert np.abs(want).max() <= 448


def test_scales_are_the_least_power_of_two():
    tops = [0.0, 2.0 ** -120, fp8.LEAST, np.nextafter(fp8.LEAST, 1), 448.0, np.nextafter(448.0, 500), 224.0, 1.0, 3e38]
    for top in tops:
        x = np.zeros((1, 130))
        x[0, 7] = -top
        s = fp8.group_scales(x)
        assert s[0, 1] == 2.0 ** -100
        v = s[0, 0]
        assert v >= 2.0 ** -100 and np.log2(v) == np.round(np.log2(v)) and top <= 448 * v
        assert v == 2.0 ** -100 or top > 448 * v / 2
    for bad in (np.inf, -np.inf, np.nan):
        x = np.ones((1, 256))
        x[0, 200] = bad
        s = fp8.group_scales(x)
        assert s[0, 0] == 2.0 ** -8 and np.isnan(s[0, 1])
        assert np.isnan(fp8.quantized(x)[0, 128:]).all()


def test_rounding_is_half_a_step_at_most():
    rng = np.random.default_rng(1)
    x = rng.standard_normal((20, 256))
    s = fp8.spread(fp8.group_scales(x), 256)
    err = np.abs(fp8.quantized(x) - x)
    # half a step: 2^-4 of the value, and of the least normal code (2^-6) below it
    assert (err <= 2.0 ** -4 * np.maximum(np.abs(x), 2.0 ** -6 * s)).all()
