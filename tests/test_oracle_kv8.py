"""The plain restatement of the 8-bit cache against torch's own e4m3 casts, and its
block rules on small examples."""

import math

import numpy as np
import pytest
import torch

from oracle import kv8


def test_codes_are_torch_e4m3():
    bits = torch.arange(256, dtype=torch.uint8)
    v = bits.view(torch.float8_e4m3fn).to(torch.float64).numpy()
    assert np.array_equal(v, kv8.CODE_VALUES, equal_nan=True)


def test_encode_rounds_as_torch():
    fine = np.linspace(-448.0, 448.0, 20011, dtype=np.float32)
    p = kv8.CODE_VALUES[:127]
    ties = ((p[1:] + p[:-1]) / 2).astype(np.float32)
    x = np.concatenate([fine, fine * np.float32(2.0 ** -12), ties, -ties, np.nextafter(ties, np.float32(1e9)),
                        np.nextafter(ties, np.float32(-1e9)), np.array([0.0, -0.0, 1e-30, 448.0], np.float32)])
    want = torch.from_numpy(x).to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert np.array_equal(kv8.encode(x), want)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_what_is_not_finite_is_nan(bad):
    assert math.isnan(kv8.CODE_VALUES[kv8.encode(np.array([bad]))[0]])


@pytest.mark.parametrize("amax,e", [(0.0, -100), (448.0, 0), (448.0001, 1), (449.0, 1), (1.0, -8), (1.75, -8), (1.7500001, -7),
                                    (2.0 ** -120, -100), (1.875 * 2.0 ** 127, 120)])
def test_exponent_is_the_least(amax, e):
    assert kv8.exponent(amax) == e


def test_a_block_grows_and_starts_anew():
    codes, scale = np.zeros((1, 2, 4, 1, 64), np.uint8), np.zeros((1, 2, 1), np.uint8)
    one = np.ones((1, 1, 64), np.float32)
    kv8.append(codes, scale, [0], [0], one, one, "bfloat16")
    assert scale[0, 0, 0] == 127 - 8
    kv8.append(codes, scale, [0], [1], one * 1000, one * 0.001, "bfloat16")
    v = kv8.values(codes, scale)
    assert scale[0, 0, 0] == 127 + 2 and scale[0, 1, 0] == 127 - 8          # K grew, V did not
    assert np.all(v[0, 0, 0] == 1.0) and np.all(v[0, 0, 1] == 1024.0)       # exact through the rescale
    assert np.all(v[0, 1, 0] == 1.0) and abs(v[0, 1, 1, 0, 0] - 0.001) <= 0.001 * 2.0 ** -4
    kv8.append(codes, scale, [0], [0], one * 0.001, one, "bfloat16")
    assert scale[0, 0, 0] == 127 - 18                                       # slot 0: anew


def test_values_keep_half_a_step():
    """Values down to 2^-14 of the block's largest are within 2^-4 of themselves."""
    g = np.random.default_rng(3)
    x = (np.exp2(g.uniform(-13.9, 0.0, (16, 1, 64))) * g.choice([-1.0, 1.0], (16, 1, 64)) * 37.0).astype(np.float32)
    x[0, 0, 0] = 37.0
    codes, scale = np.zeros((1, 2, 16, 1, 64), np.uint8), np.zeros((1, 2, 1), np.uint8)
    kv8.append(codes, scale, [0] * 16, range(16), x, x, "float16")
    v = kv8.values(codes, scale)[0, 0]
    assert np.all(np.abs(v - x) <= np.abs(x) * 2.0 ** -4)
