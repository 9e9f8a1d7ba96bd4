"""Decode attention over a shared prefix with scales far from 1: a power of two that moves
from the scale of the scores to the scales of K changes no product, and so no bit."""
import numpy as np
import pytest

from gpu_util import print_case
from test_paged_prefix_gpu import COLUMNS, call, check, pool, queries
from test_serving_gpu import dev_, host, rng

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("power", [-110, -90, 60, 90])
@pytest.mark.parametrize("window", [0, 100])
@pytest.mark.parametrize("B,G", COLUMNS)
def test_prefix_scale_and_k_scales_far_from_one(dev, power, window, B, G):
    print_case("prefix far scales", power, window, B, G)
    g = rng(B, G)
    p = pool(g, 333, [0, 7, 40] + [3] * (B - 3), 1, 64, 16, True).upload()
    q = queries(g, B, G, 64)
    near = host(call(p, dev_(q), G, 0.125, window))
    check(p, near, q, G, 0.125, window)
    p.ks *= np.float32(2.0 ** -power)
    p.upload()
    far = host(call(p, dev_(q), G, 0.125 * 2.0 ** power, window))
    assert np.array_equal(near.view(np.uint16), far.view(np.uint16))


@pytest.mark.parametrize("B,G", COLUMNS)
def test_prefix_largest_scales(dev, B, G):
    """A scale that is finite, but not with the 2^24 that a form's codes carry."""
    print_case("prefix largest scales", B, G)
    g = rng(B, G)
    p = pool(g, 333, [0, 7, 40] + [3] * (B - 3), 1, 64, 16, True).upload()
    q = queries(g, B, G, 64)
    near = host(call(p, dev_(q), G, 0.125))
    p.ks *= np.float32(2.0 ** -112)
    p.upload()
    far = host(call(p, dev_(q), G, 2.0 ** 109))
    assert np.array_equal(near.view(np.uint16), far.view(np.uint16))
