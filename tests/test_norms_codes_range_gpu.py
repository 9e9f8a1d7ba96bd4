"""GPU parity of the codes of the norms between two blocks where h times its norm's weights
leaves fp32's range though the normed row does not, against numpy in float64.  Tolerances
as test_layer_i8_gpu's, and half a step of fp32's subnormal numbers for scales that small
(2^-150)."""
import numpy as np
import pytest

from gpu_util import print_case
from test_layer_i8_gpu import U, norms_call, norms_ref, stored
from test_serving_gpu import host, rng

pytestmark = pytest.mark.gpu


def close(codes, scales, y, ty):
    top, at = np.abs(y).max(1), np.abs(y).argmax(1)
    s = scales.astype(np.float64)
    ts = np.maximum(ty.max(1), ty[np.arange(len(y)), at]) / 127 + 4 * U * top / 127 + 2.0 ** -150
    assert np.all(np.abs(s - top / 127) <= ts)
    # (the codes are those of top / 127 itself, whatever the stored scale's rounding was)
    got = codes.astype(np.float64) * (top / 127)[:, None]
    assert np.all(np.abs(got - y) <= 0.5 * (top / 127)[:, None] * (1 + 8 * U) + ty + 127 * (ty.max(1)[:, None] / 127 + 4 * U * top[:, None] / 127))
    assert np.all(np.abs(codes.astype(int)).max(1) == 127)


@pytest.mark.parametrize("rows,H", [(5, 64), (5, 2560), (600, 6000), (4, 8192), (3, 9728), (2, 28672)])
@pytest.mark.parametrize("weight,rest", [(100, (0, 40, 55, -40)), (-100, (0, -50, -30, -45)), (-60, (-40, -55, 0, 50)), (120, (20, -10, 4, 0)),
                                         (-118, (0, -20, -45, 30))])
def test_norms_codes_of_far_weights(dev, rows, H, weight, rest):
    """Norm weights about 2^weight on rows about 2^rest: products from 2^-163 to 2^155, rows y of
    2^weight throughout."""
    print_case("norms far weights", rows, H, weight)
    g = rng(rows, H, weight + 200)
    i = dict(x=np.zeros((rows, H), np.float16), post=None, gate=None,
             r=(g.standard_normal((rows, H)) * 2.0 ** np.resize(rest, rows)[:, None]).astype(np.float32),
             pre=((1 + 0.3 * g.standard_normal(H)) * 2.0 ** weight).astype(np.float32))
    o = {k: host(v) for k, v in norms_call(i, True, eps=0.0, y=False, codes=True).items()}
    h, y, E, ty = norms_ref(i, eps=0.0)
    stored(o["h"], h, E, True)
    close(o["codes"], o["scales"][:rows], y, ty)
    assert np.all(o["scales"][rows:] == 9)


@pytest.mark.parametrize("H", [64, 2560, 9728])
def test_norms_codes_rows_beyond_fp32(dev, H):
    """Rows whose y itself passes fp32 have codes 0 and the scale NaN, as rows of infinities and
    NaN have; rows of zeros under an eps codes and scale 0."""
    g = rng(H)
    i = dict(x=np.zeros((4, H), np.float16), post=None, gate=None, r=g.standard_normal((4, H)).astype(np.float32),
             pre=np.full(H, 2.0 ** 100, np.float32))
    i["r"][0] = 0
    i["r"][1, 5] = np.inf
    i["r"][2, 7] = np.nan
    o = {k: host(v) for k, v in norms_call(i, True, eps=1e-6, y=False, codes=True).items()}
    assert not o["codes"][:3].any() and o["scales"][0] == 0 and np.isnan(o["scales"][1:3]).all()
    h, y, E, ty = norms_ref({k: v if v is None or k == "pre" else v[3:] for k, v in i.items()}, eps=1e-6)
    close(o["codes"][3:], o["scales"][3:4], y, ty)
    i["pre"][:] = 2.0 ** 127
    i["r"][3, 3] = 100 * H
    o = {k: host(v) for k, v in norms_call(i, True, eps=1e-6, y=False, codes=True).items()}
    assert not o["codes"].any() and o["scales"][0] == 0 and np.isnan(o["scales"][1:4]).all()
