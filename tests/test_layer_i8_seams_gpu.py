"""Where the operators of a layer with 8-bit projections hand over: the codes of the
attention's output and of the activation against what they were made of, the activation
against its products, and the K and V rows that the front stored against the projection,
each against numpy in float64.

Tolerances: codes and scales as test_layer_i8_gpu's codes_close from exact inputs (a scale
is the largest magnitude over 127 with two roundings, a code's product three).  The
activation: exp, quotient and product within 16 u of |silu(g) u|, then fp16's rounding.  Stored
rows as test_serving_gpu's check_front."""
import numpy as np
import pytest

import jllm  # noqa: F401
from gpu_util import print_case
from test_layer_i8_gpu import codes_close
from test_layer_i8_run_gpu import D, EPS, H, HD, KV, PAGE, THETA, Batch
from test_serving_gpu import U, fp16_close, front_ref, host, rng

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("P,lens", [(70, [3, 0, 17, -1, 40]), (300, [5] * 20)])
def test_layer_seams(dev, int8, P, lens):
    print_case("layer seams", int8, P, len(lens))
    b = Batch(rng(P, len(lens), 3), P, lens, int8)
    B = len(lens)
    for _ in range(2):
        pages = [host(t).copy() for t in (b.kp, b.vp, b.ks, b.vs)]
        b.step()
        att, act, gate, up = (host(t).astype(np.float64) for t in (b.att, b.act, b.gate, b.up))
        for y, name in ((att, "att"), (act, "act")):
            codes, scales = (host(t) for t in b.c[name])
            codes_close(codes, scales, y, 4 * U * np.abs(y))
            zero = np.abs(y).max(1) == 0
            assert not codes[zero].any() and not scales[zero].any()
        want = gate / (1 + np.exp(-gate)) * up
        assert np.all(np.abs(act - want) <= 16 * U * np.abs(want) + 2.0 ** -11 * np.abs(want) + 2.0 ** -25)
        # the step's K and V rows: in their slots, and nowhere else
        qkv, pos, slots = host(b.qkv).astype(np.float64), host(b.pos), host(b.slots)
        live = slots >= 0
        assert np.array_equal(live, np.array(lens) >= 0)
        assert np.array_equal(pos[live], P + host(b.own)[live] - 1)
        k = front_ref(qkv[:, H * HD:(H + KV) * HD].reshape(B, KV, HD), b.kn.astype(np.float64), pos, THETA, True, EPS)
        v = qkv[:, (H + KV) * HD:].reshape(B, KV, HD)
        table, own = host(b.table), host(b.own)
        at = own[live] - 1
        assert np.array_equal(slots[live], table[1:][live, at // PAGE] * PAGE + at % PAGE)
        for pool, scale, before, sbefore, w64 in ((b.kp, b.ks, pages[0], pages[2], k), (b.vp, b.vs, pages[1], pages[3], v)):
            got, sc = host(pool).reshape(-1, KV, HD), host(scale).reshape(-1, KV)
            other = np.ones(len(got), bool)
            other[slots[live]] = False
            assert np.array_equal(got[other].view(np.uint8), before.reshape(got.shape)[other].view(np.uint8))
            assert np.array_equal(sc[other].view(np.uint8), sbefore.reshape(sc.shape)[other].view(np.uint8))
            rows, w = got[slots[live]], w64[live]
            top = np.abs(w).max(-1, keepdims=True)
            if int8:
                step = sc[slots[live]][..., None].astype(np.float64)
                assert np.all(np.abs(step - top / 127) <= 40 * U * top)
                assert np.all(np.abs(rows * step - w) <= (0.5 + 127 * 40 * U) * step + 32 * U * top)
            else:
                assert fp16_close(rows, w, top)
    assert b.x.shape == (B, D)
