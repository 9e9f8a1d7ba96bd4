"""GPU checks of the batched serving operators where values are extreme: INT8
scales that are zero, subnormal or NaN under scores far from zero, values that
cancel.  References and tolerances are those of test_serving_gpu where none is given.
"""
import numpy as np
import pytest
import torch

import jllm
from gpu_util import print_case
from test_serving_gpu import Pool, attn_call, attn_check, attn_ref, check_front, dev_, host, rng, run_front

pytestmark = pytest.mark.gpu


def far_pool(g, lens, KV, hd, sign, zero, tiny=0.0):
    """INT8 sequences whose scores under q = 1, scale 1 / 8 all lie near 150 * sign;
    the V scales where zero(b, t) holds are `tiny`."""
    p = Pool(g, lens, KV, hd, 16, True)
    for b, n in enumerate(lens):
        pg, off = p.table[b][np.arange(n) // 16], np.arange(n) % 16
        k = np.full((n, KV, hd), 100 * sign, np.int8)
        k[:, :, 0] += g.integers(-9, 10, (n, KV)).astype(np.int8)
        ks = np.full((n, KV), 150.0 * 8 / 100 / hd, np.float32)
        p.kp[pg, off, :, :hd], p.ks[pg, off] = k, ks
        gone = np.array([zero(b, t) for t in range(n)], bool)
        p.vs[pg[gone], off[gone]] = tiny
        p.k[b] = k * ks[..., None].astype(np.float64)
        p.v[b] = p.vp[pg, off, :, :hd] * p.vs[pg, off][..., None].astype(np.float64)
    return p.upload()


ZERO = {
    "all": lambda b, t: True,
    "one tile": lambda b, t: 32 <= t < 64,             # of one wave, whole and cut
    "one wave": lambda b, t: t // 32 % 4 == 1,
    "one part": lambda b, t: 128 <= t < 256,
    "but one key": lambda b, t: t != 40,
    "half": lambda b, t: (t * 7919 >> 3) % 2 == 0,
}


@pytest.mark.parametrize("which", list(ZERO))
@pytest.mark.parametrize("sign", [-1, 1])
@pytest.mark.parametrize("lens", [[1, 64, 300, 41], [3000, 1, 0, 130, 700]])
def test_attention_value_scales_of_zero(dev, which, sign, lens):
    """Keys whose V scale is 0, as the front stores a zero V row, take part in the
    softmax and add nothing, however far from zero the scores are.  (Scores: integer
    sums, exact; four roundings after, 4 u * 150 * log2(e) < 2^-14 in a weight.)"""
    print_case("zero V scales", which, sign, lens)
    H, KV, hd = 8, 2, 64
    p = far_pool(rng(len(lens), sign + 1), lens, KV, hd, sign, ZERO[which])
    q = np.ones((len(lens), H * hd), np.float16)
    attn_check(p, host(attn_call(p, dev_(q), H, 0.125)), q, H, 0.125)


@pytest.mark.parametrize("lens", [[1, 64, 300], [3000, 5]])
def test_attention_value_scales_below_the_normal_range(dev, lens):
    """A scale of 1e-39 times a code is below every fp16: the key adds nothing."""
    H, KV, hd = 8, 2, 64
    p = far_pool(rng(len(lens), 5), lens, KV, hd, -1, ZERO["one wave"], tiny=1e-39)
    q = np.ones((len(lens), H * hd), np.float16)
    attn_check(p, host(attn_call(p, dev_(q), H, 0.125)), q, H, 0.125)


@pytest.mark.parametrize("lens", [[1, 64, 300], [3000, 5]])
@pytest.mark.parametrize("which", ["ks", "vs"])
def test_attention_nan_scales_of_live_keys(dev, which, lens):
    """A row stored from NaN or infinite values has a NaN scale: the heads of its KV
    head are NaN, the others are as they were; beside zero V scales too."""
    H, KV, hd = 8, 2, 64
    p = far_pool(rng(len(lens), 6), lens, KV, hd, -1, ZERO["one wave"])
    b, t = len(lens) - 1, lens[-1] - 1
    getattr(p, which)[p.table[b, t // 16], t % 16, 1] = np.nan
    p.upload()
    q = np.ones((len(lens), H * hd), np.float16)
    got = host(attn_call(p, dev_(q), H, 0.125)).reshape(len(lens), H, hd)
    bad = np.zeros((len(lens), H), bool)
    bad[b, H // 2:] = True
    assert np.isnan(got[bad]).all() and np.isfinite(got[~bad]).all()


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("H,KV,hd", [(8, 2, 64), (32, 8, 128), (12, 1, 96), (4, 4, 32)])
@pytest.mark.parametrize("lens", [[2, 3, 40, 300], [2, 700, 3000, 9]])
def test_attention_weights_keep_more_than_fp16(dev, int8, H, KV, hd, lens):
    """Values that nearly cancel: up to eight keys of a row have almost the same
    weight and values of either sign, the others values of 0 and weights below 2^-28,
    so the output is a small difference that weights of 11 bits do not have.

    Error of a weight: 2^-21 where it is held in two fp16 parts, 2^-22 for exp2,
    2^-21 for the exponent (int8: |log2| < 8 of a V scale, itself 1 ulp); of the sums
    of 8 terms, 4 joins and the matrix cores' steps 24 u < 2^-19.4; together below
    2^-18 of sum w |v|.  INT8 sums codes + 128, up to 255 / 64 of the values that count, so
    four times that, 2^-16.  Two weights rounded to fp16 are off by up to 2^-12."""
    print_case("weights", int8, H, KV, hd, lens)
    g = rng(H, KV, hd, len(lens), lens[1])
    p = Pool(g, lens, KV, hd, 16, int8)
    for b, n in enumerate(lens):
        pg, off = p.table[b][np.arange(n) // 16], np.arange(n) % 16
        live = g.permutation(n)[:min(n, 8)]
        live = live[:len(live) // 2 * 2] if n > 2 else live
        # q has one 1 per head, in d = 0: scores are k[0], within 2^-6 of each other
        if int8:
            k, v = np.zeros((n, KV, hd), np.int8), np.zeros((n, KV, hd), np.int8)
            ks = np.full((n, KV), 0.25, np.float32)
            vs = np.full((n, KV), 0.01, np.float32)
            k[:, :, 0] = -100
            k[live, :, 0] = 100
            ks[live] = 0.01 * (1 + 2.0 ** -7 * g.random((len(live), KV)))
            v[live] = g.integers(100, 128, (1, KV, hd)).astype(np.int8)
            v[live[::2]] *= -1
            p.ks[pg, off], p.vs[pg, off] = ks, vs
            p.k[b], p.v[b] = k * ks[..., None].astype(np.float64), v * vs[..., None].astype(np.float64)
        else:
            k, v = np.zeros((n, KV, hd), np.float16), np.zeros((n, KV, hd), np.float16)
            k[:, :, 0] = -24
            k[live, :, 0] = 2.0 ** -7 * g.random((len(live), KV))
            v[live] = 1 + g.random((1, KV, hd))
            v[live[::2]] *= -1
            p.k[b], p.v[b] = k.astype(np.float64), v.astype(np.float64)
        p.kp[pg, off, :, :hd], p.vp[pg, off, :, :hd] = k, v
    p.upload()
    q = np.zeros((len(lens), H, hd), np.float16)
    q[..., 0] = 1.0
    q = q.reshape(len(lens), -1)
    got = host(attn_call(p, dev_(q), H, 1.0)).reshape(-1, H, hd).astype(np.float64)
    for b, n in enumerate(lens):
        want, size = attn_ref(q[b].reshape(H, hd).astype(np.float64), p.k[b], p.v[b], 1.0, 0, n)
        tol = 2.0 ** -11 * np.abs(want) + 2.0 ** (-16 if int8 else -18) * size + 2.0 ** -25
        err = np.abs(got[b] - want)
        assert np.all(err <= tol), (b, n, float((err / tol).max()))


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("norm", ["f32", "f16"])
@pytest.mark.parametrize("eps", [1e-40, 1.4e-45, 1.2e-38])
def test_front_eps_below_the_normal_range(dev, int8, norm, eps):
    """An eps that is subnormal is an eps: rows of zeros stay zero, the others are
    normed as if it were not there."""
    H, KV, hd = 4, 2, 64
    x = rng(8).standard_normal((4, (H + 2 * KV) * hd)).astype(np.float16)
    x[1] = 0
    x[2] = 6e-8                    # the smallest fp16
    r = run_front(rng(9), 4, H, KV, hd, int8=int8, x=x, norm=norm, eps=eps)
    check_front(*r, H, hd, int8)


# lengths of the rows at each step: over a unit's and a part's border, from several
# pieces to one and to none and back, all short, all empty, all at max_seq
STEPS = [[3000, 1, 0, 700, 5999, 127, 2000, 33],
         [3001, 2, 1, 701, 6000, 128, 2001, 34],
         [3002, 3, 0, 640, 12, 129, 0, 35],
         [40, 6000, 5, 0, 0, 256, 6000, 1],
         [0, 0, 0, 0, 0, 0, 0, 0],
         [1, 0, 33, 7, 2, 100, 3, 129],
         [6000, 6000, 6000, 6000, 6000, 6000, 6000, 6000],
         [7000, 1, -5, 700, 5999, 127, 2000, 33]]       # (above max_seq: max_seq; below 0: empty)


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("short", [0, 62])
def test_attention_captured_while_lengths_change(dev, int8, short):
    """One captured call that cuts its rows, replayed while the lengths change in
    place, its workspace holding the pieces of the steps before; and the same calls
    eagerly on another such workspace.  Eager work and synchronizations between."""
    print_case("captured parts", int8, short)
    H, KV, hd, most = 8, 2, 64, 6000
    B = len(STEPS[0]) + short
    g = rng(90, short, int8)
    p = Pool(g, [most] * len(STEPS[0]) + [40] * short, KV, hd, 32, int8, max_seq=most).upload()
    q = (g.standard_normal((B, H * hd)) * 1.2).astype(np.float16)
    Q, out = dev_(q), torch.full((B, H * hd), 7.0, dtype=torch.float16, device="cuda:0")
    need = jllm.lib().jllm_hip_flash_attention_decode_paged_workspace(B, H, KV, hd, most, 0)
    assert need > 0                                     # rows are cut
    ws, ws2 = [torch.full((need,), 0xFF, dtype=torch.uint8, device="cuda:0") for _ in range(2)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        attn_call(p, Q, H, 0.125, out=out, ws=ws)       # warm-up outside the capture
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        attn_call(p, Q, H, 0.125, out=out, ws=ws)
    for i, step in enumerate(STEPS + STEPS[::-1]):
        lens = step + [(i + j) % 41 for j in range(short)]
        p.d[5].copy_(dev_(np.array(lens, np.int32)))
        out.fill_(7.0)
        gr.replay()
        got = host(out).copy()
        attn_check(p, got, q, H, 0.125, lens=[min(n, most) for n in lens])
        torch.ones(1000, device="cuda:0").cumsum(0)
        eager = host(attn_call(p, Q, H, 0.125, ws=ws2))
        assert np.array_equal(got.view(np.uint16), eager.view(np.uint16)), i


@pytest.mark.parametrize("lens", [[1, 2, 40, 300], [3000, 1, 17]])
@pytest.mark.parametrize("bad", [np.inf, -np.inf])
def test_attention_infinite_values_of_any_weight(dev, bad, lens):
    """An infinite V value of a key that has a weight makes its own dimension
    infinite, whatever the weight (1, equal shares, 2^-30 of the others), and no other."""
    print_case("infinite values", bad, lens)
    H, KV, hd = 8, 2, 64
    for s_low in (0.0, -20.0):                    # the key's score; the others' are 0
        p = Pool(rng(len(lens), 70), lens, KV, hd, 16, False)
        for b, n in enumerate(lens):
            pg, off = p.table[b][np.arange(n) // 16], np.arange(n) % 16
            p.kp[pg, off, :, :hd] = 0
            t = n // 2
            p.kp[pg[t], off[t], :, 0] = s_low
            p.vp[pg[t], off[t], 1, 5] = bad
        p.upload()
        q = np.zeros((len(lens), H, hd), np.float16)
        q[..., 0] = 1
        got = host(attn_call(p, dev_(q.reshape(len(lens), -1)), H, 1.0)).reshape(-1, H, hd)
        want = np.zeros(got.shape, bool)
        want[:, H // 2:, 5] = True
        assert np.all(got[want] == bad) and np.isfinite(got[~want]).all()
