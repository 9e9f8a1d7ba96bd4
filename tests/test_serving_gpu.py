"""GPU parity of the batched serving operators (paged attention front, paged
decode attention, logits processing) against numpy in float64.

Tolerances, from the arithmetic (u = 2^-24, one fp32 rounding):

* front, fp16 results: fp32 throughout (sum of squares of hd <= 128 values, root,
  quotient, two products: <= 24 u; rotation: products and sum 3 u, sine and
  cosine 2 u, angle 2 u), at most 32 u of the row's largest value, then one
  fp16 rounding: 2^-11 of the value, 2^-25 among subnormals.
* front, int8: scale within 40 u; code times scale within half a step plus the
  row's fp32 error.
* attention: scores of |s| <= 34 summed over 128 products of magnitude <= 34 in
  total: 128 * 34 * u = 2^-12 absolute, so relative in each weight and in their sum;
  weights may be rounded to fp16, 2^-11; so (2^-11 + 2 * 2^-12) A with A = sum w |v|,
  then the output's own rounding 2^-11 |out| + 2^-25.
* logits: the same fp32 operations in the same order, so the same bits.
"""
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import jllm
from gpu_util import print_case

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def rng(*key):
    return np.random.default_rng(list(key))


def dev_(a):
    return None if a is None else torch.from_numpy(np.ascontiguousarray(a)).to("cuda:0")


def host(t):
    torch.cuda.synchronize()
    return t.cpu().numpy()


# ---- front --------------------------------------------------------------------------

def front_ref(x, w, pos, theta, neox, eps):
    """x [N][heads][hd] float64 -> normed and rotated."""
    hd = x.shape[-1]
    if w is not None:
        x = x / np.sqrt((x ** 2).mean(-1, keepdims=True) + eps) * w
    ang = (pos.astype(np.float64)[:, None] * float(np.float32(theta)) ** (-np.arange(0, hd, 2) / hd))[:, None]
    c, s = np.cos(ang), np.sin(ang)
    y = np.empty_like(x)
    a, b = (x[..., :hd // 2], x[..., hd // 2:]) if neox else (x[..., 0::2], x[..., 1::2])
    u, v = a * c - b * s, a * s + b * c
    if neox:
        y[..., :hd // 2], y[..., hd // 2:] = u, v
    else:
        y[..., 0::2], y[..., 1::2] = u, v
    return y


def fp16_close(got, want, size):
    """got fp16 of a value computed in fp32 to 32 u of `size`."""
    tol = 32 * U * size + 2.0 ** -11 * np.abs(want) + 2.0 ** -25
    return np.all(np.abs(got.astype(np.float64) - want) <= tol)


def run_front(g, N, H, KV, hd, chd=None, int8=False, neox=True, norm="f32", fused=False, n_slots=None, slots=None,
              pos=None, in_place=False, theta=1e6, eps=1e-6, x=None):
    chd = chd or hd
    W = (H + 2 * KV) * hd
    if x is None:
        x = (g.standard_normal((N, W)) * 1.5).astype(np.float16)
    n_slots = n_slots or N + 5
    slots = g.permutation(n_slots)[:N].astype(np.int32) if slots is None else np.asarray(slots, np.int32)
    pos = g.integers(0, 40000, N).astype(np.int32) if pos is None else np.asarray(pos, np.int32)
    qw = kw = None
    if norm:
        t = np.float32 if norm == "f32" else np.float16
        qw, kw = [(1 + 0.3 * g.standard_normal(hd)).astype(t) for _ in range(2)]
    X = dev_(x)
    q, k, v = X.split([H * hd, KV * hd, KV * hd], dim=1)
    if not fused:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    out = q if in_place else torch.full((N, H * hd + 4), 7.0, dtype=torch.float16, device="cuda:0")
    kind = torch.int8 if int8 else torch.float16
    kp, vp = [torch.full((n_slots, KV, chd), 9, dtype=kind, device="cuda:0") for _ in range(2)]
    ks, vs = [torch.full((n_slots, KV), 9.0, device="cuda:0") for _ in range(2)]
    jllm.call("jllm_hip_qk_norm_rope_store_kv_paged", out, out.stride(0), q, q.stride(0), k, k.stride(0), v,
              v.stride(0), dev_(qw), dev_(kw), int(norm == "f32"), eps, kp, vp, ks if int8 else None,
              vs if int8 else None, n_slots, dev_(pos), dev_(slots), H, KV, hd, chd, N, theta, int(neox), int(int8))
    res = [host(t) for t in (out, kp, vp, ks, vs)]
    xs = x.astype(np.float64)
    q64 = front_ref(xs[:, :H * hd].reshape(N, H, hd), None if qw is None else qw.astype(np.float64), pos, theta, neox, eps)
    k64 = front_ref(xs[:, H * hd:(H + KV) * hd].reshape(N, KV, hd), None if kw is None else kw.astype(np.float64), pos,
                    theta, neox, eps)
    v64 = xs[:, (H + KV) * hd:].reshape(N, KV, hd)
    return res, (q64, k64, v64), slots, n_slots, x


def check_front(res, want, slots, n_slots, x, H, hd, int8, in_place=False):
    out, kp, vp, ks, vs = res
    q64, k64, v64 = want
    N = len(slots)
    live = (slots >= 0) & (slots < n_slots)
    got = out[:, :H * hd].reshape(N, H, hd)
    size = np.abs(q64).max(-1, keepdims=True)
    assert fp16_close(got[live], q64[live], size[live])
    before = x[:, :H * hd].reshape(N, H, hd) if in_place else np.float16(7.0)
    assert np.array_equal(got[~live], np.broadcast_to(before, got.shape)[~live])
    if not in_place:
        assert np.all(out[:, H * hd:] == 7.0)
    at = slots[live]
    other = np.ones(n_slots, bool)
    other[at] = False
    for pool, sc, w64 in ((kp, ks, k64), (vp, vs, v64)):
        assert np.all(pool[other] == 9) and np.all(pool[..., hd:] == 9) and np.all(sc[other] == 9.0)
        rows, w = pool[at][..., :hd], w64[live]
        top = np.abs(w).max(-1, keepdims=True)
        if int8:
            step = sc[at][..., None].astype(np.float64)
            assert np.all(np.abs(step - top / 127) <= 40 * U * top)
            assert np.all(np.abs(rows * step - w) <= (0.5 + 127 * 40 * U) * step + 32 * U * top)
            assert np.all(np.abs(rows).max(-1)[top[..., 0] > 0] == 127)
        else:
            assert fp16_close(rows, w, top)


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("N,H,KV,hd,chd,neox,norm,fused", [
    (1, 32, 8, 128, 128, True, "f32", False), (1, 1, 1, 8, 16, True, "f16", False), (3, 5, 3, 24, 32, False, "f32", True),
    (7, 4, 1, 32, 32, True, None, True), (33, 8, 2, 64, 64, False, None, False), (65, 12, 1, 96, 96, True, "f16", True),
    (129, 16, 2, 128, 160, True, "f32", True), (5, 3, 2, 40, 48, True, "f32", False), (2, 7, 7, 72, 80, False, "f16", True),
    (1000, 32, 8, 128, 128, False, "f32", True), (3001, 2, 1, 64, 64, True, "f32", False)])
def test_front(dev, int8, N, H, KV, hd, chd, neox, norm, fused):
    print_case("front", int8, N, H, KV, hd, chd, neox, norm, fused)
    r = run_front(rng(N, H, hd), N, H, KV, hd, chd, int8, neox, norm, fused)
    check_front(*r, H, hd, int8)


@pytest.mark.parametrize("int8", [False, True])
def test_front_padding_and_bad_slots(dev, int8):
    slots = [3, -1, 0, 20, 19, -2 ** 31, 2 ** 31 - 1, 7, 21]
    r = run_front(rng(4), 9, 8, 2, 128, int8=int8, fused=True, n_slots=20, slots=slots)
    check_front(*r, 8, 128, int8)


def test_front_nothing_but_padding(dev):
    r = run_front(rng(5), 4, 8, 2, 128, n_slots=20, slots=[-1] * 4)
    check_front(*r, 8, 128, False)


@pytest.mark.parametrize("neox", [False, True])
@pytest.mark.parametrize("theta", [1e4, 5e5, 1.5, 1.0, 0.75])
def test_front_far_positions(dev, neox, theta):
    pos = [0, 1, 131071, 1 << 20, (1 << 24) + 1, 2 ** 31 - 1, -1, -2 ** 31]
    r = run_front(rng(6), len(pos), 4, 2, 128, neox=neox, pos=pos, theta=theta)
    check_front(*r, 4, 128, False)


@pytest.mark.parametrize("fused", [False, True])
def test_front_in_place(dev, fused):
    r = run_front(rng(7), 9, 8, 2, 64, fused=fused, in_place=True, n_slots=12, slots=[0, 1, 2, -1, 4, 5, 6, 12, 8])
    check_front(*r, 8, 64, False, in_place=True)


@pytest.mark.parametrize("int8", [False, True])
def test_front_zero_and_tiny_rows(dev, int8):
    H, KV, hd = 4, 2, 64
    x = np.zeros((4, (H + 2 * KV) * hd), np.float16)
    x[1] = 6e-8                    # the smallest fp16
    x[2, ::hd] = 60000.0
    x[3, 5] = 1.0
    r = run_front(rng(8), 4, H, KV, hd, int8=int8, x=x, norm=None)
    check_front(*r, H, hd, int8)
    r = run_front(rng(8), 4, H, KV, hd, int8=int8, x=x, norm="f32")
    check_front(*r, H, hd, int8)


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_front_nonfinite_int8_rows_read_as_nan(dev, bad):
    H, KV, hd = 2, 2, 128
    x = rng(9).standard_normal((3, (H + 2 * KV) * hd)).astype(np.float16)
    x[1, H * hd + 5] = bad                       # k, head 0
    x[2, (H + KV) * hd + hd + 77] = bad          # v, head 1
    (out, kp, vp, ks, vs), want, slots, n, _ = run_front(rng(9), 3, H, KV, hd, int8=True, x=x, norm=None)
    nk, nv = np.zeros((3, KV), bool), np.zeros((3, KV), bool)
    nk[1, 0] = nv[2, 1] = True
    assert np.array_equal(np.isnan(ks[slots]), nk) and np.array_equal(np.isnan(vs[slots]), nv)
    assert not kp[slots][nk].any() and not vp[slots][nv].any()


def test_front_agrees_with_the_contiguous_front(dev):
    """At near positions the contiguous front's values, up to its intermediate
    fp16 roundings: norm 2^-11, rotation 2^-11 of the pair, angle p * 2^-24."""
    H, KV, hd, N = 32, 8, 128, 50
    g = rng(10)
    x = (g.standard_normal((N, (H + 2 * KV) * hd)) * 1.5).astype(np.float16)
    (out, kp, vp, _, _), _, slots, n, _ = run_front(rng(10, 1), N, H, KV, hd, x=x, norm=None, n_slots=N,
                                                     slots=np.arange(N), pos=np.arange(100, 100 + N))
    q, k, v = [dev_(np.ascontiguousarray(a)) for a in np.split(x, [H * hd, (H + KV) * hd], 1)]
    kc, vc = [torch.zeros((N, KV, hd), dtype=torch.float16, device="cuda:0") for _ in range(2)]
    jllm.call("jllm_hip_qk_norm_rope_store_kv", q, k, v, None, None, 1, 1e-6, kc, vc, None, None, KV * hd, H, KV, hd,
              hd, 100, N, 1e6, 1, 0)
    assert np.array_equal(vp, host(vc))
    for a, b in ((out[:, :H * hd], host(q)), (kp.reshape(N, -1), host(kc).reshape(N, -1))):
        a, b = a.astype(np.float64), b.astype(np.float64)
        assert np.all(np.abs(a - b) <= 2.0 ** -10 * np.abs(b) + 8 * 200 * U + 2.0 ** -24)


def test_front_values_get_the_codes_of_the_kv_quantiser(dev):
    """V rows: the codes and scales of fp16_to_int8, bit for bit."""
    H, KV, hd, N = 4, 8, 128, 300
    g = rng(11)
    x = (g.standard_normal((N, (H + 2 * KV) * hd)) * np.exp(g.standard_normal((N, 1)) * 3)).astype(np.float16)
    (_, _, vp, _, vs), _, slots, _, _ = run_front(rng(11, 1), N, H, KV, hd, int8=True, x=x)
    codes = torch.zeros((N * KV, hd), dtype=torch.int8, device="cuda:0")
    scales = torch.zeros((N * KV,), device="cuda:0")
    jllm.call("jllm_hip_fp16_to_int8", codes, scales, dev_(x[:, (H + KV) * hd:]), N * KV, hd)
    assert np.array_equal(vp[slots].reshape(-1, hd), host(codes))
    assert np.array_equal(vs[slots].reshape(-1), host(scales))


# ---- attention ----------------------------------------------------------------------

class Pool:
    """Sequences of the given lengths on random pages; everything else poisoned."""

    def __init__(self, g, lens, KV, hd, page, int8, chd=None, max_seq=None, amp=1.0, poison=True):
        chd = chd or hd
        self.lens, self.page, self.KV, self.hd, self.int8, self.chd = list(lens), page, KV, hd, int8, chd
        self.max_seq = max(self.lens + [0]) if max_seq is None else max_seq
        used = [(max(n, 0) + page - 1) // page for n in self.lens]
        self.n_pages = sum(used) + 2
        ids = g.permutation(self.n_pages)[:sum(used)]
        width = max((self.max_seq + page - 1) // page, 1)
        self.table = np.full((len(lens), width), -7, np.int32)
        shape = (self.n_pages, page, KV, chd)
        if int8:
            self.kp = np.full(shape, 127, np.int8)
            self.vp = np.full(shape, 127, np.int8)
        else:
            bad = np.nan if poison else 1.0
            self.kp = np.full(shape, bad, np.float16)
            self.vp = np.full(shape, bad, np.float16)
            self.vp[::2] = np.inf
        self.ks = np.full(shape[:3], np.nan, np.float32)
        self.vs = np.full(shape[:3], np.nan, np.float32)
        self.k, self.v = [], []
        at = 0
        for b, n in enumerate(self.lens):
            n = max(n, 0)
            mine = ids[at:at + used[b]]
            at += used[b]
            m = min(used[b], width)
            self.table[b, :m] = mine[:m]
            pg, off = mine[np.arange(n) // page], np.arange(n) % page
            if int8:
                k, v = [g.integers(-127, 128, (n, KV, hd)).astype(np.int8) for _ in range(2)]
                ks, vs = [(g.random((n, KV)) * 0.02 + 0.005).astype(np.float32) * amp for _ in range(2)]
                self.ks[pg, off], self.vs[pg, off] = ks, vs
                k64, v64 = k * ks[..., None].astype(np.float64), v * vs[..., None].astype(np.float64)
            else:
                k, v = [(g.standard_normal((n, KV, hd)) * amp).astype(np.float16) for _ in range(2)]
                k64, v64 = k.astype(np.float64), v.astype(np.float64)
            self.kp[pg, off, :, :hd], self.vp[pg, off, :, :hd] = k, v
            self.k.append(k64)
            self.v.append(v64)

    def upload(self):
        self.d = [dev_(a) for a in (self.kp, self.vp, self.ks, self.vs, self.table, np.array(self.lens, np.int32))]
        return self


def attn_ref(q, k, v, scale, lo, n):
    """(out, A): float64 attention of one row's q [H][hd] over k, v [n][KV][hd]."""
    H, KV = q.shape[0], k.shape[1]
    out = np.zeros(q.shape)
    size = np.zeros(q.shape)
    if n > lo:
        for h in range(H):
            kk, vv = k[lo:n, h // (H // KV)], v[lo:n, h // (H // KV)]
            s = kk @ q[h] * scale
            e = np.exp(s - s.max())
            w = e / e.sum()
            out[h], size[h] = w @ vv, w @ np.abs(vv)
    return out, size


def attn_call(p, q, H, scale, window=0, max_seq=None, stream=None, out=None, ws=None, q_stride=None):
    B = len(p.lens)
    max_seq = p.max_seq if max_seq is None else max_seq
    out = torch.full((B, H * p.hd), 7.0, dtype=torch.float16, device="cuda:0") if out is None else out
    if ws is None:
        need = jllm.lib().jllm_hip_flash_attention_decode_paged_workspace(B, H, p.KV, p.hd, max_seq, window)
        assert need >= 0
        ws = torch.full((max(need, 16),), 0xFF, dtype=torch.uint8, device="cuda:0")     # any content: NaNs here
    kp, vp, ks, vs, table, lens = p.d
    jllm.call("jllm_hip_flash_attention_decode_paged", out, q, q.stride(0) if q_stride is None else q_stride, kp, vp,
              ks if p.int8 else None, vs if p.int8 else None, p.n_pages, p.page, table, table.stride(0), lens, B, H,
              p.KV, p.hd, p.chd, max_seq, scale, int(p.int8), window, ws, ws.numel(), stream=stream)
    return out


def attn_check(p, got, q, H, scale, window=0, lens=None):
    got = got.reshape(-1, H, p.hd).astype(np.float64)
    for b, n in enumerate(lens or p.lens):
        n = max(n, 0)
        lo = max(0, n - window) if window else 0
        want, size = attn_ref(q[b].reshape(H, p.hd).astype(np.float64), p.k[b], p.v[b], scale, lo, n)
        tol = 2.0 ** -11 * np.abs(want) + 2.0 ** -10 * size + 2.0 ** -25
        err = np.abs(got[b] - want)
        assert np.all(err <= tol), (b, n, float((err / tol).max()))


HEADS = [(32, 8, 128, 128), (16, 1, 128, 128), (7, 7, 32, 32), (12, 1, 96, 112), (10, 2, 64, 64), (16, 2, 128, 160)]


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("H,KV,hd,chd", HEADS)
def test_attention(dev, int8, page, H, KV, hd, chd):
    print_case("paged attn", int8, page, H, KV, hd, chd)
    g = rng(H, KV, hd, page)
    lens = [1, 0, 15, 16, 17, 31, 32, 33, 63, 64, 65, 100, 127, 128, 129, 255, 257, 511, 513, 700]
    p = Pool(g, lens, KV, hd, page, int8, chd).upload()
    q = (g.standard_normal((len(lens), H * hd)) * 1.2).astype(np.float16)
    scale = 1 / np.sqrt(hd)
    attn_check(p, host(attn_call(p, dev_(q), H, scale)), q, H, scale)


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("lens", [[1], [700], [5000], [20000], [0], [2048, 3, 1025, 4096, 0, 1000],
                                  [300] * 70])
def test_attention_lengths(dev, int8, lens):
    print_case("paged attn lens", int8, lens[:6])
    H, KV, hd = 32, 8, 128
    g = rng(len(lens), lens[0])
    p = Pool(g, lens, KV, hd, 32, int8).upload()
    q = (g.standard_normal((len(lens), H * hd)) * 1.2).astype(np.float16)
    scale = 1 / np.sqrt(hd)
    attn_check(p, host(attn_call(p, dev_(q), H, scale)), q, H, scale)


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("window", [1, 5, 16, 31, 200, 1000, 5000])
def test_attention_window(dev, int8, window):
    print_case("paged attn window", int8, window)
    H, KV, hd = 8, 2, 64
    g = rng(window)
    lens = [3000, 1, 0, 200, 201, 17, 1234, 999, 1000, 1001]
    p = Pool(g, lens, KV, hd, 16, int8).upload()
    q = (g.standard_normal((len(lens), H * hd)) * 1.2).astype(np.float16)
    attn_check(p, host(attn_call(p, dev_(q), H, 0.125, window)), q, H, 0.125, window)


@pytest.mark.parametrize("int8", [False, True])
def test_attention_pages_in_front_of_the_window_may_be_gone(dev, int8):
    H, KV, hd, window = 8, 2, 64, 100
    g = rng(3)
    lens = [1000, 333, 90]
    p = Pool(g, lens, KV, hd, 16, int8)
    for b, n in enumerate(lens):
        p.table[b, :max(0, n - window) // 16] = -1
    p.upload()
    q = g.standard_normal((3, H * hd)).astype(np.float16)
    attn_check(p, host(attn_call(p, dev_(q), H, 0.125, window)), q, H, 0.125, window)


@pytest.mark.parametrize("int8", [False, True])
def test_attention_bad_pages_and_lengths(dev, int8):
    """Page ids outside the pool: their keys are skipped.  Negative lengths are
    empty rows, lengths above max_seq count as max_seq."""
    H, KV, hd = 8, 2, 128
    g = rng(4)
    lens = [200, 64, 300, 40]
    p = Pool(g, lens, KV, hd, 16, int8)
    for b, pages in ((0, [0, 3, 12]), (1, [0, 1, 2, 3])):
        keep = np.ones(lens[b], bool)
        for i, pg in enumerate(pages):
            p.table[b, pg] = [-1, p.n_pages, 2 ** 31 - 1, -2 ** 31][i]
            keep[16 * pg:16 * pg + 16] = False
        p.k[b], p.v[b] = p.k[b][keep], p.v[b][keep]
    p.upload()
    p.d[5] = dev_(np.array([200, 64, 1000, -3], np.int32))
    q = g.standard_normal((4, H * hd)).astype(np.float16)
    got = host(attn_call(p, dev_(q), H, 0.08, max_seq=304))
    # row 2: pages 0..18 (304 keys), the last of them 4 slots behind its 300 written ones
    attn_check(p, got[:2], q, H, 0.08, lens=[len(p.k[0]), 0])
    assert not got[3].any()
    got = host(attn_call(p, dev_(q), H, 0.08, max_seq=300))
    attn_check(p, got, q, H, 0.08, lens=[len(p.k[0]), 0, 300, 0])


def test_attention_nonfinite_keys(dev):
    """A key of score -inf has no weight, a row of such keys is zero; NaN and
    +inf scores give NaN, in their own head and row only."""
    H, KV, hd = 4, 2, 64
    g = rng(5)
    lens = [40, 40, 40, 300, 40]
    p = Pool(g, lens, KV, hd, 16, False)
    q = np.abs(g.standard_normal((5, H * hd))).astype(np.float16)

    def put(b, t, kvh, val):
        p.kp[p.table[b, t // 16], t % 16, kvh, 3] = val

    put(0, 7, 0, -np.inf)
    for t in range(40):
        put(1, t, 1, -np.inf)
    put(2, 39, 0, np.nan)
    put(3, 299, 1, -np.inf)
    put(4, 0, 1, np.inf)
    p.upload()
    got = host(attn_call(p, dev_(q), H, 0.125)).reshape(5, H, hd).astype(np.float64)
    bad = np.zeros((5, H), bool)
    bad[2, :2] = bad[4, 2:] = True
    assert np.array_equal(np.isnan(got).all(-1), bad) and np.array_equal(np.isnan(got).any(-1), bad)
    assert not got[1, 2:].any()
    k, v = np.delete(p.k[0], 7, 0), np.delete(p.v[0], 7, 0)
    want, size = attn_ref(q[0].reshape(H, hd).astype(np.float64), k, v, 0.125, 0, 39)
    assert np.all(np.abs(got[0, :2] - want[:2]) <= 2.0 ** -11 * np.abs(want[:2]) + 2.0 ** -10 * size[:2] + 2.0 ** -25)
    want, size = attn_ref(q[3].reshape(H, hd).astype(np.float64), p.k[3][:299], p.v[3][:299], 0.125, 0, 299)
    assert np.all(np.abs(got[3, 2:] - want[2:]) <= 2.0 ** -11 * np.abs(want[2:]) + 2.0 ** -10 * size[2:] + 2.0 ** -25)


def test_attention_infinite_values_stay_in_their_dimension(dev):
    H, KV, hd = 4, 2, 64
    g = rng(6)
    p = Pool(g, [50, 200], KV, hd, 16, False)
    p.vp[p.table[0, 1], 4, 0, 9] = np.inf          # key 20, KV head 0, d = 9
    p.vp[p.table[1, 3], 0, 1, 63] = np.nan
    p.upload()
    q = (g.standard_normal((2, H * hd)) * 0.5).astype(np.float16)
    got = host(attn_call(p, dev_(q), H, 0.125)).reshape(2, H, hd)
    assert np.all(got[0, :2, 9] == np.inf) and np.isnan(got[1, 2:, 63]).all()
    fine = np.ones((2, H, hd), bool)
    fine[0, :2, 9] = fine[1, 2:, 63] = False
    assert np.isfinite(got[fine]).all()


@pytest.mark.parametrize("spread", [1e-6, 1e3])
def test_attention_value_scales_of_any_size(dev, spread):
    """INT8 value scales that differ by many orders of magnitude, the weight on
    the small ones as well as on the large."""
    H, KV, hd = 8, 2, 64
    g = rng(7)
    p = Pool(g, [400, 33], KV, hd, 16, True)
    for b in range(2):
        n = p.lens[b]
        f = np.where(g.random((n, KV)) < 0.5, spread, 1.0).astype(np.float32)
        pg, off = p.table[b][np.arange(n) // 16], np.arange(n) % 16
        p.vs[pg, off] *= f
        p.v[b] = p.vp[pg, off].astype(np.float64) * p.vs[pg, off][..., None]
    p.upload()
    q = g.standard_normal((2, H * hd)).astype(np.float16)
    attn_check(p, host(attn_call(p, dev_(q), H, 0.125)), q, H, 0.125)


def test_attention_scales_null_are_one(dev):
    H, KV, hd = 8, 2, 64
    g = rng(8)
    p = Pool(g, [100, 250], KV, hd, 16, True).upload()
    q = (g.standard_normal((2, H * hd)) * 0.01).astype(np.float16)
    out = torch.zeros((2, H * hd), dtype=torch.float16, device="cuda:0")
    need = jllm.lib().jllm_hip_flash_attention_decode_paged_workspace(2, H, KV, hd, 250, 0)
    ws = torch.empty((max(need, 16),), dtype=torch.uint8, device="cuda:0")
    Q = dev_(q)
    jllm.call("jllm_hip_flash_attention_decode_paged", out, Q, H * hd, p.d[0], p.d[1], None, None, p.n_pages, 16,
              p.d[4], p.d[4].stride(0), p.d[5], 2, H, KV, hd, hd, 250, 0.125, 1, 0, ws, ws.numel())
    for b, n in enumerate(p.lens):
        pg, off = p.table[b][np.arange(n) // 16], np.arange(n) % 16
        p.k[b], p.v[b] = p.kp[pg, off].astype(np.float64), p.vp[pg, off].astype(np.float64)
    attn_check(p, host(out), q, H, 0.125)


def test_attention_equal_scores_of_every_size(dev):
    """Large equal scores (softmax shift), one key far above the others, and
    all weight on the last key."""
    H, KV, hd = 4, 1, 32
    g = rng(9)
    p = Pool(g, [100, 1000, 77], KV, hd, 16, False)
    for b, n in enumerate(p.lens):
        pg, off = p.table[b][np.arange(n) // 16], np.arange(n) % 16
        k = np.full((n, KV, hd), 20.0, np.float16)
        if b:
            k[n - 1 if b == 2 else 500] = 22.0
        p.kp[pg, off], p.k[b] = k, k.astype(np.float64)
    p.upload()
    q = np.full((3, H * hd), 8.0, np.float16)
    got = host(attn_call(p, dev_(q), H, 1.0))
    attn_check(p, got, q, H, 1.0)          # exact scores: every product and sum is an integer below 2^24


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("H,KV,hd,lens,max_seq", [
    (32, 32, 32, [40000], None),                       # parts of more than 1024 keys: several page look-ups
    (4, 2, 32, [3000] + [5] * 70 + [0] * 60 + [1500] + [1] * 3, None),   # rows counted in groups of 64
    (4, 2, 32, [0] * 130 + [2000], None),
    (4, 2, 32, [0] * 70, 4000),                        # nothing to do
    (4, 2, 32, [1, 0, 33, 2], 100000),                 # lengths far below what they could be
    (2, 1, 32, [37, 90] * 500 + [3000, 0, 2000] + [1] * 97, None),       # more rows than are counted
    (4, 1, 64, [1023, 1024, 1025, 2047, 2049, 1100], None)])
def test_attention_parts(dev, int8, H, KV, hd, lens, max_seq):
    print_case("paged attn parts", int8, H, KV, len(lens))
    g = rng(H, KV, len(lens))
    p = Pool(g, lens, KV, hd, 16, int8, max_seq=max_seq).upload()
    q = (g.standard_normal((len(lens), H * hd)) * 1.2).astype(np.float16)
    attn_check(p, host(attn_call(p, dev_(q), H, 0.15)), q, H, 0.15)


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("hd", [32, 64, 96, 128])
@pytest.mark.parametrize("H,KV,lens", [
    (8, 8, [40, 17, 33, 0] * 64),                      # whole rows, four KV heads to a workgroup
    (16, 8, [70, 1, 31] * 22),                         # two
    (4, 2, [200, 90]),                                 # one
    (4, 2, [3000, 2900, 40] * 8),                      # parts, int8: two
    (2, 2, [1500, 700])])                              # parts, one
def test_attention_heads_side_by_side(dev, int8, hd, H, KV, lens):
    print_case("paged attn heads", int8, hd, H, KV, len(lens))
    g = rng(hd, H, KV, len(lens))
    p = Pool(g, lens, KV, hd, 16, int8).upload()
    q = (g.standard_normal((len(lens), H * hd)) * 1.2).astype(np.float16)
    scale = 1 / np.sqrt(hd)
    attn_check(p, host(attn_call(p, dev_(q), H, scale)), q, H, scale)


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("H,KV,hd", [(16, 8, 128), (8, 8, 96), (24, 8, 64), (8, 8, 32), (16, 2, 32), (6, 6, 96)])
def test_attention_parts_of_batches_that_could_be_long(dev, int8, H, KV, hd):
    print_case("paged attn long bound", int8, H, KV, hd)
    g = rng(H, KV, hd, 5)
    lens = [3000, 0, 40, 1500, 700, 33, 1, 2900]
    p = Pool(g, lens, KV, hd, 64, int8, max_seq=2 ** 17 // KV + 100).upload()
    q = (g.standard_normal((len(lens), H * hd)) * 1.2).astype(np.float16)
    scale = 1 / np.sqrt(hd)
    attn_check(p, host(attn_call(p, dev_(q), H, scale)), q, H, scale)


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("B", [63, 64, 65, 127, 128, 129, 1000, 1023, 1024])
def test_attention_parts_of_many_rows(dev, int8, B):
    print_case("paged attn many rows", int8, B)
    g = rng(B, 6)
    lens = [int(n) for n in g.integers(0, 1200, B) * (g.random(B) < 0.4)]
    lens[-1] = 1100
    p = Pool(g, lens, 1, 32, 16, int8).upload()
    q = (g.standard_normal((B, 2 * 32)) * 1.2).astype(np.float16)
    attn_check(p, host(attn_call(p, dev_(q), 2, 0.2)), q, 2, 0.2)


@pytest.mark.parametrize("page", [32, 256, 1024, 4096])
def test_attention_page_sizes(dev, page):
    g = rng(page)
    p = Pool(g, [5000, 1, 0, 256, 1025], 2, 64, page, True).upload()
    q = g.standard_normal((5, 8 * 64)).astype(np.float16)
    attn_check(p, host(attn_call(p, dev_(q), 8, 0.125)), q, 8, 0.125)


@pytest.mark.parametrize("lens", [[100, 250], [2500, 40, 300]])
@pytest.mark.parametrize("which", ["ks", "vs"])
def test_attention_scales_of_either_sign_and_one_null(dev, lens, which):
    """Scales may be negative; with only one array given the other side's codes
    stand for themselves."""
    H, KV, hd = 8, 2, 64
    g = rng(len(lens), ord(which[0]))
    p = Pool(g, lens, KV, hd, 16, True)
    sc = getattr(p, which)
    sc *= np.where(g.random(sc.shape) < 0.4, -1.0, 1.0).astype(np.float32)
    p.upload()
    p.d[2 if which == "vs" else 3] = None
    q = (g.standard_normal((len(lens), H * hd)) * 0.02).astype(np.float16)
    for b, n in enumerate(lens):
        pg, off = p.table[b][np.arange(n) // 16], np.arange(n) % 16
        p.k[b] = p.kp[pg, off].astype(np.float64) * (p.ks[pg, off][..., None].astype(np.float64) if which == "ks" else 1)
        p.v[b] = p.vp[pg, off].astype(np.float64) * (p.vs[pg, off][..., None].astype(np.float64) if which == "vs" else 1)
    attn_check(p, host(attn_call(p, dev_(q), H, 0.125)), q, H, 0.125)


@pytest.mark.parametrize("lens", [[50, 0, 3], [3000, 0, 20]])
def test_attention_writes_its_rows_and_no_others(dev, lens):
    H, KV, hd = 8, 2, 64
    g = rng(77)
    p = Pool(g, lens, KV, hd, 16, False).upload()
    q = g.standard_normal((3, H * hd)).astype(np.float16)
    out = torch.full((6, H * hd), 7.0, dtype=torch.float16, device="cuda:0")
    need = jllm.lib().jllm_hip_flash_attention_decode_paged_workspace(3, H, KV, hd, p.max_seq, 0)
    ws = torch.full((need + 64,), 0xFF, dtype=torch.uint8, device="cuda:0")
    attn_call(p, dev_(q), H, 0.125, out=out[1:4], ws=ws[:max(need, 16)])
    got = host(out)
    attn_check(p, got[1:4], q, H, 0.125)
    assert np.all(got[0] == 7.0) and np.all(got[4:] == 7.0)
    assert np.all(host(ws)[need:] == 0xFF)             # the workspace is as large as it says


def test_attention_whole_rows_by_environment(dev):
    """JLLM_SPLITK=0 (read once: a process of its own) leaves long rows whole."""
    code = (
        "import numpy as np, jllm, test_serving_gpu as t\n"
        "assert jllm.lib().jllm_hip_flash_attention_decode_paged_workspace(3, 8, 4, 64, 9000, 0) == 0\n"
        "for int8 in (False, True):\n"
        "    g = t.rng(5)\n"
        "    p = t.Pool(g, [9000, 0, 1500], 4, 64, 16, int8).upload()\n"
        "    q = g.standard_normal((3, 8 * 64)).astype(np.float16)\n"
        "    t.attn_check(p, t.host(t.attn_call(p, t.dev_(q), 8, 0.125)), q, 8, 0.125)\n"
        "print('whole rows ok')\n")
    here = os.path.dirname(os.path.abspath(__file__))
    path = os.pathsep.join([here, os.path.join(os.path.dirname(here), "genie-ai-runtime_amd"), os.environ.get("PYTHONPATH", "")])
    r = subprocess.run([sys.executable, "-c", code], env=dict(os.environ, JLLM_SPLITK="0", PYTHONPATH=path),
                       capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and "whole rows ok" in r.stdout, r.stdout + r.stderr


@pytest.mark.parametrize("window", [1100, 3000])
def test_attention_parts_with_a_window(dev, window):
    H, KV, hd = 8, 2, 64
    g = rng(window, 2)
    lens = [9000, 1, 0, window, window + 1, window + 15, window + 16, 5000] + [2500] * 66
    p = Pool(g, lens, KV, hd, 16, True).upload()
    q = g.standard_normal((len(lens), H * hd)).astype(np.float16)
    attn_check(p, host(attn_call(p, dev_(q), H, 0.125, window)), q, H, 0.125, window)


@pytest.mark.parametrize("int8", [False, True])
def test_attention_strided_q(dev, int8):
    H, KV, hd = 32, 8, 128
    g = rng(10)
    lens = [100, 7, 600]
    p = Pool(g, lens, KV, hd, 16, int8).upload()
    qkv = g.standard_normal((3, (H + 2 * KV) * hd)).astype(np.float16)
    Q = dev_(qkv)
    got = host(attn_call(p, Q, H, 0.09, q_stride=Q.stride(0)))
    attn_check(p, got, qkv[:, :H * hd], H, 0.09)


def test_attention_same_bits_twice_and_with_any_max_seq_slack(dev):
    H, KV, hd = 32, 8, 128
    g = rng(11)
    lens = [1500, 3, 0, 800]
    p = Pool(g, lens, KV, hd, 16, True, max_seq=6000).upload()
    q = g.standard_normal((4, H * hd)).astype(np.float16)
    a = host(attn_call(p, dev_(q), H, 0.09))
    b = host(attn_call(p, dev_(q), H, 0.09))
    assert np.array_equal(a.view(np.uint16), b.view(np.uint16))
    attn_check(p, a, q, H, 0.09)
    attn_check(p, host(attn_call(p, dev_(q), H, 0.09, max_seq=1500)), q, H, 0.09)


@pytest.mark.parametrize("int8", [False, True])
def test_attention_offsets_past_32_bits(dev, int8):
    """A pool of more than 2^32 bytes a side, pages at both ends."""
    H, KV, hd, page = 16, 8, 128, 16
    g = rng(12)
    lens = [40, 100]
    small = Pool(g, lens, KV, hd, page, int8)
    n_pages = (5 << 30) // (page * KV * hd * (1 if int8 else 2))
    used = np.unique(small.table[small.table >= 0])
    # every second page of the small pool goes to the far end of the large one
    move = {int(o): int(i if i % 2 else n_pages - 1 - i) for i, o in enumerate(used)}
    kind = torch.int8 if int8 else torch.float16
    kp, vp = [torch.empty((n_pages, page, KV, hd), dtype=kind, device="cuda:0") for _ in range(2)]
    ks, vs = [torch.empty((n_pages, page, KV), device="cuda:0") for _ in range(2)]
    for o, n in move.items():
        for big, src in ((kp, small.kp), (vp, small.vp), (ks, small.ks), (vs, small.vs)):
            big[n] = dev_(src[o])
    small.table = np.where(small.table >= 0, np.vectorize(lambda i: move.get(int(i), -1))(small.table), -1).astype(np.int32)
    small.n_pages = n_pages
    small.d = [kp, vp, ks, vs, dev_(small.table), dev_(np.array(lens, np.int32))]
    q = g.standard_normal((2, H * hd)).astype(np.float16)
    attn_check(small, host(attn_call(small, dev_(q), H, 0.09)), q, H, 0.09)


def test_front_offsets_past_32_bits(dev):
    KV, hd, H = 8, 128, 8
    n_slots = (5 << 30) // (KV * hd * 2)
    g = rng(13)
    x = g.standard_normal((4, (H + 2 * KV) * hd)).astype(np.float16)
    slots = np.array([0, n_slots - 1, n_slots // 2, n_slots - 17], np.int32)
    kp, vp = [torch.empty((n_slots, KV, hd), dtype=torch.float16, device="cuda:0") for _ in range(2)]
    q, k, v = [dev_(np.ascontiguousarray(a)) for a in np.split(x, [H * hd, (H + KV) * hd], 1)]
    pos = np.array([5, 6, 7, 8], np.int32)
    jllm.call("jllm_hip_qk_norm_rope_store_kv_paged", q, H * hd, q, H * hd, k, KV * hd, v, KV * hd, None, None, 0, 1e-6,
              kp, vp, None, None, n_slots, dev_(pos), dev_(slots), H, KV, hd, hd, 4, 1e6, 1, 0)
    at = torch.from_numpy(slots.astype(np.int64)).to("cuda:0")
    want = front_ref(x[:, H * hd:(H + KV) * hd].astype(np.float64).reshape(4, KV, hd), None, pos, 1e6, True, 1e-6)
    assert fp16_close(host(kp[at]), want, np.abs(want).max(-1, keepdims=True))
    assert np.array_equal(host(vp[at]).reshape(4, -1), x[:, (H + KV) * hd:])


# ---- logits -------------------------------------------------------------------------

def logits_ref(x, c, t=np.float32):
    """The definition, one row at a time, every operation rounded to type t."""
    y = x.astype(t).copy()
    B, V = y.shape
    for b in range(B):
        if c.get("tokens") is not None:
            n = int(np.clip(c["n_tokens"][b], 0, c["tokens"].shape[1]))
            p = int(np.clip(c["n_prompt"][b], 0, n)) if c.get("n_prompt") is not None else 0
            ids = c["tokens"][b, :n].astype(np.int64)
            ok = (ids >= 0) & (ids < V)
            cnt = np.bincount(ids[p:][ok[p:]], minlength=V)
            old = np.unique(ids[ok])
            r = t(c["rep"][b]) if c.get("rep") is not None else t(1)
            with np.errstate(all="ignore"):
                y[b, old] = np.where(y[b, old] > 0, y[b, old] / r, y[b, old] * r)
                at = np.nonzero(cnt)[0]
                if c.get("freq") is not None:
                    y[b, at] = y[b, at] - t(c["freq"][b]) * cnt[at].astype(t)
                if c.get("pres") is not None:
                    y[b, at] = y[b, at] - t(c["pres"][b])
        if c.get("bias_ids") is not None:
            for j in {int(i): j for j, i in enumerate(c["bias_ids"][b, :max(0, int(c["n_bias"][b]))])}.items():
                if 0 <= j[0] < V:
                    y[b, j[0]] = y[b, j[0]] + t(c["bias"][b, j[1]])
        if c.get("mask") is not None:
            bits = (c["mask"][b].astype(np.uint32)[:, None] >> np.arange(32, dtype=np.uint32)) & 1
            y[b, bits.reshape(-1)[:V] == 0] = -np.inf
    tok = np.full(B, -1, np.int32)
    for b in range(B):
        fine = np.isfinite(y[b])
        if fine.any():
            tok[b] = int(np.argmax(np.where(fine, y[b], -np.inf)))
    return y, tok


def logits_case(g, B, V, hist=0, bias=0, mask=False, prompt=True):
    c = {}
    if hist:
        c["tokens"] = (g.random((B, hist)) ** 3 * V).astype(np.int32)
        c["n_tokens"] = g.integers(0, hist + 1, B).astype(np.int32)
        if prompt:
            c["n_prompt"] = (c["n_tokens"] // 2).astype(np.int32)
        c["rep"] = (1 + g.random(B) * 0.5).astype(np.float32)
        c["freq"] = g.random(B).astype(np.float32)
        c["pres"] = g.random(B).astype(np.float32)
    if bias:
        c["bias_ids"] = g.integers(0, V, (B, bias)).astype(np.int32)
        c["bias"] = (g.standard_normal((B, bias)) * 4).astype(np.float32)
        c["n_bias"] = g.integers(0, bias + 1, B).astype(np.int32)
    if mask:
        c["mask"] = g.integers(0, 2 ** 32, (B, (V + 31) // 32), dtype=np.uint32)
    return c


def logits_call(x, c, in_place=False, pick=True, out_stride=None, x_stride=None, offset=0):
    B, V = x.shape
    xs = x_stride or V
    buf = torch.full((offset + B * xs,), 5.0, device="cuda:0")
    X = torch.as_strided(buf, (B, V), (xs, 1), offset)
    X.copy_(dev_(x))
    os_ = xs if in_place else (out_stride or V)
    obuf = buf if in_place else torch.full((offset + B * os_,), 5.0, device="cuda:0")
    O = torch.as_strided(obuf, (B, V), (os_, 1), offset)
    d = {k: dev_(v.view(np.int32) if v.dtype == np.uint32 else v) for k, v in c.items()}
    stride = lambda n: c[n].shape[1] if c.get(n) is not None else 0  # noqa: E731
    tok = torch.full((B,), -9, dtype=torch.int32, device="cuda:0") if pick else None
    ws = torch.full((max(jllm.lib().jllm_hip_logits_process_workspace(B, V), 16),), 0xFF, dtype=torch.uint8,
                    device="cuda:0")
    jllm.call("jllm_hip_logits_process", O, os_, X, xs, B, V, d.get("tokens"), stride("tokens"), d.get("n_prompt"),
              d.get("n_tokens"), d.get("rep"), d.get("freq"), d.get("pres"), d.get("bias_ids"), d.get("bias"),
              stride("bias_ids"), d.get("n_bias"), d.get("mask"), stride("mask"), tok, ws if pick else None,
              ws.numel() if pick else 0)
    got = host(O)
    rest = host(obuf).copy()
    if os_ > V:                            # nothing between the rows is touched
        gaps = np.ones(len(rest), bool)
        for b in range(B):
            gaps[offset + b * os_:offset + b * os_ + V] = False
        assert np.all(rest[gaps] == 5.0)
    return got, None if tok is None else host(tok)


def same(a, b):
    return np.array_equal(a.view(np.uint32), b.view(np.uint32))


@pytest.mark.parametrize("B,V,hist,bias,mask", [
    (1, 1, 3, 2, True), (1, 31, 10, 0, False), (3, 32, 10, 3, True), (2, 33, 0, 3, True), (5, 1000, 50, 0, True),
    (3, 4095, 100, 9, False), (3, 4096, 100, 9, True), (3, 4097, 100, 9, True), (2, 8193, 3000, 300, True),
    (4, 32003, 500, 20, True), (1, 151936, 700, 0, False), (2, 151936, 20000, 300, True), (70, 5000, 64, 4, True),
    (2, 12289, 0, 0, False), (300, 129, 20, 5, True)])
def test_logits(dev, B, V, hist, bias, mask):
    print_case("logits", B, V, hist, bias, mask)
    g = rng(B, V, hist)
    x = (g.standard_normal((B, V)) * 4).astype(np.float32)
    c = logits_case(g, B, V, hist, bias, mask)
    want, tok = logits_ref(x, c)
    got, t = logits_call(x, c)
    assert same(got, want) and np.array_equal(t, tok)
    far, _ = logits_ref(x, c, np.float64)     # 5 roundings of terms below 2^13
    fine = np.isfinite(far)
    assert np.array_equal(fine, np.isfinite(got))
    assert np.all(np.abs(got[fine] - far[fine]) <= 5 * U * (np.abs(far[fine]) + 2.0 ** 13))


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("offset,gap", [(0, 0), (1, 1), (3, 6), (2, 0)])
def test_logits_strides_and_alignment(dev, in_place, offset, gap):
    g = rng(offset, gap)
    B, V = 5, 5003
    x = g.standard_normal((B, V)).astype(np.float32)
    c = logits_case(g, B, V, 40, 5, True)
    want, tok = logits_ref(x, c)
    got, t = logits_call(x, c, in_place=in_place, x_stride=V + gap, out_stride=V + 2 * gap, offset=offset)
    assert same(got, want) and np.array_equal(t, tok)


@pytest.mark.parametrize("drop", ["n_prompt", "rep", "freq", "pres"])
def test_logits_optional_arrays(dev, drop):
    g = rng(3)
    x = g.standard_normal((4, 3001)).astype(np.float32)
    c = logits_case(g, 4, 3001, 80, 4, True)
    del c[drop]
    want, tok = logits_ref(x, c)
    got, t = logits_call(x, c)
    assert same(got, want) and np.array_equal(t, tok)
    got, _ = logits_call(x, c, pick=False)
    assert same(got, want)


def test_logits_bad_ids_and_counts(dev):
    g = rng(4)
    B, V = 4, 9000
    x = g.standard_normal((B, V)).astype(np.float32)
    c = logits_case(g, B, V, 30, 6, False)
    c["tokens"][:, ::3] = [-1, V, 2 ** 31 - 1, -2 ** 31, V + 4096, -4096, 0, V - 1, 5, 5]
    c["bias_ids"][:, ::2] = [-1, V, -2 ** 31]
    c["n_tokens"][:] = [30, 31, -5, 2 ** 31 - 1]
    c["n_prompt"][:] = [-7, 100, 3, 15]
    c["n_bias"][:] = [6, 7, -1, 2 ** 31 - 1]
    want, tok = logits_ref(x, c)
    got, t = logits_call(x, c)
    assert same(got, want) and np.array_equal(t, tok)


@pytest.mark.parametrize("B,hist,bias", [(1, 1, 1), (1, 1500, 300), (3, 1027, 259), (2, 5, 7)])
def test_logits_lists_inside_wider_rows(dev, B, hist, bias):
    """Lists that are columns of wider arrays, the last row ending where the
    array ends."""
    g = rng(B, hist, bias)
    V = 5000
    x = g.standard_normal((B, V)).astype(np.float32)
    c = logits_case(g, B, V, hist, bias, False)
    c["n_tokens"][-1], c["n_bias"][-1] = hist, bias
    want, tok = logits_ref(x, c)
    wide, bwide = np.full((B, hist + 9), 17, np.int32), np.full((B, bias + 5), 17, np.int32)
    bval = np.full((B, bias + 5), 1e6, np.float32)
    wide[:, 9:], bwide[:, 5:], bval[:, 5:] = c["tokens"], c["bias_ids"], c["bias"]
    d = {k: dev_(v) for k, v in c.items()}
    W, BW, BV = dev_(wide)[:, 9:], dev_(bwide)[:, 5:], dev_(bval)[:, 5:]
    out, t = torch.zeros((B, V), device="cuda:0"), torch.zeros((B,), dtype=torch.int32, device="cuda:0")
    ws = torch.empty((max(jllm.lib().jllm_hip_logits_process_workspace(B, V), 16),), dtype=torch.uint8, device="cuda:0")
    jllm.call("jllm_hip_logits_process", out, V, dev_(x), V, B, V, W, W.stride(0), d["n_prompt"], d["n_tokens"], d["rep"],
              d["freq"], d["pres"], BW, BV, BW.stride(0), d["n_bias"], None, 0, t, ws, ws.numel())
    assert same(host(out), want) and np.array_equal(host(t), tok)


def test_logits_token_listed_often(dev):
    """One token 20000 times in the output, and a bias list of one token: the
    count is whole, the last bias counts."""
    V = 6000
    x = np.zeros((2, V), np.float32)
    x[0, 17], x[1, 17] = 3.0, -3.0
    c = {"tokens": np.full((2, 20000), 17, np.int32), "n_tokens": np.array([20000, 19999], np.int32),
         "n_prompt": np.array([1, 19999], np.int32), "rep": np.array([1.5, 1.5], np.float32),
         "freq": np.array([0.25, 0.25], np.float32), "pres": np.array([0.5, 0.5], np.float32),
         "bias_ids": np.full((2, 700), 17, np.int32), "bias": np.arange(1400, dtype=np.float32).reshape(2, 700),
         "n_bias": np.array([700, 3], np.int32)}
    got, t = logits_call(x, c)
    assert got[0, 17] == np.float32(2.0) - np.float32(0.25 * 19999) - np.float32(0.5) + np.float32(699)
    assert got[1, 17] == np.float32(-4.5) + np.float32(702)
    want, tok = logits_ref(x, c)
    assert same(got, want) and np.array_equal(t, tok)


def test_logits_ties_and_nonfinite(dev):
    V = 10000
    x = np.full((9, V), -2.0, np.float32)
    x[0, [9999, 5000, 4096]] = 7.0                 # tie across chunks: lowest index
    x[1, [130, 129]] = 7.0
    x[2, 300], x[2, 20] = np.inf, 1.0              # infinities and NaN are not picked
    x[3, 300], x[3, 20] = np.nan, 1.0
    x[4] = np.nan
    x[5] = -np.inf
    x[6, 8000] = -0.0                              # -0 and +0 tie
    x[6, 9000] = 0.0
    x[6][x[6] == -2.0] = -1.0
    x[7] = -3.4028235e38                           # the type's lowest value is a value
    x[8] = 3.4028235e38
    want = [4096, 129, 20, 20, -1, -1, 8000, 0, 0]
    got, t = logits_call(x, {})
    assert same(got, x) and list(t) == want


def test_logits_masks_that_leave_nothing_or_one(dev):
    V = 4500
    g = rng(5)
    x = g.standard_normal((4, V)).astype(np.float32)
    x[3, 4499] = np.nan
    m = np.zeros((4, (V + 31) // 32), np.uint32)
    m[1, 4499 // 32] = 1 << (4499 % 32)
    m[2, 0] = 1
    m[3, 4499 // 32] = 1 << (4499 % 32)
    m[0, -1] = 0xFFFFFFFF << (V % 32) & 0xFFFFFFFF          # bits behind V are no tokens
    got, t = logits_call(x, {"mask": m})
    assert list(t) == [-1, 4499, 0, -1]
    assert np.isneginf(got[0]).all() and np.isneginf(got[1, :-1]).all() and got[1, 4499] == x[1, 4499]
    assert np.isnan(got[3, 4499])


# ---- streams, graphs, a serving step ---------------------------------------------------

def test_calls_on_two_streams(dev):
    """Two independent calls of each operator, each on a stream and with a
    workspace of its own, many times in a row."""
    H, KV, hd = 32, 8, 128
    jobs = []
    for i in range(2):
        g = rng(20, i)
        p = Pool(g, [1500 + 100 * i, 40, 700], KV, hd, 16, bool(i)).upload()
        q = g.standard_normal((3, H * hd)).astype(np.float16)
        x = g.standard_normal((3, 40000)).astype(np.float32)
        jobs.append((p, q, dev_(q), x, dev_(x), torch.cuda.Stream()))
    torch.cuda.synchronize()
    res = [[], []]
    lib = jllm.lib()
    bufs = []
    for i, (p, q, Q, x, X, st) in enumerate(jobs):
        need = lib.jllm_hip_flash_attention_decode_paged_workspace(3, H, KV, hd, p.max_seq, 0)
        bufs.append((torch.empty(max(need, 16), dtype=torch.uint8, device="cuda:0"),
                     torch.empty(max(lib.jllm_hip_logits_process_workspace(3, 40000), 16), dtype=torch.uint8, device="cuda:0"),
                     [torch.zeros((3, H * hd), dtype=torch.float16, device="cuda:0") for _ in range(10)],
                     [torch.zeros((3,), dtype=torch.int32, device="cuda:0") for _ in range(10)],
                     torch.empty_like(X)))
    torch.cuda.synchronize()
    for r in range(10):
        for i, (p, q, Q, x, X, st) in enumerate(jobs):
            aw, lw, outs, toks, Y = bufs[i]
            attn_call(p, Q, H, 0.09, stream=st.cuda_stream, out=outs[r], ws=aw)
            jllm.call("jllm_hip_logits_process", Y, 40000, X, 40000, 3, 40000, None, 0, None, None, None, None, None,
                      None, None, 0, None, None, 0, toks[r], lw, lw.numel(), stream=st.cuda_stream)
    torch.cuda.synchronize()
    for i, (p, q, Q, x, X, st) in enumerate(jobs):
        _, _, outs, toks, Y = bufs[i]
        for o, t in zip(outs, toks):
            attn_check(p, host(o), q, H, 0.09)
            assert np.array_equal(host(t), x.argmax(-1))


class Server:
    """A toy model over the three operators: fixed random projections around a
    paged layer, several sequences, greedy; the oracle does the same in float64."""

    H, KV, hd, page, V = 8, 2, 64, 16, 5000

    def __init__(self, seed, prompts, steps, int8):
        g = rng(30, seed)
        self.int8, self.steps = int8, steps
        self.prompts = prompts
        self.B = len(prompts)
        W = (self.H + 2 * self.KV) * self.hd
        self.emb = (g.standard_normal((self.V, W)) * 0.8).astype(np.float16)
        self.head = (g.standard_normal((self.H * self.hd, self.V)) * 0.2).astype(np.float32)
        self.qw, self.kw = [(1 + 0.2 * g.standard_normal(self.hd)).astype(np.float32) for _ in range(2)]
        most = max(len(p) for p in prompts) + steps
        self.max_seq = most
        per = (most + self.page - 1) // self.page
        self.n_pages = self.B * per + 1
        self.table = g.permutation(self.n_pages)[:self.B * per].reshape(self.B, per).astype(np.int32)
        self.mask = g.integers(0, 2 ** 32, (self.B, (self.V + 31) // 32), dtype=np.uint32)
        self.scale = 1 / np.sqrt(self.hd)

    def slot(self, b, t):
        return int(self.table[b, t // self.page]) * self.page + t % self.page

    def device(self):
        d = self.__dict__.setdefault("d", {})
        for n in ("emb", "qw", "kw", "table"):
            d[n] = dev_(getattr(self, n))
        d["head"] = dev_(self.head.T)
        d["mask"] = dev_(self.mask.view(np.int32))
        kind = torch.int8 if self.int8 else torch.float16
        n = self.n_pages * self.page
        z = lambda *s, t=torch.float32: torch.zeros(s, dtype=t, device="cuda:0")  # noqa: E731
        d["kp"], d["vp"] = z(n, self.KV, self.hd, t=kind), z(n, self.KV, self.hd, t=kind)
        d["ks"], d["vs"] = z(n, self.KV), z(n, self.KV)
        return d

    def front(self, qkv, pos, slots):
        d, H, KV, hd = self.d, self.H, self.KV, self.hd
        q, k, v = qkv.split([H * hd, KV * hd, KV * hd], dim=1)
        W = qkv.stride(0)
        jllm.call("jllm_hip_qk_norm_rope_store_kv_paged", q, W, q, W, k, W, v, W, d["qw"], d["kw"], 1, 1e-6, d["kp"],
                  d["vp"], d["ks"] if self.int8 else None, d["vs"] if self.int8 else None, self.n_pages * self.page,
                  pos, slots, H, KV, hd, hd, qkv.shape[0], 1e4, 1, int(self.int8))

    def attn(self, qkv, table, lens, out, ws):
        d, H, KV, hd = self.d, self.H, self.KV, self.hd
        jllm.call("jllm_hip_flash_attention_decode_paged", out, qkv, qkv.stride(0), d["kp"], d["vp"],
                  d["ks"] if self.int8 else None, d["vs"] if self.int8 else None, self.n_pages, self.page, table,
                  table.stride(0), lens, qkv.shape[0], H, KV, hd, hd, self.max_seq, self.scale, int(self.int8), 0, ws,
                  ws.numel())

    def ws(self, B):
        n = jllm.lib().jllm_hip_flash_attention_decode_paged_workspace(B, self.H, self.KV, self.hd, self.max_seq, 0)
        return torch.empty(max(n, 16), dtype=torch.uint8, device="cuda:0")

    def start(self):
        """Prompts in one chunk, one row per token; returns each sequence's first state."""
        d = self.device()
        rows = [(b, t) for b, p in enumerate(self.prompts) for t in range(len(p))]
        qkv = d["emb"][torch.tensor([self.prompts[b][t] for b, t in rows], device="cuda:0")]
        pos = dev_(np.array([t for _, t in rows], np.int32))
        self.front(qkv, pos, dev_(np.array([self.slot(b, t) for b, t in rows], np.int32)))
        out = torch.empty((len(rows), self.H * self.hd), dtype=torch.float16, device="cuda:0")
        self.attn(qkv, d["table"][torch.tensor([b for b, _ in rows], device="cuda:0")].contiguous(), pos + 1, out,
                  self.ws(len(rows)))
        self.state(out[torch.tensor([i for i, (b, t) in enumerate(rows) if t == len(self.prompts[b]) - 1], device="cuda:0")])
        return host(out)

    def state(self, x):
        """Buffers of the decode step; tokens of the prompts picked from x."""
        d, B = self.d, self.B
        most = self.max_seq + 1
        hist = np.zeros((B, most), np.int32)
        for b, p in enumerate(self.prompts):
            hist[b, :len(p)] = p
        n = np.array([len(p) for p in self.prompts], np.int32)
        d["hist"], d["n"], d["np"] = dev_(hist), dev_(n), dev_(n.copy())
        d["rep"], d["freq"], d["pres"] = [torch.full((B,), v, device="cuda:0") for v in (1.25, 0.25, 0.5)]
        d["x"] = x.clone()
        d["tok"] = torch.zeros((B,), dtype=torch.int32, device="cuda:0")
        d["half"] = torch.zeros((B, self.V), dtype=torch.float16, device="cuda:0")
        d["logits"] = torch.zeros((B, self.V), device="cuda:0")
        d["lw"] = torch.empty(max(jllm.lib().jllm_hip_logits_process_workspace(B, self.V), 16), dtype=torch.uint8, device="cuda:0")
        d["aw"] = self.ws(B)
        d["out"] = torch.zeros((B, self.H * self.hd), dtype=torch.float16, device="cuda:0")
        self.pick()

    def pick(self):
        d = self.d
        jllm.call("jllm_hip_gemm_dense_batched", d["half"], d["head"], 0, d["x"], self.V, self.B, self.H * self.hd)
        d["logits"].copy_(d["half"])
        jllm.call("jllm_hip_logits_process", d["logits"], self.V, d["logits"], self.V, self.B, self.V, d["hist"],
                  d["hist"].shape[1], d["np"], d["n"], d["rep"], d["freq"], d["pres"], None, None, 0, None, d["mask"],
                  d["mask"].shape[1], d["tok"], d["lw"], d["lw"].numel())
        d["hist"].scatter_(1, d["n"].long()[:, None], d["tok"][:, None])

    def step(self):
        """The picked tokens go in, the next ones come out; nothing is read on the host."""
        d = self.d
        qkv = d["emb"][d["tok"].long()]
        t = d["n"]
        slots = d["table"].gather(1, (t // self.page).long()[:, None])[:, 0] * self.page + t % self.page
        self.front(qkv, t, slots)
        d["n"].add_(1)
        self.attn(qkv, d["table"], d["n"], d["out"], d["aw"])
        d["x"].copy_(d["out"])
        self.pick()

    def oracle(self, tokens):
        """float64 logits before each of tokens[b] of sequence b (teacher-forced), and
        how far they may be off (see replayed)."""
        res = []
        for b, p in enumerate(self.prompts):
            ids = list(p) + list(tokens[b])
            x = self.emb[ids].astype(np.float64)
            pos = np.arange(len(ids))
            q, k, v = np.split(x, [self.H * self.hd, (self.H + self.KV) * self.hd], 1)
            q = front_ref(q.reshape(-1, self.H, self.hd), self.qw.astype(np.float64), pos, 1e4, True, 1e-6)
            k = front_ref(k.reshape(-1, self.KV, self.hd), self.kw.astype(np.float64), pos, 1e4, True, 1e-6)
            v = v.reshape(-1, self.KV, self.hd)
            if self.int8:
                k, v = [np.rint(a / (s := np.abs(a).max(-1, keepdims=True) / 127)) * s for a in (k, v)]
            head, size = self.head.astype(np.float64), np.abs(self.head).astype(np.float64)
            rows = []
            for i in range(len(p), len(ids) + 1):
                o, A = attn_ref(q[i - 1], k, v, self.scale, 0, i)
                qa = np.abs(q[i - 1]).reshape(self.KV, -1, self.hd)
                s = np.einsum("jhd,tjd->jht", qa, np.abs(k[:i])).max() * self.scale
                err = 2.0 ** -11 * np.abs(o) + (2.0 ** -10 + 2.0 ** -11 + 2 * s * 2.0 ** -10) * A
                tol = err.reshape(-1) @ size
                if self.int8:
                    kstep, vstep = np.abs(k[:i]).max() / 127, np.abs(v[:i]).max() / 127
                    tol += size.max() * vstep + 2 * self.scale * qa.max() * kstep * (A.reshape(-1) @ size)
                y = o.reshape(-1) @ head
                rows.append((y, tol + 2.0 ** -11 * np.abs(y)))
            res.append(rows)
        return res


def prompts_of(seed, lens):
    g = rng(31, seed)
    return [list(map(int, g.integers(0, Server.V, n))) for n in lens]


def replayed(s, tokens, got_logits):
    """Every step's processed logits against the float64 oracle; the picked token
    has to be within twice the error of the best.  Error before the penalties: of an
    attention output the bound above, with the fp16 roundings of q, k (2^-10 of the
    largest sum of |q k| in the scores, twice in the weights) and v (2^-11 A); of a
    logit the sum over the head's column, and its rounding to fp16.  INT8: at most
    one code in a row falls on the other side of a step."""
    raw = s.oracle([t[:-1] for t in tokens])
    for b, p in enumerate(s.prompts):
        for i in range(len(tokens[b])):
            c = {"tokens": np.array([list(p) + list(tokens[b][:i])], np.int32), "n_tokens": np.array([len(p) + i]),
                 "n_prompt": np.array([len(p)]), "rep": np.array([1.25]), "freq": np.array([0.25]),
                 "pres": np.array([0.5]), "mask": s.mask[b:b + 1]}
            y, tol = raw[b][i]
            want, _ = logits_ref(y[None], c, np.float64)
            want, got, tol = want[0], got_logits[i][b], 1.25 * tol
            fine = np.isfinite(want)
            assert np.array_equal(fine, np.isfinite(got))
            assert np.all(np.abs(want[fine] - got[fine]) <= tol[fine])
            assert want[tokens[b][i]] >= want[fine].max() - 2 * tol.max()


@pytest.mark.parametrize("int8", [False, True])
def test_serving_run(dev, int8):
    """Prompts and 12 greedy steps of four sequences, eager."""
    s = Server(1, prompts_of(1, [1, 16, 40, 131]), 13, int8)
    s.start()
    toks, logits = [host(s.d["tok"]).copy()], [host(s.d["logits"]).copy()]
    for _ in range(12):
        s.step()
        toks.append(host(s.d["tok"]).copy())
        logits.append(host(s.d["logits"]).copy())
    replayed(s, np.array(toks).T, logits)


@pytest.mark.parametrize("int8", [False, True])
def test_serving_run_captured(dev, int8):
    """The step of two servers captured into a graph each, replayed in turn with eager
    work between: the tokens and logits of the eager runs."""
    cases = [(2, [5, 20, 33]), (3, [60, 2, 17])]
    eager = []
    for seed, lens in cases:
        s = Server(seed, prompts_of(seed, lens), 10, int8)
        s.start()
        rows = []
        for _ in range(8):
            s.step()
            rows.append((host(s.d["tok"]).copy(), host(s.d["logits"]).copy()))
        eager.append(rows)
    pairs = []
    for seed, lens in cases:
        s = Server(seed, prompts_of(seed, lens), 10, int8)
        s.start()
        torch.cuda.synchronize()
        keep = {k: v.clone() for k, v in s.d.items()}
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            s.step()                       # warm-up outside the capture
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            s.step()
        for k, v in keep.items():
            s.d[k].copy_(v)
        pairs.append((s, gr))
    torch.cuda.synchronize()
    for i in range(8):
        for j, (s, gr) in enumerate(pairs):
            gr.replay()
            if i % 3 == 1:
                torch.cuda.synchronize()
            torch.ones(1000, device="cuda:0").cumsum(0)
            tok, lg = host(s.d["tok"]), host(s.d["logits"])
            assert np.array_equal(tok, eager[j][i][0]) and same(lg, eager[j][i][1]), (i, j)


def test_prompt_chunk_rows_equal_single_tokens(dev):
    """A prompt passed as one row per token in one call gives what one call per
    token gives, up to the split of the keys."""
    s = Server(4, prompts_of(4, [70]), 4, False)
    chunk = s.start().astype(np.float64)
    d = s.device()
    for t in range(70):
        qkv = d["emb"][torch.tensor([s.prompts[0][t]], device="cuda:0")]
        s.front(qkv, dev_(np.array([t], np.int32)), dev_(np.array([s.slot(0, t)], np.int32)))
        out = torch.empty((1, s.H * s.hd), dtype=torch.float16, device="cuda:0")
        s.attn(qkv, d["table"], dev_(np.array([t + 1], np.int32)), out, s.ws(1))
        # two results, each within 2^-10 of weights times values (|v| < 4) and one rounding
        assert np.all(np.abs(host(out)[0] - chunk[t]) <= 2 * (2.0 ** -10 * 4 + 2.0 ** -11 * 4))
