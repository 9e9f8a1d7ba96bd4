"""GPU parity of decode attention over a shared prefix at the ends of its ranges, against
numpy in float64.  Tolerances as test_paged_prefix_gpu's."""
import numpy as np
import pytest
import torch

import jllm
from gpu_util import print_case
from test_paged_prefix_gpu import call, pool, queries, reference
from test_serving_gpu import attn_ref, dev_, host, rng

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("B,G", [(4, 4), (5, 12), (9, 16), (18, 16)])
@pytest.mark.parametrize("P,longest", [(1500000000, 1200000000), (2 ** 31 - 1, 2 ** 31 - 1), (2 ** 31 - 1, 70)])
def test_prefix_and_own_tokens_past_31_bits_in_a_window(dev, int8, B, G, P, longest):
    """A prefix and a row's own tokens that together pass 2^31, seen through a window (the page
    tables name the same few pages again and again): that row leaves the others their share of
    the prefix."""
    hd, page, window = 64, 4096, 100
    print_case("prefix past 31 bits", int8, B, G, P, longest)
    g = rng(B, G, P, longest)
    n_pages = 6
    kp, vp = [g.integers(-127, 128, (n_pages, page, 1, hd)).astype(np.int8) if int8 else
              g.standard_normal((n_pages, page, 1, hd)).astype(np.float16) for _ in range(2)]
    ks, vs = [(g.random((n_pages, page, 1)) * 0.02 + 0.005).astype(np.float32) for _ in range(2)]
    width = (longest + page - 1) // page
    prefix_table = g.integers(0, n_pages, (P + page - 1) // page).astype(np.int32)
    table = g.integers(0, n_pages, (B, width)).astype(np.int32)
    lens = np.array([longest, 0, 40, -1, 99, 100, 101, 1, 7][:B] + [3] * (B - 9), np.int32)
    lens = np.minimum(lens, longest)
    max_prefix, max_seq = P, longest
    q = queries(g, B, G, hd)
    out = torch.full((B, G * hd), 7.0, dtype=torch.float16, device="cuda:0")
    need = jllm.lib().jllm_hip_flash_attention_decode_paged_prefix_workspace(B, G, 1, hd, max_prefix, max_seq, window)
    d = [dev_(a) for a in (q, kp, vp, ks, vs, prefix_table, np.array([P], np.int32), table, lens)]
    ws = torch.full((need,), 0xFF, dtype=torch.uint8, device="cuda:0")
    jllm.call("jllm_hip_flash_attention_decode_paged_prefix", out, d[0], G * hd, d[1], d[2], d[3] if int8 else None,
              d[4] if int8 else None, n_pages, page, d[5], d[6], max_prefix, d[7], width, d[8], B, G, 1, hd, hd, max_seq,
              0.1, int(int8), window, ws, need)
    got = host(out).reshape(B, G, hd).astype(np.float64)
    k64, v64 = [(a * s[..., None].astype(np.float64) if int8 else a.astype(np.float64)).reshape(-1, 1, hd)
                for a, s in ((kp, ks), (vp, vs))]

    def slots(ids, pos):
        return ids[pos // page].astype(np.int64) * page + pos % page

    for b, n in enumerate(lens.tolist()):
        if n < 0:
            assert not got[b].any()
            continue
        lo = max(0, P + n - window)
        at = np.concatenate([slots(prefix_table, np.arange(min(lo, P), P)), slots(table[b], np.arange(max(0, lo - P), n))])
        assert len(at) == window
        want, size = attn_ref(q[b].reshape(G, hd).astype(np.float64), k64[at], v64[at], float(np.float32(0.1)), 0, window)
        tol = 2.0 ** -11 * np.abs(want) + 2.0 ** -10 * size + 2.0 ** -25
        assert np.all(np.abs(got[b] - want) <= tol), (b, float((np.abs(got[b] - want) / tol).max()))


@pytest.mark.parametrize("scale", [-0.09, 2.0])
@pytest.mark.parametrize("B,G", [(20, 4), (17, 8), (40, 16)])
def test_prefix_int8_codes_through_lds_are_exact(dev, scale, B, G):
    """Of more than 64 columns the prefix's INT8 codes meet the weights as they are, without the
    128 that the form for few columns adds and takes off: what that may leave, 2 n 2^-24 255
    max |vs| over n keys, remains for a row's own 7 keys alone."""
    print_case("prefix exact codes", scale, B, G)
    g = rng(B, G, 9)
    p = pool(g, 333, [7] * B, 1, 64, 16, True).upload()
    q = queries(g, B, G, 64)
    offset = 2 * 7 * 2.0 ** -24 * 255 * np.nanmax(p.vs)
    got = host(call(p, dev_(q), G, scale)).reshape(B, G, 64).astype(np.float64)
    for b, (want, size) in enumerate(reference(p, q, G, scale)):
        assert np.all(np.abs(got[b] - want) <= 2.0 ** -11 * np.abs(want) + 2.0 ** -10 * size + 2.0 ** -25 + offset), b
