"""GPU checks of calls of the batched serving operators at the ends of what their
header allows: the largest batches, no pages, no keys, pages that several places
share, scores scaled by zero or below it.  References and tolerances are those of
test_serving_gpu.
"""
import numpy as np
import pytest
import torch

import jllm
from gpu_util import print_case
from test_serving_gpu import Pool, attn_call, attn_check, dev_, host, logits_call, logits_ref, rng, same

pytestmark = pytest.mark.gpu


def shared_rows(g, B, KV, hd, int8, page=16, n=48):
    """B rows over one sequence's pages, with lengths of their own."""
    p = Pool(g, [n], KV, hd, page, int8)
    lens = g.integers(0, n + 1, B)
    p.table = np.repeat(p.table, B, 0)
    p.k, p.v, p.lens = p.k * B, p.v * B, [int(x) for x in lens]
    return p.upload()


@pytest.mark.parametrize("int8", [False, True])
def test_attention_largest_batch(dev, int8):
    print_case("65535 rows", int8)
    g = rng(1, int8)
    p = shared_rows(g, 65535, 1, 32, int8)
    q = g.standard_normal((65535, 32)).astype(np.float16)
    got = host(attn_call(p, dev_(q), 1, 0.2))
    # rows of every length from all over the batch, the first and the last
    at = np.unique(np.r_[0, 65534, g.integers(0, 65535, 3000)])
    p.k, p.v = [p.k[b] for b in at], [p.v[b] for b in at]
    attn_check(p, got[at], q[at], 1, 0.2, lens=[p.lens[b] for b in at])


def test_logits_largest_batch(dev):
    print_case("65535 rows of logits")
    g = rng(2)
    x = g.standard_normal((65535, 37)).astype(np.float32)
    c = {"mask": g.integers(0, 2 ** 32, (65535, 2), dtype=np.uint32)}
    got, t = logits_call(x, c)
    bits = ((c["mask"][:, :, None] >> np.arange(32, dtype=np.uint32)) & 1).reshape(65535, -1)[:, :37]
    want = np.where(bits == 1, x, -np.inf).astype(np.float32)
    assert same(got, want)
    assert np.array_equal(t, np.where(bits.any(-1), want.argmax(-1), -1))


@pytest.mark.parametrize("max_seq", [100, 5000])
@pytest.mark.parametrize("int8", [0, 1])
def test_attention_without_pages_or_keys(dev, max_seq, int8):
    """A pool of no pages: every key is skipped.  No key at all: no table either."""
    print_case("no pages", max_seq, int8)
    H, KV, hd, B = 8, 2, 64, 3
    f = jllm.lib().jllm_hip_flash_attention_decode_paged_workspace
    q = dev_(rng(3).standard_normal((B, H * hd)).astype(np.float16))
    table = torch.zeros((B, max_seq), dtype=torch.int32, device="cuda:0")
    lens = dev_(np.array([max_seq, 1, 0], np.int32))
    for table, seq in ((table, max_seq), (None, 0)):
        out = torch.full((B, H * hd), 7.0, dtype=torch.float16, device="cuda:0")
        ws = torch.full((max(f(B, H, KV, hd, seq, 0), 16),), 0xFF, dtype=torch.uint8, device="cuda:0")
        jllm.call("jllm_hip_flash_attention_decode_paged", out, q, H * hd, None, None, None, None, 0, 16, table, max_seq,
                  lens, B, H, KV, hd, hd, seq, 0.125, int8, 0, ws, ws.numel())
        assert not host(out).any()


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("n", [90, 3000])
def test_attention_a_page_in_several_places(dev, int8, n):
    """One page twice in a sequence, and in several sequences."""
    print_case("pages shared", int8, n)
    H, KV, hd, page = 8, 2, 64, 16
    g = rng(4, n)
    p = Pool(g, [n, n, 40], KV, hd, page, int8)
    p.table[1] = p.table[0]
    p.table[1, 1] = p.table[1, 3]
    p.table[2, :2] = p.table[0, 2]
    k, v = p.k[0].copy(), p.v[0].copy()
    k[16:32], v[16:32] = p.k[0][48:64], p.v[0][48:64]
    p.k[1], p.v[1] = k, v
    for x, y in ((p.k, p.k[0]), (p.v, p.v[0])):
        x[2] = np.concatenate([y[32:48], y[32:48], x[2][32:]])
    p.upload()
    q = g.standard_normal((3, H * hd)).astype(np.float16)
    attn_check(p, host(attn_call(p, dev_(q), H, 0.125)), q, H, 0.125)


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("scale", [0.0, -0.125])
@pytest.mark.parametrize("lens", [[1, 33, 0, 300], [2500, 17]])
def test_attention_scale_of_zero_or_below(dev, int8, scale, lens):
    print_case("scale", int8, scale, lens)
    H, KV, hd = 8, 2, 64
    g = rng(5, len(lens))
    p = Pool(g, lens, KV, hd, 16, int8).upload()
    q = g.standard_normal((len(lens), H * hd)).astype(np.float16)
    attn_check(p, host(attn_call(p, dev_(q), H, scale)), q, H, scale)


@pytest.mark.parametrize("drop", [False, True])
def test_logits_lists_of_no_width(dev, drop):
    """Lists with a stride of 0 hold nothing, whatever the counts say."""
    g = rng(6)
    x = g.standard_normal((3, 3000)).astype(np.float32)
    c = {"tokens": np.zeros((3, 0), np.int32), "n_tokens": np.array([5, 0, 2 ** 31 - 1], np.int32),
         "bias_ids": np.zeros((3, 0), np.int32), "bias": np.zeros((3, 0), np.float32),
         "n_bias": np.array([1, 7, -1], np.int32)}
    some = {k: np.zeros((3, 1), v.dtype) if v.ndim == 2 else v for k, v in c.items()}    # (arrays that have an address)
    d = {k: dev_(v) for k, v in some.items()}
    out, tok = torch.empty((3, 3000), device="cuda:0"), torch.empty((3,), dtype=torch.int32, device="cuda:0")
    ws = torch.empty((max(jllm.lib().jllm_hip_logits_process_workspace(3, 3000), 16),), dtype=torch.uint8, device="cuda:0")
    jllm.call("jllm_hip_logits_process", out, 3000, dev_(x), 3000, 3, 3000, d["tokens"], 0, None, d["n_tokens"], None, None,
              None, None if drop else d["bias_ids"], d["bias"], 0, d["n_bias"], None, 0, tok, ws, ws.numel())
    want, t = logits_ref(x, {})
    assert same(host(out), want) and np.array_equal(host(tok), t)
