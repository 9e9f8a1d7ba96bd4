"""CPU checks of the batched serving entry points: what they refuse, before any
HIP call is made, and the workspace sizes they ask for."""
import ctypes

import pytest

import jllm

INVALID = -1
A = 1 << 20          # an aligned address that is never read: every call here is refused first


def front(**kw):
    a = dict(q_out=A, q_out_stride=4096, q=A, q_stride=4096, k=A, k_stride=1024, v=A, v_stride=1024, q_norm=A,
             k_norm=A, norm_fp32=1, eps=1e-6, k_pages=A, v_pages=A, k_scales=A, v_scales=A, n_slots=1024,
             positions=A, slots=A, n_heads=32, n_kv=8, hd=128, chd=128, N=4, theta=1e6, neox=1, kv_int8=1,
             stream=None)
    assert not set(kw) - set(a)
    a.update(kw)
    return jllm.lib().jllm_hip_qk_norm_rope_store_kv_paged(*a.values())


@pytest.mark.parametrize("kw", [
    dict(N=-1), dict(n_heads=0), dict(n_kv=0), dict(n_heads=5000), dict(n_slots=-1), dict(n_slots=1 << 31),
    dict(hd=0), dict(hd=12), dict(hd=136), dict(chd=120), dict(chd=132), dict(chd=132, kv_int8=0),
    dict(theta=0.0), dict(theta=-1.0), dict(theta=float("inf")), dict(theta=float("nan")), dict(eps=-1e-6),
    dict(eps=float("nan")), dict(q_stride=4095), dict(q_stride=4098), dict(q_out_stride=4092), dict(k_stride=1020),
    dict(v_stride=1022), dict(q_out_stride=4100), dict(q=None), dict(q_out=None), dict(k=None), dict(v=None),
    dict(k_pages=None), dict(v_pages=None), dict(positions=None), dict(slots=None), dict(q_norm=None),
    dict(k_norm=None), dict(k_scales=None), dict(v_scales=None), dict(q=A + 2), dict(k=A + 4), dict(v=A + 2),
    dict(q_out=A + 4), dict(k_pages=A + 8), dict(v_pages=A + 4), dict(positions=A + 2), dict(slots=A + 1),
    dict(k_scales=A + 2), dict(q_norm=A + 2), dict(k_norm=A + 1, norm_fp32=0), dict(N=2 ** 31 - 1),
    dict(hd=128, q_stride=0, q_out_stride=0)])
def test_front_refuses(kw):
    assert front(**kw) == INVALID


def test_front_no_tokens():
    assert front(N=0, q=None, slots=None) == 0


def attn(**kw):
    a = dict(out=A, q=A, q_stride=4096, k_pages=A, v_pages=A, k_scales=A, v_scales=A, n_pages=64, page_size=16,
             table=A, table_stride=64, lens=A, B=2, n_heads=32, n_kv=8, hd=128, chd=128, max_seq=1024, scale=0.1,
             kv_int8=1, window=0, ws=A, ws_bytes=1 << 40, stream=None)
    assert not set(kw) - set(a)
    a.update(kw)
    return jllm.lib().jllm_hip_flash_attention_decode_paged(*a.values())


@pytest.mark.parametrize("kw", [
    dict(B=-1), dict(B=65536), dict(n_heads=0), dict(n_kv=0), dict(n_heads=30), dict(n_heads=136),
    dict(n_heads=8192, n_kv=512, q_stride=1 << 20), dict(hd=48), dict(hd=0), dict(hd=160, chd=160, q_stride=5120),
    dict(chd=96), dict(chd=136), dict(page_size=8), dict(page_size=24), dict(page_size=0), dict(page_size=8192),
    dict(n_pages=-1), dict(n_pages=1 << 27), dict(table_stride=63), dict(max_seq=-1), dict(max_seq=1025),
    dict(window=-1), dict(q_stride=4095), dict(q_stride=4100), dict(q_stride=2048), dict(scale=float("nan")),
    dict(scale=float("inf")), dict(out=None), dict(q=None), dict(lens=None), dict(table=None), dict(k_pages=None),
    dict(v_pages=None), dict(out=A + 8), dict(q=A + 8), dict(k_pages=A + 8), dict(v_pages=A + 8), dict(lens=A + 2),
    dict(table=A + 1), dict(k_scales=A + 2), dict(v_scales=A + 1)])
def test_attention_refuses(kw):
    assert attn(**kw) == INVALID


def test_attention_no_rows():
    assert attn(B=0, out=None, q=None, ws=None, ws_bytes=0) == 0


WS = [(1, 32, 8, 128, 131072, 0), (48, 32, 8, 128, 4096, 0), (17, 12, 1, 96, 5000, 1024), (1, 32, 8, 128, 1, 0),
      (65535, 16, 1, 32, 1 << 20, 0), (3, 4, 4, 64, 2 ** 31 - 1, 0)]


@pytest.mark.parametrize("size", WS)
def test_attention_workspace(size):
    f = jllm.lib().jllm_hip_flash_attention_decode_paged_workspace
    need = f(*size)
    assert need >= 0 and need % 16 == 0
    B, H, KV, hd, seq, window = size
    if need:
        kw = dict(B=B, n_heads=H, n_kv=KV, hd=hd, chd=hd, max_seq=seq, window=window, q_stride=H * hd,
                  table_stride=(seq + 15) // 16)
        assert attn(ws=None, **kw) == INVALID
        assert attn(ws=A + 8, **kw) == INVALID
        assert attn(ws_bytes=need - 1, **kw) == INVALID
        assert attn(ws_bytes=0, **kw) == INVALID


@pytest.mark.parametrize("bad", [(-1, 32, 8, 128, 10, 0), (1, 31, 8, 128, 10, 0), (1, 32, 8, 100, 10, 0),
                                 (1, 32, 8, 128, -1, 0), (1, 32, 8, 128, 10, -1), (1, 32, 0, 128, 10, 0)])
def test_attention_workspace_refuses(bad):
    assert jllm.lib().jllm_hip_flash_attention_decode_paged_workspace(*bad) == INVALID


def logits(**kw):
    a = dict(out=A, out_stride=1000, x=A, x_stride=1000, B=2, V=1000, tokens=A, token_stride=64, n_prompt=A,
             n_tokens=A, rep=A, freq=A, pres=A, bias_ids=A, bias=A, bias_stride=8, n_bias=A, mask=A, mask_stride=32,
             next_token=A, ws=A, ws_bytes=1 << 40, stream=None)
    assert not set(kw) - set(a)
    a.update(kw)
    return jllm.lib().jllm_hip_logits_process(*a.values())


@pytest.mark.parametrize("kw", [
    dict(B=-1), dict(B=65536), dict(V=0), dict(V=-5), dict(out_stride=999), dict(x_stride=999), dict(n_tokens=None),
    dict(token_stride=-1), dict(token_stride=1 << 31), dict(bias=None), dict(n_bias=None), dict(bias_stride=-1),
    dict(mask_stride=31), dict(out=None), dict(x=None), dict(x_stride=1004), dict(out=A + 2), dict(tokens=A + 2),
    dict(mask=A + 1), dict(rep=A + 3), dict(bias=A + 2), dict(next_token=A + 2), dict(bias_stride=1 << 31)])
def test_logits_refuses(kw):
    assert logits(**kw) == INVALID


def test_logits_no_rows():
    assert logits(B=0, out=None, x=None) == 0


@pytest.mark.parametrize("B,V", [(1, 151936), (64, 151936), (65535, 500), (3, 2 ** 31 - 1)])
def test_logits_workspace(B, V):
    need = jllm.lib().jllm_hip_logits_process_workspace(B, V)
    assert need >= 0 and need % 8 == 0
    if need:
        kw = dict(B=B, V=V, out_stride=V, x_stride=V, mask_stride=(V + 31) // 32)
        assert logits(ws=None, **kw) == INVALID
        assert logits(ws=A + 4, **kw) == INVALID
        assert logits(ws_bytes=need - 8, **kw) == INVALID


def test_logits_workspace_refuses():
    f = jllm.lib().jllm_hip_logits_process_workspace
    assert f(-1, 10) == f(65536, 10) == f(1, 0) == INVALID


def test_workspace_results_are_64_bit():
    lib = jllm.lib()
    for n in ("jllm_hip_flash_attention_decode_paged_workspace", "jllm_hip_logits_process_workspace"):
        assert getattr(lib, n).restype is ctypes.c_int64
