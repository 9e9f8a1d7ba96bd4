"""GPU parity of the product of 8-bit codes with its documented order of operations, bit by
bit in every form: the exact sum rounded to fp32, times the token's scale, times the
channel's, plus the bias, each rounded to fp32, and fp16 outputs once more.  So a token's
outputs do not depend on the tokens beside it.  No tolerance."""
import numpy as np
import pytest
import torch

import jllm
from gpu_util import print_case
from test_layer_i8_gpu import codes_of, gemm_call
from test_serving_gpu import dev_, host, rng

pytestmark = pytest.mark.gpu

# few tokens (three forms), tiles of 256 x 256 in rounds and alone, 128 x 256, 128 x 128, 64 x 64,
# 32 x 64, each with rows that are whole 16-byte pieces and with rows that are not, and with K cut
FORMS = [(1030, 3, 4112), (16400, 3, 48), (35, 5, 8192), (6691, 1253, 144), (6696, 1253, 144), (4099, 4300, 272),
         (4104, 4300, 272), (32003, 251, 272), (32008, 251, 272), (2700, 2001, 400), (2704, 2001, 400), (2049, 1030, 656),
         (2056, 1030, 656), (8001, 251, 1040), (8008, 251, 1040), (903, 900, 400), (904, 900, 400), (100, 40, 400), (104, 40, 400),
         (70, 4618, 10704), (2705, 67, 8416), (47, 31, 20016), (48, 31, 20016)]


def in_order(x, xs, w, ws, bias, fp32):
    s = np.matmul(x.astype(np.float64), w.astype(np.float64).T).astype(np.float32)
    y = s * xs[:, None] * ws
    y = y if bias is None else y + bias
    assert y.dtype == np.float32
    return y if fp32 else y.astype(np.float16)


@pytest.mark.parametrize("M,N,K", FORMS)
@pytest.mark.parametrize("fp32,bias", [(True, True), (False, True), (False, False)])
def test_gemm_rounds_in_order(dev, M, N, K, fp32, bias):
    print_case("gemm i8 in order", M, N, K, fp32, bias)
    g = rng(M, N, K)
    (x, xs), (w, ws) = codes_of(g, N, K), codes_of(g, M, K)
    # (biases of the outputs' size: that is where a product that is not rounded shows)
    b = (g.standard_normal(M) * 100).astype(np.float32) if bias else None
    got = gemm_call(x, xs, w, ws, b, fp32)
    want = in_order(x, xs, w, ws, b, fp32)
    assert np.array_equal(got, want), int((got != want).sum())


@pytest.mark.parametrize("N", [3, 20, 90])
def test_gemm_far_rows_round_in_order(dev, N):
    """Rows of codes 2^23 bytes apart, which have a form of their own."""
    g = rng(N)
    M, K, step = 70, 96, 1 << 23
    (x, xs), (w, ws) = codes_of(g, N, K), codes_of(g, M, K)
    b = (g.standard_normal(M) * 10).astype(np.float32)
    big = torch.zeros((M * step,), dtype=torch.int8, device="cuda:0")
    big.view(M, step)[:, :K] = dev_(w)
    y = torch.zeros((N, M), dtype=torch.float32, device="cuda:0")
    need = jllm.lib().jllm_hip_gemm_i8_workspace(M, N, K)
    t = [dev_(a) for a in (x, xs, ws, b)]
    space = torch.zeros((max(need, 16),), dtype=torch.uint8, device="cuda:0")
    jllm.call("jllm_hip_gemm_i8", y, M, 1, t[0], K, t[1], big, step, t[2], t[3], M, N, K, space, need)
    assert np.array_equal(host(y), in_order(x, xs, w, ws, b, True))
