"""The int8 MLP call is its parts: RMSNorm to int8, a product with GELU in fp32, its rows quantised, a product with the
residual. The hidden rows are quantised here in the same fp32 roundings, so the result is the same bit for bit."""

import pytest

torch = pytest.importorskip("torch")

from test_int8_gpu import EPS, gen, normal, ops, weight  # noqa: E402, F401

pytestmark = pytest.mark.gpu


def quantise_fp32(h):
    amax = h.abs().amax(1)
    q = torch.round(h * (amax.reciprocal() * 127.0)[:, None])  # fp32: reciprocal, product, product
    return q.to(torch.int8), amax / torch.full_like(amax, 127.0)


@pytest.mark.parametrize("m,k,h,n", [(1, 256, 1024, 256), (2, 100, 333, 50), (7, 512, 5000, 96), (16, 1024, 4096, 1024),
                                     (24, 300, 1001, 300), (40, 2048, 8192, 2048), (100, 512, 2056, 512),
                                     (129, 256, 700, 256), (300, 1024, 16400, 512), (1100, 640, 2050, 640),
                                     (3, 64, 33000, 64), (200, 64, 40004, 64), (150, 96, 32768, 64)])
@pytest.mark.parametrize("gelu,with_bias", [("erf", True), ("tanh", False)])
def test_mlp_is_its_parts(ops, m, k, h, n, gelu, with_bias):  # noqa: F811
    g = gen(m + k + h)
    x, gamma = normal(g, m, k).bfloat16(), (torch.rand(k, generator=g, device="cuda") + 0.5).bfloat16()
    w1, s1 = weight(ops, g, h, k)
    w2, s2 = weight(ops, g, n, h)
    b1 = (normal(g, h) * 0.1).bfloat16() if with_bias else None
    res = normal(g, m, n).bfloat16()
    q, scale = ops.rmsnorm_int8(x, gamma, EPS)
    hidden = ops.matmul_int8(q, scale, w1, s1, bias=b1, gelu=gelu, out_dtype=torch.float32)
    hq, hs = quantise_fp32(hidden)
    want = ops.matmul_int8(hq, hs, w2, s2, residual=res)
    assert torch.equal(ops.fused_mlp_int8(x, gamma, w1, s1, b1, w2, s2, res, EPS, gelu=gelu), want)
