"""Where the int8 operators round, and how far: the quantised integer for every bf16 significand, the rows whose norm
leaves fp32, and the GELU of the instructions in use."""

import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from test_int8_gpu import EPS, gen, normal, ops  # noqa: E402, F401

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24


@pytest.mark.parametrize("e", [-100, -20, 0, 100, 118])
def test_quantize_every_significand(ops, e):  # noqa: F811
    """A row for each significand of amax, holding every bf16 value down to 2^-10 of it: q is the fp32 product rounded,
    and the integer next to the exact quotient; of exact halves only amax / 2 may miss the even one."""
    m = np.arange(128, 256)
    x = np.concatenate([np.arange(128, 256) * 2.0 ** -j for j in range(11)])
    x = np.where(x[None] <= m[:, None], x[None], m[:, None])
    x[:, 0] = m
    want = np.rint((x * 2.0 ** e).astype(np.float32)
                   * ((np.float32(1) / (m * 2.0 ** e).astype(np.float32)) * np.float32(127))[:, None])
    q, scale = ops.quantize_int8(torch.from_numpy(x * 2.0 ** e).cuda().bfloat16())
    q = q.cpu().numpy().astype(np.float64)
    assert (q == want).all()
    assert (scale.cpu().numpy() == (m * 2.0 ** e).astype(np.float32) / np.float32(127)).all()
    exact = x * 127  # times 1 / m, kept as a fraction: all of it is exact in fp64
    twice = np.abs(2 * (q * m[:, None] - exact))
    assert (twice <= m[:, None]).all()  # |q - exact / m| <= 1 / 2
    odd = (twice == m[:, None]) & (q % 2 != 0)
    assert (2 * x == m[:, None])[odd].all()
    assert len(set(m[odd.any(1)])) == 20


@pytest.mark.parametrize("k", [700, 4096, 8192, 40000])
@pytest.mark.parametrize("residual", [False, True])
def test_norm_overflow_bound(ops, k, residual):  # noqa: F811
    """A row of equal values v has a norm up to K v^2 = 3.4e38 and counts as not finite beyond."""
    top = math.sqrt(3.4028e38 / k)
    v = torch.tensor([0.97 * top, 1.03 * top, 1.0], device="cuda").bfloat16()[:, None].expand(3, k).contiguous()
    gamma = torch.ones(k, dtype=torch.bfloat16, device="cuda")
    q, scale = ops.rmsnorm_int8(v, gamma, EPS, residual=torch.zeros_like(v) if residual else None)[:2]
    assert scale[1].isnan() and (q[1] == 0).all()
    assert (q[[0, 2]] == 127).all()
    # the norm of a constant row is 1: 60 U32 for the sum, the root and the divisions, EPS beside 1 in the last row
    assert ((scale[[0, 2]] - 1 / 127).abs() <= (60 * U32 + EPS) / 127).all()


def test_norm_product_overflow(ops):  # noqa: F811
    """The norm is finite, its product with gamma is not before the division."""
    x = torch.full((2, 64), 1e10, device="cuda").bfloat16()
    x[1] = 1.0
    gamma = torch.full((64,), 1e30, device="cuda").bfloat16()
    q, scale = ops.rmsnorm_int8(x, gamma, EPS)
    assert scale[0].isnan() and (q[0] == 0).all()
    assert torch.isfinite(scale[1]) and (q[1] == 127).all()


@pytest.mark.parametrize("m", [1, 8, 40, 200])
def test_tanh_gelu_error(ops, m):  # noqa: F811
    """x / (1 + 2^a), a = x (k1 + k2 x^2): a is off by 4 U32 of itself (x^2 and k2 1 each beside k1's 1, the sum 1,
    the product 1), which moves 2^a by 4 |2 z| U32, z = a's tanh argument; ex2.approx by 2^-22 = 4 U32. The sum adds 1,
    the reciprocal 2 (1 ulp), the product 1. A reciprocal below 2^-126 is 0."""
    n, k = 4096, 16
    g = gen(m)
    a = torch.zeros(m, k, dtype=torch.int8, device="cuda")
    a[:, 0] = 1
    b = torch.zeros(n, k, dtype=torch.int8, device="cuda")
    b[:, 0] = torch.randint(-127, 128, (n,), generator=g, device="cuda", dtype=torch.int8)
    sa = 10 ** (normal(g, m) * 0.5)
    sb = 10 ** (normal(g, n) * 0.8 - 2)
    x = ((b[:, 0].float()[None] * sa[:, None]) * sb).double()  # the kernel's own roundings
    y = ops.matmul_int8(a, sa, b, sb, gelu="tanh", out_dtype=torch.float32).double()
    z2 = 2 * math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3)
    ref = x * torch.sigmoid(z2)
    tol = ref.abs() * (8 + 4 * z2.abs()) * 1.01 * U32 + x.abs() * 2.0 ** -125
    bad = ~((y - ref).abs() <= tol)
    assert not bad.any(), f"{int(bad.sum())} off, worst {((y - ref).abs() / tol).max():.3g} x"
