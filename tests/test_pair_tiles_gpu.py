"""The bf16 CTA-pair kernel on short tiles: over more than one wave of the 74 pairs, with a last column tile that ends
after an odd number of 32-column blocks, so that the next tile's results are staged right behind it.

Tolerance: K fp32 sums of exact bf16 products, each sum off by at most 2^-24 of the sum of magnitudes, doubled for an
accumulator that truncates; then one rounding to bf16.
"""

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m,n,k", [(8192, 4128, 64), (4500, 8288, 64), (12000, 352, 600), (9000, 544, 200),
                                   (8192, 2208, 128)])
def test_matmul_short_tiles(m, n, k):
    from tfb200 import ops

    g = torch.Generator(device="cuda").manual_seed(m + n + k)
    a = torch.randn(m, k, generator=g, device="cuda").bfloat16()
    b = torch.randn(k, n, generator=g, device="cuda").bfloat16()
    y = ops.matmul(a, b)
    ref = a.double() @ b.double()
    tol = 2 * k * 2.0 ** -24 * (a.double().abs() @ b.double().abs())
    tol = tol + (tol + ref.abs()) * 2.0 ** -8
    assert ((y.double() - ref).abs() <= tol).all()
    gamma = torch.ones(k, dtype=torch.bfloat16, device="cuda")
    z = ops.fused_rmsnorm_matmul(a, gamma, b, 1e-5)
    for _ in range(20):
        assert torch.equal(ops.matmul(a, b), y)
        assert torch.equal(ops.fused_rmsnorm_matmul(a, gamma, b, 1e-5), z)
