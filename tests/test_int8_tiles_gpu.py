"""int8 products of more than 128 rows whose CTA pairs run through several output tiles in quick succession.

A short inner dimension makes a tile's products short, so the next tile's epilogue follows at once on the last one's:
accumulators, column scales and the buffers that results are staged in change hands as fast as they ever do. The shapes
take 64-, 128- and 256-column tiles over more than one wave of the 74 pairs of CTAs, with last column tiles that end
after an odd number of 32-column blocks.
"""

import pytest

torch = pytest.importorskip("torch")

from test_int8_gpu import EPS, aligned, check, gen, mlp64, normal, operands, ops, product64, weight  # noqa: E402, F401

pytestmark = pytest.mark.gpu

# (M, N, K)
TILES = [
    # 64 columns: one block for each epilogue warp
    (2048, 2368, 128), (8192, 512, 64), (8192, 448, 100), (1000, 3000, 200), (16384, 96, 256), (4100, 1056, 16),
    # 128 columns, an odd last block
    (6000, 1120, 200), (8192, 608, 384), (12000, 352, 600),
    # 256 columns, an odd last block
    (8192, 4128, 100), (4500, 8288, 64),
]


@pytest.mark.parametrize("m,n,k", TILES)
def test_matmul_short_tiles(ops, m, n, k):  # noqa: F811
    a, sa, b, sb, bias, res = operands(m + 7 * n + 13 * k, m, n, k)
    a, b = aligned(a), aligned(b)
    ref = product64(a, sa, b, sb)
    y = ops.matmul_int8(a, sa, b, sb)
    check(y, ref)
    check(ops.matmul_int8(a, sa, b, sb, out_dtype=torch.float32), product64(a, sa, b, sb, dtype=torch.float32))
    z = ops.matmul_int8(a, sa, b, sb, bias=bias, gelu="tanh", residual=res)
    check(z, product64(a, sa, b, sb, bias, "tanh", res))
    for _ in range(20):
        assert torch.equal(ops.matmul_int8(a, sa, b, sb), y)
        assert torch.equal(ops.matmul_int8(a, sa, b, sb, bias=bias, gelu="tanh", residual=res), z)


@pytest.mark.parametrize("m,k,h,n", [(8192, 64, 512, 96), (2048, 128, 2368, 64), (8192, 100, 448, 100),
                                     (12000, 600, 352, 128), (8192, 100, 4128, 64)])
def test_mlp_short_tiles(ops, m, k, h, n):  # noqa: F811
    """The up projection of these has such tiles, the down projection of some."""
    g = gen(k + n + h)
    x, gamma = normal(g, m, k).bfloat16(), (torch.rand(k, generator=g, device="cuda") + 0.5).bfloat16()
    w1, s1 = weight(ops, g, h, k)
    w2, s2 = weight(ops, g, n, h)
    b1, res = (normal(g, h) * 0.1).bfloat16(), normal(g, m, n).bfloat16()
    y = ops.fused_mlp_int8(x, gamma, w1, s1, b1, w2, s2, res, EPS, gelu="tanh")
    q, scale = ops.rmsnorm_int8(x, gamma, EPS)
    check(y, mlp64(q, scale, w1, s1, b1, w2, s2, res, "tanh"))
    for _ in range(20):
        assert torch.equal(ops.fused_mlp_int8(x, gamma, w1, s1, b1, w2, s2, res, EPS, gelu="tanh"), y)
