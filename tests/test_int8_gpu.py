"""The 8-bit integer operators against their definitions in 64 bits.

Tolerances come from the arithmetic, each rounding off by at most half a step
(U32 = 2^-24 relative in fp32, half an eps of the output type):

* q = rn(v) with v = t * 127 / amax evaluated in fp32: |q - v| <= 1/2 plus v's
  own error, ROUNDINGS * U32 * 127.
* The integer sums are exact; scale, bias, GELU and residual add a few U32 of
  their operands, and the output one rounding.
"""

import math

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24
EPS = 1e-5


@pytest.fixture(scope="module")
def ops():
    assert torch.cuda.is_available()
    from tfb200 import ops as _ops

    return _ops


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def ints(g, *shape, lo=-127, hi=128):
    return torch.randint(lo, hi, shape, generator=g, device="cuda", dtype=torch.int8)


def rows_at(t, offset, ld):
    """The matrix t in a buffer that starts `offset` elements after an aligned address, rows `ld` apart; the
    elements around it hold a pattern."""
    m, k = t.shape
    buf = torch.full((offset + m * ld + 8,), 77, dtype=t.dtype, device=t.device)
    v = buf[offset:offset + m * ld].view(m, ld)[:, :k]
    v.copy_(t)
    return v, buf


def check_q(q, scale, t64, scale64, roundings, sum_roundings=0):
    v = t64 * (127.0 / t64.abs().amax(-1, keepdim=True))
    assert (q.double() - v).abs().max().item() <= 0.5 + 127 * roundings * U32
    assert (q.double().abs().amax(-1) == 127).all()
    assert ((scale.double() - scale64).abs() <= scale64 * (roundings + sum_roundings) * U32).all()


def norm64(x, gamma, residual=None, eps=EPS):
    s = x.double() if residual is None else x.double() + residual.double()
    t = s * gamma.double()
    return s, t, t.abs().amax(-1) / torch.sqrt(s.pow(2).mean(-1) + eps) / 127.0


# (rows, K): one value, a warp's row, the borders between block sizes, odd widths, rows past a block's registers
ROWS = [(1, 1), (3, 7), (5, 8), (2, 1000), (1, 1024), (4, 1025), (7, 4096), (2, 4099), (3, 8200), (2, 16384),
        (33, 16392), (1, 28672), (2, 32768), (2, 32769), (3, 40008)]


@pytest.mark.parametrize("m,k", ROWS)
def test_quantize(ops, m, k):
    x = (normal(gen(m * 131 + k), m, k) * 3).bfloat16()
    q, scale = ops.quantize_int8(x)
    assert q.shape == x.shape and q.dtype == torch.int8 and scale.shape == (m,)
    assert q.stride(0) % 16 == 0 or m == 1
    # v: one division, one product.
    check_q(q, scale, x.double(), x.double().abs().amax(-1) / 127.0, 3)


@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("m,k", ROWS)
def test_rmsnorm(ops, m, k, residual):
    g = gen(m * 131 + k)
    x, gamma = normal(g, m, k).bfloat16(), (torch.rand(k, generator=g, device="cuda") + 0.5).bfloat16()
    r = (normal(g, m, k) * 2).bfloat16() if residual else None
    res = ops.rmsnorm_int8(x, gamma, EPS, residual=r)
    s, t, scale64 = norm64(x, gamma, r)
    # t: sum and product, in the value and in amax, then division and product. The sum of squares: the longest chain
    # is a thread's 64 terms and ten levels of the tree, halved by the root; root, division and products after it.
    check_q(res[0], res[1], t, scale64, 8, 50)
    if residual:
        assert torch.equal(res[2], (x.float() + r.float()).bfloat16())
    else:
        assert len(res) == 2


@pytest.mark.parametrize("k", [256, 259, 4096, 20000, 40008])
def test_quantize_ties(ops, k):
    """Values halfway between two steps go to the even one, whatever the row's scale: x = j / 2 * 2^e * c with amax
    127 * 2^e * c, all exact in bf16, lies j / 2 steps from zero."""
    j = torch.arange(k, device="cuda") % 255 - 127
    for e in (-100, -3, 0, 5, 90):
        x = (j.double() / 2 * 2.0 ** e).bfloat16()
        x[0] = 127 * 2.0 ** e
        q, scale = ops.quantize_int8(x.repeat(3, 1))
        want = torch.round(j.double() / 2)  # half to even
        want[0] = 127
        assert torch.equal(q[1].double(), want) and scale[1].double() == 2.0 ** e
    # amax = 4.03125: 127 / amax is not exact, 2.015625 is half of amax
    x = torch.full((2, k), 2.015625, device="cuda").bfloat16()
    x[:, 1] = -4.03125
    q, _ = ops.quantize_int8(x)
    assert (q[:, 0] == 64).all() and (q[:, 1] == -127).all()


@pytest.mark.parametrize("k", [64, 1000, 1001, 5000, 33000])
@pytest.mark.parametrize("offset,pad", [(0, 0), (1, 0), (8, 8), (3, 5)])
def test_rows_strides_and_surroundings(ops, k, offset, pad):
    g = gen(k)
    m = 6
    x, r = normal(g, m, k).bfloat16(), normal(g, m, k).bfloat16()
    gamma = (torch.rand(k + 1, generator=g, device="cuda") + 0.5).bfloat16()[offset % 2:][:k]
    want = ops.rmsnorm_int8(x.clone(), gamma.clone(), EPS, residual=r.clone())
    xv, _ = rows_at(x, offset, k + pad)
    rv, _ = rows_at(r, offset, k + pad)
    qv, qbuf = rows_at(torch.zeros(m, k, dtype=torch.int8, device="cuda"), offset, k + pad)
    sv, sbuf = rows_at(torch.zeros_like(x), offset, k + pad)
    scale = torch.empty(m, device="cuda")
    ops.rmsnorm_int8(xv, gamma, EPS, residual=rv, out=(qv, scale, sv))
    # The sum of squares is added in another order on other strides.
    assert torch.equal(qv, want[0]) and torch.equal(sv, want[2])
    assert torch.allclose(scale, want[1], rtol=100 * U32, atol=0)
    for buf, view in ((qbuf, qv), (sbuf, sv)):
        view.fill_(77)
        assert (buf == 77).all(), "wrote outside the rows"
    # In place: the sum over x.
    x2 = x.clone()
    q2, s2, t2 = ops.rmsnorm_int8(x2, gamma, EPS, residual=r, out=(torch.empty_like(want[0]), scale, x2))
    assert t2 is x2 and torch.equal(x2, want[2]) and torch.equal(q2, want[0])


@pytest.mark.parametrize("m,k", [(3000, 1), (3000, 9), (2500, 1001), (2500, 1032), (700, 4099), (700, 4104), (300, 16383)])
@pytest.mark.parametrize("offset", [0, 1, 5])
def test_rows_many_in_place(ops, m, k, offset):
    """Many rows of odd width, starting anywhere, the sum written over x; q in its usual layout."""
    g = gen(m + k)
    x, r = normal(g, m, k).bfloat16(), normal(g, m, k).bfloat16()
    gamma = (torch.rand(k, generator=g, device="cuda") + 0.5).bfloat16()
    s = x.float() + r.float()
    t = s * gamma.float()
    amax = t.abs().amax(1, keepdim=True)
    want = torch.where(amax > 0, torch.round(t * (127.0 / amax)), amax)  # the same fp32 roundings
    xv, xbuf = rows_at(x, offset, k)
    rv, _ = rows_at(r, offset, k)
    qp = torch.full((m, (k + 15) // 16 * 16), 77, dtype=torch.int8, device="cuda")
    scale = torch.empty(m, device="cuda")
    ops.rmsnorm_int8(xv, gamma, EPS, residual=rv, out=(qp[:, :k], scale, xv))
    assert torch.equal(qp[:, :k].float(), want) and torch.equal(xv, s.bfloat16())
    assert (qp[:, k:] == 77).all()
    assert (xbuf[:offset] == 77).all() and (xbuf[offset + m * k:] == 77).all()
    ref = amax[:, 0].double() / torch.sqrt(s.double().pow(2).mean(1) + EPS) / 127
    assert ((scale.double() - ref).abs() <= 60 * U32 * ref).all()
    xv.copy_(x)
    q, _ = ops.quantize_int8(xv)
    xa = x.float().abs().amax(1, keepdim=True)
    assert torch.equal(q.float(), torch.where(xa > 0, torch.round(x.float() * (127.0 / xa)), xa))


@pytest.mark.parametrize("k", [5, 256, 3001, 40000])
def test_rows_special_values(ops, k):
    x = normal(gen(k), 8, k).bfloat16()
    x[0] = 0
    x[1, k // 2] = float("inf")
    x[2, k - 1] = float("nan")
    x[3] = 0
    x[3, 0] = float("-inf")
    x[4] *= 1e-38  # 127 / amax is above the largest fp32
    x[5] = 2.0 ** -130  # subnormal in fp32
    x[6] = 3.0e38
    q, scale = ops.quantize_int8(x)
    assert (q[:4] == 0).all()
    assert scale[0] == 0 and scale[1:4].isnan().all()
    v = x.double() * (127.0 / x.double().abs().amax(-1, keepdim=True))
    assert ((q.double() - v)[4:].abs() <= 0.5 + 1e-4).all()
    assert (q[5:7] == 127).all()
    assert torch.isfinite(scale[4:]).all()
    gamma = torch.ones(k, device="cuda", dtype=torch.bfloat16)
    q, scale = ops.rmsnorm_int8(x, gamma, EPS)
    assert (q[:4] == 0).all() and scale[0] == 0 and scale[1:4].isnan().all()
    assert scale[6].isnan()  # the sum of squares leaves fp32
    assert torch.isfinite(scale[7]) and torch.isfinite(scale[4])
    # eps = 0: 0 / 0, as the bf16 operator's
    assert ops.rmsnorm_int8(x[:1], gamma, 0.0)[1].isnan().all()


@pytest.mark.parametrize("k", [5, 520, 3001, 8192, 40000])
def test_rows_without_a_norm(ops, k):
    """eps = 0: rows whose mean square is 0 in fp32 have no norm; the rows beside them do."""
    x = normal(gen(k), 4, k).bfloat16()
    x[1] = 0
    x[2] *= 1e-30  # its squares are below the smallest fp32
    gamma = torch.ones(k, device="cuda", dtype=torch.bfloat16)
    for residual in (None, torch.zeros_like(x)):
        q, scale = ops.rmsnorm_int8(x, gamma, 0.0, residual=residual)[:2]
        assert scale[1:3].isnan().all()
        for i in (0, 3):
            qi, si = ops.rmsnorm_int8(x[i:i + 1], gamma, 0.0)[:2]
            ref = norm64(x[i:i + 1], gamma, eps=0.0)[2]
            # one row alone may be summed over more threads: mean of squares, root and two divisions, and the sum
            assert ((scale[i] - ref).abs() <= 60 * U32 * ref).all() and ((si - ref).abs() <= 60 * U32 * ref).all()
            assert torch.equal(q[i:i + 1], qi)


def test_rows_empty_and_long_offsets(ops):
    q, scale = ops.quantize_int8(torch.empty(0, 64, dtype=torch.bfloat16, device="cuda"))
    assert q.shape == (0, 64) and scale.shape == (0,)
    q, scale = ops.quantize_int8(torch.empty(3, 0, dtype=torch.bfloat16, device="cuda"))
    assert q.shape == (3, 0) and (scale == 0).all()
    # Rows whose offsets pass 2^31 elements.
    ld, m, k = 1 << 28, 10, 520
    big = torch.empty(9 * ld + k, dtype=torch.bfloat16, device="cuda")
    x = torch.as_strided(big, (m, k), (ld, 1))
    x.copy_(normal(gen(5), m, k))
    assert torch.equal(ops.quantize_int8(x)[0], ops.quantize_int8(x.contiguous())[0])


def test_rows_batched_and_transposed(ops):
    g = gen(3)
    x = normal(g, 2, 3, 100).bfloat16()
    q, scale = ops.quantize_int8(x)
    assert q.shape == (2, 3, 100) and scale.shape == (2, 3)
    q2, s2 = ops.quantize_int8(x.reshape(6, 100))
    assert torch.equal(q.reshape(6, 100), q2) and torch.equal(scale.reshape(6), s2)
    w = normal(g, 100, 37).bfloat16()
    assert torch.equal(ops.quantize_int8(w.t())[0], ops.quantize_int8(w.t().contiguous())[0])
    e = normal(g, 1, 64).bfloat16().expand(5, 64)
    assert torch.equal(ops.quantize_int8(e)[0], ops.quantize_int8(e.contiguous())[0])


# ----------------------------------------------------------------- products


def gelu64(u, kind):
    if kind == "erf":
        return 0.5 * u * (1 + torch.erf(u / math.sqrt(2)))
    if kind == "tanh":
        return 0.5 * u * (1 + torch.tanh(math.sqrt(2 / math.pi) * (u + 0.044715 * u ** 3)))
    return u


def gelu_err(u, h, kind):
    """How far the fp32 GELU of an exact u may be off."""
    if kind == "erf":  # erff's 2 ulp and the roundings, relative to |u|
        return 5 * U32 * u.abs()
    if kind == "tanh":
        # exp(-2z): its argument is 5 roundings off, __expf 2 + 1.16 |2z| ulp; the division 2 ulp, the rest roundings.
        z2 = 2 * math.sqrt(2 / math.pi) * (u + 0.044715 * u ** 3).abs()
        return h.abs() * (8 + 7.4 * z2.clamp_max(100)) * U32
    return torch.zeros_like(u)


def product64(a, sa, b, sb, bias=None, gelu=None, residual=None, dtype=torch.bfloat16):
    """(value, tolerance) of a product, from exact integer sums."""
    s = (a.double() @ b.double().t()) * sa.double()[:, None] * sb.double()
    u = s if bias is None else s + bias.double()
    h = gelu64(u, gelu)
    # sum to fp32, two scales, bias; GELU's slope is at most 1.13
    tol = 1.13 * (4 * U32 * s.abs() + U32 * u.abs()) + gelu_err(u, h, gelu)
    y = h if residual is None else h + residual.double()
    tol = tol + U32 * y.abs()
    return y, tol + (tol + y.abs()) * torch.finfo(dtype).eps / 2 + torch.finfo(dtype).tiny


def check(y, want):
    ref, tol = want
    assert y.shape == ref.shape
    bad = ~((y.double() - ref).abs() <= tol)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off; worst {((y.double() - ref).abs() / tol).max():.3g} x"


def operands(seed, m, n, k, lo=-127):
    g = gen(seed)
    a, b = ints(g, m, k, lo=lo), ints(g, n, k, lo=lo)
    sa = torch.rand(m, generator=g, device="cuda") * 0.02 + 1e-3
    sb = torch.rand(n, generator=g, device="cuda") * 0.02 / math.sqrt(max(k, 1)) + 1e-5
    bias = normal(g, n).mul_(0.1).bfloat16()
    res = normal(g, m, n).bfloat16()
    return a, sa, b, sb, bias, res


def aligned(t):
    """The same int8 matrix with rows a multiple of 16 bytes apart."""
    q = torch.full((t.shape[0], (t.shape[1] + 15) // 16 * 16), 99, dtype=torch.int8, device=t.device)[:, :t.shape[1]]
    return q.copy_(t)


# (M, N, K): single values, one row, both sides of the row counts where the kernels change, ragged tiles and k blocks
SHAPES = [(1, 1, 1), (1, 4096, 4096), (1, 130, 127), (2, 5, 300), (17, 129, 128), (31, 1000, 129), (32, 512, 4096),
          (33, 257, 1000), (64, 300, 2049), (65, 520, 384), (100, 100, 50), (128, 384, 1024), (129, 700, 640),
          (200, 64, 16), (255, 513, 4100), (256, 256, 128), (257, 1023, 511), (1000, 517, 333), (1024, 2304, 768),
          (64, 8192, 512), (40, 96, 16384), (600, 4096, 2048),
          # few rows before large weights: the weight-streaming kernel, with one and many ranges to a channel block
          (1, 2500, 5000), (2, 130, 20000), (17, 3000, 4100), (33, 4097, 4111), (48, 6144, 2048), (64, 2500, 8200),
          (65, 3001, 8000), (100, 3000, 9001), (113, 28672, 1024), (128, 2000, 16384),
          # a long inner dimension: a short last wave of tiles is split over idle CTA pairs
          (130, 300, 16384), (300, 520, 9000), (1200, 4000, 10001)]


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_matmul(ops, m, n, k):
    a, sa, b, sb, bias, res = operands(m + 7 * n + 13 * k, m, n, k)
    a, b = aligned(a), aligned(b)
    check(ops.matmul_int8(a, sa, b, sb), product64(a, sa, b, sb))
    check(ops.matmul_int8(a, sa, b, sb, bias=bias, gelu="tanh"), product64(a, sa, b, sb, bias, "tanh"))
    check(ops.matmul_int8(a, sa, b, sb, bias=bias, residual=res, out_dtype=torch.float32),
          product64(a, sa, b, sb, bias, None, res, torch.float32))
    # Over the residual: an element is read before it is written.
    check(ops.matmul_int8(a, sa, b, sb, residual=res, out=res.clone()), product64(a, sa, b, sb, None, None, res))
    y = res.clone()
    check(ops.matmul_int8(a, sa, b, sb, residual=y, out=y), product64(a, sa, b, sb, None, None, res))


STREAM = object()


def c_call(ops, fn, *args):
    """A C entry point on operands as they are laid out (the Python functions copy unaligned int8 ones)."""
    from tfb200 import _lib as L

    stream = torch.cuda.current_stream().cuda_stream
    ops._call(torch.cuda.current_device(), getattr(L.lib(), fn), *(stream if a is STREAM else a for a in args))


@pytest.mark.parametrize("m,n,k", SHAPES[:-13])
@pytest.mark.parametrize("off_a,pad_a,off_b,pad_b", [(1, 0, 0, 3), (16, 16, 5, 0), (0, 1, 16, 16)])
def test_matmul_unaligned(ops, m, n, k, off_a, pad_a, off_b, pad_b):
    import ctypes

    a, sa, b, sb, bias, res = operands(m + 7 * n + 13 * k, m, n, k)
    av, _ = rows_at(a, off_a, k + pad_a)
    bv, _ = rows_at(b, off_b, k + pad_b)
    y = torch.empty(m, n, dtype=torch.bfloat16, device="cuda")
    need = ops.matmul_int8_workspace_bytes(m, k, n)
    ws = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
    mats = [ops._rows(t, "t", t.dtype, t.get_device())[2] for t in (av, bv, res, y)]
    ra, rb, rr, ry = (ctypes.byref(x) for x in mats)
    assert mats[0].data == av.data_ptr() and mats[1].data == bv.data_ptr()
    c_call(ops, "tfb200_matmul_int8", ra, sa.data_ptr(), rb, sb.data_ptr(), bias.data_ptr(), 1, rr, ry, STREAM,
           ws.data_ptr(), need)
    check(y, product64(a, sa, b, sb, bias, "tanh", res))
    # The same bits as on aligned operands.
    assert torch.equal(y, ops.matmul_int8(av, sa, bv, sb, bias=bias, gelu="tanh", residual=res))


@pytest.mark.parametrize("m,k,h,n", [(3, 50, 333, 20), (70, 100, 70, 64), (300, 129, 515, 130)])
def test_mlp_unaligned(ops, m, k, h, n):
    import ctypes

    g = gen(k)
    x, gamma = normal(g, m, k).bfloat16(), torch.ones(k, dtype=torch.bfloat16, device="cuda")
    w1, s1 = weight(ops, g, h, k)
    w2, s2 = weight(ops, g, n, h)
    res = normal(g, m, n).bfloat16()
    w1v, _ = rows_at(w1, 3, k + 1)
    w2v, _ = rows_at(w2, 1, h)
    y = torch.empty(m, n, dtype=torch.bfloat16, device="cuda")
    need = ops.mlp_int8_workspace_bytes(m, k, h, n)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    mats = [ops._rows(t, "t", t.dtype, t.get_device())[2] for t in (x, w1v, w2v, res, y)]
    rx, r1, r2, rr, ry = (ctypes.byref(t) for t in mats)
    c_call(ops, "tfb200_fused_mlp_int8", rx, gamma.data_ptr(), r1, s1.data_ptr(), None, r2, s2.data_ptr(), rr, EPS, 1,
           ry, STREAM, ws.data_ptr(), need)
    assert torch.equal(y, ops.fused_mlp_int8(x, gamma, w1, s1, None, w2, s2, res, EPS, gelu="tanh"))


@pytest.mark.parametrize("m,n,k", [(1, 300, 256), (48, 200, 129), (37, 2500, 6000), (150, 333, 400), (300, 512, 1024)])
@pytest.mark.parametrize("gelu", [None, "erf", "tanh"])
@pytest.mark.parametrize("with_bias", [False, True])
@pytest.mark.parametrize("with_res", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_matmul_epilogues(ops, m, n, k, gelu, with_bias, with_res, dtype):
    a, sa, b, sb, bias, res = operands(m, m, n, k)
    a, b = aligned(a), aligned(b)
    bias, res = bias if with_bias else None, res if with_res else None
    sb = sb * 40  # GELU over its whole range
    y = ops.matmul_int8(a, sa, b, sb, bias=bias, gelu=gelu, residual=res, out_dtype=dtype)
    assert y.dtype == dtype
    check(y, product64(a, sa, b, sb, bias, gelu, res, dtype))


@pytest.mark.parametrize("m,n,k", [(3, 200, 272), (70, 300, 272), (300, 520, 272), (19, 2500, 6000)])
def test_matmul_strides_and_surroundings(ops, m, n, k):
    a, sa, b, sb, bias, res = operands(m, m, n, k)
    want = product64(a, sa, b, sb, bias, None, res)
    first = None
    for off_in, pad_in, off_out, pad_out in [(0, 0, 0, 0), (16, 32, 8, 8), (1, 3, 1, 1), (0, 0, 4, 4), (16, 16, 0, 3)]:
        av, _ = rows_at(a, off_in, k + pad_in)
        bv, _ = rows_at(b, off_in, k + pad_in)
        rv, _ = rows_at(res, off_out, n + pad_out)
        biasv = torch.cat([bias[:1], bias])[1:] if off_out % 8 else bias
        yv, buf = rows_at(torch.zeros_like(res), off_out, n + pad_out)
        y = ops.matmul_int8(av, sa, bv, sb, bias=biasv, residual=rv, out=yv)
        assert y is yv
        check(yv, want)
        first = yv.clone() if first is None else first
        assert torch.equal(yv, first), "another layout, other bits"
        yv.fill_(77)
        assert (buf == 77).all(), "wrote outside the rows"


@pytest.mark.parametrize("m", [1, 16, 40, 100, 300])  # 131071 deep: streamed up to 128 rows
def test_matmul_extremes(ops, m):
    # The longest inner dimension with the largest products: the sums reach 2147467264 of 2147483647.
    k, n = 131071, 20
    a = torch.full((m, k), -128, dtype=torch.int8, device="cuda")
    b = torch.full((n, k), -128, dtype=torch.int8, device="cuda")
    b[1::2] = 127
    sa, sb = torch.full((m,), 2.0 ** -20, device="cuda"), torch.ones(n, device="cuda")
    y = ops.matmul_int8(a, sa, b, sb, out_dtype=torch.float32)
    check(y, product64(a, sa, b, sb, dtype=torch.float32))
    # NaN and infinite scales stay in their rows and columns.
    a, sa, b, sb, bias, res = operands(m, m, 300, 512)
    sa[0], sb[5], sb[299] = float("nan"), float("inf"), float("nan")
    y = ops.matmul_int8(a, sa, b, sb)
    assert y[0].isnan().all() and y[:, 299].isnan().all()
    keep = torch.ones(300, dtype=torch.bool, device="cuda")
    keep[[5, 299]] = False
    ref, tol = product64(a, sa, b, sb)
    assert ((y.double() - ref).abs() <= tol)[1:, keep].all()
    # No inner dimension: the epilogue of zero.
    z8 = torch.empty(m, 0, dtype=torch.int8, device="cuda"), torch.empty(300, 0, dtype=torch.int8, device="cuda")
    sb = torch.ones(300, device="cuda")
    y = ops.matmul_int8(z8[0], torch.ones(m, device="cuda"), z8[1], sb, bias=bias, residual=res)
    assert torch.equal(y, (bias.float() + res.float()).bfloat16())
    assert ops.matmul_int8(a[:0], sa[:0], b, sb).shape == (0, 300)
    assert ops.matmul_int8(a, sa, b[:0], sb[:0]).shape == (m, 0)


@pytest.mark.parametrize("m", [20, 300])
def test_matmul_long_offsets(ops, m):
    ld, n, k = 1 << 28, 10, 528
    a, sa, b, sb, _, _ = operands(m, m, n, k)
    big = torch.empty(9 * ld + k, dtype=torch.int8, device="cuda")
    bv = torch.as_strided(big, (n, k), (ld, 1))
    bv.copy_(b)
    check(ops.matmul_int8(a, sa, bv, sb), product64(a, sa, b, sb))


# (M, N, K): up to 32 rows, read straight into registers: every row count's kernel, every width of a block (8, 16, 32
# channels), ragged channels, inner dimensions that end inside a lane's 16 or 32 bytes, inside a step and after many
HANDFULS = [(1, 1, 31), (1, 7, 16), (2, 33, 48), (1, 1000, 1009), (2, 4736, 1024), (2, 4745, 1040), (1, 9480, 272),
            (1, 300, 16400), (3, 5, 31), (5, 33, 32), (8, 100, 63), (7, 1000, 1009), (8, 4745, 1040), (9, 31, 48),
            (16, 9480, 272), (13, 300, 16400), (16, 4096, 4096), (11, 2000, 8223), (17, 33, 48), (24, 1000, 1009),
            (32, 4745, 1040), (25, 9480, 272), (31, 300, 16400), (32, 7, 31),
            # more rows before larger weights: the weight-streaming kernel again
            (20, 6144, 4100), (16, 28672, 8192), (32, 28672, 1024)]


@pytest.mark.parametrize("m,n,k", HANDFULS)
@pytest.mark.parametrize("off", [0, 16])
def test_matmul_handful(ops, m, n, k, off):
    a, sa, b, sb, bias, res = operands(m + 5 * n + 11 * k, m, n, k, lo=-128)
    ld = (k + 15) // 16 * 16 + off
    a, b = rows_at(a, off, ld)[0], rows_at(b, off, ld)[0]
    check(ops.matmul_int8(a, sa, b, sb, out_dtype=torch.float32), product64(a, sa, b, sb, dtype=torch.float32))
    y = res.clone()
    check(ops.matmul_int8(a, sa, b, sb, bias=bias, gelu="erf", residual=y, out=y),
          product64(a, sa, b, sb, bias, "erf", res))


@pytest.mark.parametrize("n,k", [(33, 48), (520, 1009), (4800, 2048), (300, 16400)])
def test_matmul_row_count_keeps_the_bits(ops, n, k):
    """A row's result does not depend on how many rows are computed with it, whichever kernel that takes."""
    a, sa, b, sb, bias, res = operands(n + k, 300, n, k)
    a, b = aligned(a), aligned(b)
    want = ops.matmul_int8(a, sa, b, sb, bias=bias, gelu="tanh", residual=res)
    for m in (1, 2, 3, 8, 9, 16, 17, 24, 25, 32, 33, 128, 129):
        y = ops.matmul_int8(a[:m], sa[:m], b, sb, bias=bias, gelu="tanh", residual=res[:m])
        assert torch.equal(y, want[:m]), m


@pytest.mark.parametrize("m", [1, 2, 16, 32])
def test_matmul_handful_long_offsets(ops, m):
    ld, n, k = 1 << 28, 10, 528
    a, sa, b, sb, _, _ = operands(m, m, n, k)
    big = torch.empty(9 * ld + k, dtype=torch.int8, device="cuda")
    bv = torch.as_strided(big, (n, k), (ld, 1))
    bv.copy_(b)
    check(ops.matmul_int8(a, sa, bv, sb), product64(a, sa, b, sb))


# -------------------------------------------------------------- fused calls


def weight(ops, g, n, k):
    return ops.quantize_int8((normal(g, n, k) / math.sqrt(k)).bfloat16())


@pytest.mark.parametrize("m,k,n", [(1, 4096, 6144), (16, 1000, 520), (64, 257, 129), (65, 512, 640), (300, 768, 1000),
                                   (1024, 4096, 2048)])
def test_rmsnorm_matmul_is_its_parts(ops, m, k, n):
    g = gen(k + n)
    x, gamma = normal(g, m, k).bfloat16(), (torch.rand(k, generator=g, device="cuda") + 0.5).bfloat16()
    w, ws = weight(ops, g, n, k)
    q, scale = ops.rmsnorm_int8(x, gamma, EPS)
    y = ops.fused_rmsnorm_matmul_int8(x, gamma, w, ws, EPS)
    assert torch.equal(y, ops.matmul_int8(q, scale, w, ws))
    check(y, product64(q, scale, w, ws))


def mlp64(q, scale, w1, s1, b1, w2, s2, res, gelu):
    """(value, tolerance) of the block from its quantised input.

    The device holds hidden values as 16-bit integers of their block's maximum, half a step of which is 1 / 65534 of
    it, and the products before and after that in fp32. That moves v = 127 h / amax by at most d = 127 / 65534 (times
    block maximum / amax <= 1) plus the fp32 parts, so q moves by one where v lies within d of a half and nowhere
    else, and the row's scale by a few U32.
    """
    u = (q.double() @ w1.double().t()) * scale.double()[:, None] * s1.double()
    if b1 is not None:
        u = u + b1.double()
    h = gelu64(u, gelu)
    amax = h.abs().amax(-1, keepdim=True)
    # fp32 part of the hidden error: relative to u before the GELU, at most 16 U32 of it (gelu_err's bound included)
    e32 = 16 * U32 * (1 + u.abs() + gelu_err(u, h, gelu) / U32 / 16)
    v = h * (127.0 / amax)
    d = 127.0 / 65534 + 127 * 8 * U32 + 127.0 / amax * 2 * e32
    hq = v.round()
    hs = amax / 127.0
    may = ((v - v.floor() - 0.5).abs() <= d).double()
    w = w2.double() * s2.double()[:, None]
    y = (hq * hs) @ w.t() + res.double()
    slack = (may + (hq.abs() + 1) * 1e-5) * hs
    tol = slack @ w.abs().t() + 8 * U32 * y.abs()
    return y, tol + (tol + y.abs()) * torch.finfo(torch.bfloat16).eps / 2


MLPS = [(1, 256, 1024, 256), (7, 100, 333, 50), (32, 512, 2048, 512), (64, 257, 515, 129), (65, 512, 1024, 512),
        (200, 384, 1000, 384), (1024, 1024, 4096, 1024),
        (200, 9008, 520, 256), (1, 2100, 9001, 2000), (40, 3000, 8001, 2800), (100, 4096, 8200, 3000)]


@pytest.mark.parametrize("m,k,h,n", MLPS)
@pytest.mark.parametrize("gelu,with_bias", [("erf", True), ("tanh", True), ("tanh", False)])
def test_mlp(ops, m, k, h, n, gelu, with_bias):
    g = gen(k + n + h)
    x, gamma = normal(g, m, k).bfloat16(), (torch.rand(k, generator=g, device="cuda") + 0.5).bfloat16()
    w1, s1 = weight(ops, g, h, k)
    w2, s2 = weight(ops, g, n, h)
    b1 = (normal(g, h) * 0.1).bfloat16() if with_bias else None
    res = normal(g, m, n).bfloat16()
    y = ops.fused_mlp_int8(x, gamma, w1, s1, b1, w2, s2, res, EPS, gelu=gelu)
    q, scale = ops.rmsnorm_int8(x, gamma, EPS)
    ref, tol = mlp64(q, scale, w1, s1, b1, w2, s2, res, gelu)
    check(y, (ref, tol))
    # The worst case above adds up every possible step; on average the error is the output's rounding (2^-9 or less)
    # and a step in the few values near a half: within 0.4 % of the result's norm.
    assert (y.double() - ref).norm() <= 4e-3 * ref.norm()


@pytest.mark.parametrize("m", [5, 300])
@pytest.mark.parametrize("size", [1e-12, 1.0, 1e6, 1e15])
def test_mlp_hidden_range(ops, m, size):
    """Hidden values far below and above 16-bit floating formats' range."""
    g = gen(11)
    k, h, n = 256, 512, 128
    x, gamma = normal(g, m, k).bfloat16(), torch.ones(k, dtype=torch.bfloat16, device="cuda")
    w1, s1 = weight(ops, g, h, k)
    w2, s2 = weight(ops, g, n, h)
    s1 = s1 * size
    res = torch.zeros(m, n, dtype=torch.bfloat16, device="cuda")
    b1 = (normal(g, h) * min(size, 1e3)).bfloat16()
    y = ops.fused_mlp_int8(x, gamma, w1, s1, b1, w2, s2, res, EPS, gelu="erf")
    q, scale = ops.rmsnorm_int8(x, gamma, EPS)
    u = (q.double() @ w1.double().t()) * scale.double()[:, None] * s1.double() + b1.double()
    hid = gelu64(u, "erf")
    hs = hid.abs().amax(-1, keepdim=True) / 127.0
    # Against the unquantised hidden block: half an int8 step and the 16-bit rounding, 1 / 65534 of amax = 127 / 65534
    # of a step, for each value.
    w = w2.double() * s2.double()[:, None]
    ref = hid @ w.t()
    tol = (((0.5 + 127.0 / 65534 + 1e-4) * hs + 1e-5 * u.abs()) @ w.abs().t()) + 2.0 ** -8 * ref.abs()
    check(y, (ref, tol))
    # Same scale as the definition's own quantisation error, not only its worst case.
    assert (y.double() - ref).norm() <= 0.03 * ref.norm()


def test_mlp_bad_rows_stay_apart(ops):
    g = gen(4)
    for m in (6, 200):
        k, h, n = 128, 512, 128
        x, gamma = normal(g, m, k).bfloat16(), torch.ones(k, dtype=torch.bfloat16, device="cuda")
        w1, s1 = weight(ops, g, h, k)
        w2, s2 = weight(ops, g, n, h)
        good = ops.fused_mlp_int8(x, gamma, w1, s1, None, w2, s2, x, EPS)
        x2 = x.clone()
        x2[1, 3] = float("nan")
        x2[2, 0] = float("inf")
        x2[4] = 0
        y = ops.fused_mlp_int8(x2, gamma, w1, s1, None, w2, s2, x2, EPS)
        assert y[1].isnan().all() and y[2].isnan().all() and (y[4] == 0).all()
        rest = [i for i in range(m) if i not in (1, 2, 4)]
        assert torch.equal(y[rest], good[rest])


@pytest.mark.parametrize("k,h,n", [(100, 333, 50), (1024, 4100, 1000), (2048, 16400, 520), (9008, 520, 256)])
def test_mlp_row_count_keeps_the_bits(ops, k, h, n):
    g = gen(k + h)
    x, gamma = normal(g, 300, k).bfloat16(), (torch.rand(k, generator=g, device="cuda") + 0.5).bfloat16()
    w1, s1 = weight(ops, g, h, k)
    w2, s2 = weight(ops, g, n, h)
    b1, res = (normal(g, h) * 0.1).bfloat16(), normal(g, 300, n).bfloat16()
    x[2, 1], x[5] = float("inf"), 0
    want = ops.fused_mlp_int8(x, gamma, w1, s1, b1, w2, s2, res, EPS)
    assert want[2].isnan().all() and not want[3:].isnan().any()
    q, scale = ops.rmsnorm_int8(x, gamma, EPS)
    for m in (1, 2, 7, 8, 9, 16, 17, 25, 32, 64, 128, 129):
        # The norm's sum of squares is in the order of its block's threads, which are fewer for many rows: the scale
        # of a row may differ in its last bits (the sums of up to 64 and a few more terms a thread: 60 U32), q not.
        qm, sm = ops.rmsnorm_int8(x[:m], gamma, EPS)
        assert torch.equal(qm, q[:m]) and ((sm - scale[:m]).abs() <= 60 * U32 * sm)[sm == sm].all()
        same = sm.view(torch.int32) == scale[:m].view(torch.int32)
        assert m < 64 or same.any()
        y = ops.fused_mlp_int8(x[:m], gamma, w1, s1, b1, w2, s2, res[:m], EPS)
        assert torch.equal(y[same].view(torch.int16), want[:m][same].view(torch.int16)), m


# ------------------------------------------------------- streams and graphs


@pytest.mark.parametrize("m,d", [(8, 512), (8, 2560), (64, 512), (100, 512), (100, 4096), (512, 512)])
def test_a_layer_in_a_graph(ops, m, d):
    """norm + QKV, output projection with the residual, MLP block: captured together and replayed with new inputs."""
    g = gen(m)
    h = 3 * d
    gamma = (torch.rand(d, generator=g, device="cuda") + 0.5).bfloat16()
    wq, sq = weight(ops, g, 3 * d, d)
    wo, so = weight(ops, g, d, d)
    w1, s1 = weight(ops, g, h, d)
    w2, s2 = weight(ops, g, d, h)
    b1 = normal(g, h).bfloat16()

    def layer(x):
        qkv = ops.fused_rmsnorm_matmul_int8(x, gamma, wq, sq, EPS)
        q, s = ops.quantize_int8(qkv[:, :d])
        x = ops.matmul_int8(q, s, wo, so, residual=x)
        q, s, x = ops.rmsnorm_int8(x, gamma, EPS, residual=qkv[:, d:2 * d])
        y = ops.matmul_int8(q, s, wo, so, gelu="tanh")
        return ops.fused_mlp_int8(x, gamma, w1, s1, b1, w2, s2, y, EPS, gelu="tanh")

    xs = [normal(g, m, d).bfloat16() for _ in range(4)]
    want = [layer(x) for x in xs]
    buf = xs[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = layer(buf)
    for x, w in list(zip(xs, want)) * 3:
        buf.copy_(x)
        graph.replay()
        assert torch.equal(y, w)


def test_two_streams_at_once(ops):
    g = gen(9)
    k, n = 4096, 4096
    w, ws = weight(ops, g, n, k)
    gamma = torch.ones(k, dtype=torch.bfloat16, device="cuda")
    xs = {m: normal(g, m, k).bfloat16() for m in (4, 64, 90, 700)}
    want = {m: ops.fused_rmsnorm_matmul_int8(x, gamma, w, ws, EPS) for m, x in xs.items()}
    torch.cuda.synchronize()
    streams = {m: torch.cuda.Stream() for m in xs}
    got = {m: [] for m in xs}
    for _ in range(20):
        for m, x in xs.items():
            with torch.cuda.stream(streams[m]):
                got[m].append(ops.fused_rmsnorm_matmul_int8(x, gamma, w, ws, EPS))
    torch.cuda.synchronize()
    for m in xs:
        assert all(torch.equal(y, want[m]) for y in got[m])


def test_split_products_on_two_streams(ops):
    """Products whose last wave is split over idle CTA pairs, several at once: finishing pairs wait for helpers."""
    g = gen(10)
    k, n = 16384, 2048
    a, sa, b, sb, _, _ = operands(3, 300, n, k)
    assert ops.matmul_int8_workspace_bytes(300, k, n) > 0
    want = ops.matmul_int8(a, sa, b, sb)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(4)], []
    for _ in range(15):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(ops.matmul_int8(a, sa, b, sb))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want) for y in got)
    from tfb200 import _lib as L

    assert L.lib().tfb200_device_status() == L.TFB200_OK


@pytest.mark.parametrize("m", [1, 8, 40, 300])
def test_fused_calls_behind_their_weights(ops, m):
    """The products of the fused calls ask for weights before the launch ahead of them has ended."""
    g = gen(m)
    k, n = 2048, 4096
    x, res = normal(g, m, k).bfloat16(), normal(g, m, k).bfloat16()
    gamma = torch.ones(k, dtype=torch.bfloat16, device="cuda")
    ups, downs = ([(normal(g, *s) / 45).bfloat16() for _ in range(3)] for s in ((n, k), (k, n)))
    want = []
    for u, d in zip(ups, downs):
        (w1, s1), (w2, s2) = ops.quantize_int8(u), ops.quantize_int8(d)
        want.append((ops.fused_rmsnorm_matmul_int8(x, gamma, w1, s1, EPS),
                     ops.fused_mlp_int8(x, gamma, w1, s1, None, w2, s2, res, EPS)))
    torch.cuda.synchronize()
    for _ in range(4):
        for u, d, (y, z) in zip(ups, downs, want):
            ops.quantize_int8(u, out=(w1, s1))
            assert torch.equal(ops.fused_rmsnorm_matmul_int8(x, gamma, w1, s1, EPS), y)
            ops.quantize_int8(d, out=(w2, s2))
            ops.quantize_int8(u, out=(w1, s1))
            assert torch.equal(ops.fused_mlp_int8(x, gamma, w1, s1, None, w2, s2, res, EPS), z)


@pytest.mark.parametrize("m", [16, 80, 384])
def test_weights_written_just_before(ops, m):
    """A product right behind the launch that writes its weights and scales."""
    g = gen(m)
    k, n = 2048, 4096
    x = normal(g, m, k).bfloat16()
    q, s = ops.quantize_int8(x)
    ws = [normal(g, n, k).bfloat16() for _ in range(3)]
    want = [ops.matmul_int8(q, s, *ops.quantize_int8(w)) for w in ws]
    torch.cuda.synchronize()
    wq, sc = ops.quantize_int8(ws[0])
    for _ in range(4):
        for w, y in zip(ws, want):
            ops.quantize_int8(w, out=(wq, sc))
            assert torch.equal(ops.matmul_int8(q, s, wq, sc), y)


def test_workspace_reuse_and_checks(ops):
    g = gen(2)
    for m, n, k in ((8, 1000, 8192), (100, 3000, 8192), (400, 1000, 2048), (200, 300, 16384)):
        a, sa, b, sb, _, _ = operands(m, m, n, k)
        a, b = aligned(a), aligned(b)
        need = ops.matmul_int8_workspace_bytes(m, k, n)
        assert (need > 0) == (m in (100, 200))
        ws = torch.full((need + 256,), 255, dtype=torch.uint8, device="cuda")  # whatever it held before
        y = ops.matmul_int8(a, sa, b, sb, workspace=ws)
        assert torch.equal(y, ops.matmul_int8(a, sa, b, sb))
        assert torch.equal(y, ops.matmul_int8(a, sa, b, sb, workspace=ws))
        if need:
            assert (ws[need:] == 255).all()
            with pytest.raises(ValueError, match="workspace"):
                ops.matmul_int8(a, sa, b, sb, workspace=ws[:need - 1])


def test_one_workspace_behind_one_another(ops):
    """Calls of every row count's kernels share a workspace on one stream, each launched while the last still runs."""
    g = gen(12)
    k, h = 1024, 4096
    gamma = torch.ones(k, dtype=torch.bfloat16, device="cuda")
    w1, s1 = weight(ops, g, h, k)
    w2, s2 = weight(ops, g, k, h)
    xs = [normal(g, m, k).bfloat16() for m in (1, 8, 24, 60, 100, 150, 300)]
    hs = [ops.quantize_int8(normal(g, m, h).bfloat16()) for m in (1, 8, 24, 60, 100, 150, 300)]
    need = max(max(ops.mlp_int8_workspace_bytes(x.shape[0], k, h, k), ops.matmul_int8_workspace_bytes(x.shape[0], h, k),
                   ops.rmsnorm_matmul_int8_workspace_bytes(x.shape[0], k, h)) for x in xs)
    ws = torch.full((need,), 255, dtype=torch.uint8, device="cuda")

    def calls(**kw):
        for x, (q, s) in zip(xs, hs):
            yield ops.fused_mlp_int8(x, gamma, w1, s1, None, w2, s2, x, EPS, **kw)
            yield ops.matmul_int8(q, s, w2, s2, residual=x, **kw)
            yield ops.fused_rmsnorm_matmul_int8(x, gamma, w1, s1, EPS, **kw)

    want = list(calls())
    torch.cuda.synchronize()
    got = [list(calls(workspace=ws)) for _ in range(5)]
    torch.cuda.synchronize()
    for ys in got:
        assert all(torch.equal(y, w) for y, w in zip(ys, want))


def test_refusals(ops):
    g = gen(1)
    x = normal(g, 4, 64).bfloat16()
    q, s = ops.quantize_int8(x)
    gamma = torch.ones(64, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(TypeError):
        ops.quantize_int8(x.float())
    with pytest.raises(ValueError):
        ops.quantize_int8(x[0])
    with pytest.raises(ValueError):
        ops.quantize_int8(x, out=(q[:2], s))
    with pytest.raises(ValueError):
        ops.quantize_int8(x, out=(q, s[:2]))
    with pytest.raises(ValueError):
        ops.rmsnorm_int8(x, gamma[:10], EPS)
    with pytest.raises(ValueError):
        ops.rmsnorm_int8(x, gamma, EPS, residual=x[:2])
    with pytest.raises(ValueError):
        ops.rmsnorm_int8(x, gamma, EPS, residual=x, out=(q, s))
    from tfb200._lib import TFB200Error
    with pytest.raises(TFB200Error):
        ops.rmsnorm_int8(x, gamma, -1.0)
    with pytest.raises(ValueError):
        ops.matmul_int8(q, s, q[:, :32], s)
    with pytest.raises(ValueError):
        ops.matmul_int8(q, s[:3], q, s)
    with pytest.raises(TypeError):
        ops.matmul_int8(q, s.half(), q, s)
    with pytest.raises(TypeError):
        ops.matmul_int8(x, s, q, s)
    with pytest.raises(ValueError):
        ops.matmul_int8(q, s, q, s, gelu="relu")
    with pytest.raises(TypeError):
        ops.matmul_int8(q, s, q, s, out_dtype=torch.float16)
    with pytest.raises(TypeError):
        ops.matmul_int8(q, s, q, s, out=torch.empty(4, 4, device="cuda"))
    with pytest.raises(ValueError):
        ops.matmul_int8(q, s, q, s, out=torch.empty(4, 8, device="cuda", dtype=torch.bfloat16)[:, ::2])
    with pytest.raises(ValueError):
        ops.matmul_int8(q, s, q.unsqueeze(0), s)
    with pytest.raises(TypeError):
        ops.matmul_int8(q.cpu(), s, q, s)
    long = torch.zeros(1, 131072, dtype=torch.int8, device="cuda")
    with pytest.raises(TFB200Error, match="131071"):
        ops.matmul_int8(long, s[:1], long, s[:1])
    with pytest.raises(ValueError):
        ops.fused_rmsnorm_matmul_int8(x, gamma, q[:, :32], s)
    with pytest.raises(ValueError):
        ops.fused_mlp_int8(x, gamma, q, s, None, q, s, x, EPS)
    with pytest.raises(ValueError):
        ops.fused_mlp_int8(x, gamma, q, s, None, q[:, :4], s, x, EPS, gelu="none")
