"""The 8-bit integer entry points' argument checks and workspace sizes: calls that reach no device."""

import ctypes

import pytest

from tfb200 import _lib as L

R = ctypes.byref


def mat(rows, cols, dtype, ld=None, data=4096):
    return L.Mat(data, rows, cols, max(cols, 1) if ld is None else ld, dtype)


@pytest.fixture(scope="module")
def lib():
    return L.lib()


def refused(lib, code, text, fn, *args):
    assert getattr(lib, fn)(*args) == code
    msg = lib.tfb200_last_error().decode()
    assert msg.startswith(fn + ": ") and text in msg, msg


def test_quantize_refusals(lib):
    x, q = mat(4, 64, L.TFB200_BF16), mat(4, 64, L.TFB200_I8)
    fn = "tfb200_quantize_int8"
    refused(lib, L.TFB200_EINVAL, "null descriptor", fn, None, R(q), 4096, None)
    refused(lib, L.TFB200_EINVAL, "dtype", fn, R(mat(4, 64, L.TFB200_F32)), R(q), 4096, None)
    refused(lib, L.TFB200_EINVAL, "dtype", fn, R(x), R(mat(4, 64, L.TFB200_BF16)), 4096, None)
    refused(lib, L.TFB200_EINVAL, "shape", fn, R(x), R(mat(4, 63, L.TFB200_I8)), 4096, None)
    refused(lib, L.TFB200_EINVAL, "leading dimension", fn, R(x), R(mat(4, 64, L.TFB200_I8, 63)), 4096, None)
    refused(lib, L.TFB200_EINVAL, "null data", fn, R(mat(4, 64, L.TFB200_BF16, data=None)), R(q), 4096, None)
    refused(lib, L.TFB200_EINVAL, "not aligned", fn, R(mat(4, 64, L.TFB200_BF16, data=4097)), R(q), 4096, None)
    refused(lib, L.TFB200_EINVAL, "negative", fn, R(mat(-1, 64, L.TFB200_BF16)), R(q), 4096, None)
    refused(lib, L.TFB200_EINVAL, "2^30", fn, R(mat((1 << 30) + 1, 64, L.TFB200_BF16)), R(q), 4096, None)
    refused(lib, L.TFB200_EINVAL, "null scale", fn, R(x), R(q), None, None)
    refused(lib, L.TFB200_EINVAL, "scale: not aligned", fn, R(x), R(q), 4098, None)
    assert lib.tfb200_quantize_int8(R(mat(0, 64, L.TFB200_BF16)), R(mat(0, 64, L.TFB200_I8)), None, None) == 0


def test_rmsnorm_refusals(lib):
    x, q = mat(4, 64, L.TFB200_BF16), mat(4, 64, L.TFB200_I8)
    fn = "tfb200_rmsnorm_int8"
    refused(lib, L.TFB200_EINVAL, "null gamma", fn, R(x), None, None, 1e-5, None, R(q), 4096, None)
    refused(lib, L.TFB200_EINVAL, "eps", fn, R(x), None, 4096, -1.0, None, R(q), 4096, None)
    refused(lib, L.TFB200_EINVAL, "gamma: not aligned", fn, R(x), None, 4097, 1e-5, None, R(q), 4096, None)
    refused(lib, L.TFB200_EINVAL, "eps", fn, R(x), None, 4096, float("nan"), None, R(q), 4096, None)
    refused(lib, L.TFB200_EINVAL, "sum", fn, R(x), R(x), 4096, 1e-5, None, R(q), 4096, None)
    refused(lib, L.TFB200_EINVAL, "without a residual", fn, R(x), None, 4096, 1e-5, R(x), R(q), 4096, None)
    refused(lib, L.TFB200_EINVAL, "shape", fn, R(x), R(mat(3, 64, L.TFB200_BF16)), 4096, 1e-5, R(x), R(q), 4096, None)
    e, qe = mat(4, 0, L.TFB200_BF16), mat(4, 0, L.TFB200_I8)
    refused(lib, L.TFB200_EINVAL, "empty dimension", fn, R(e), None, 4096, 1e-5, None, R(qe), 4096, None)


def test_matmul_refusals(lib):
    a, b, c = mat(4, 64, L.TFB200_I8), mat(8, 64, L.TFB200_I8), mat(4, 8, L.TFB200_BF16)
    fn = "tfb200_matmul_int8"

    def call(a=a, b=b, c=c, sa=4096, sb=4096, gelu=L.TFB200_GELU_NONE, res=None, ws=4096, n=1 << 40):
        return (R(a) if a else None, sa, R(b), sb, None, gelu, R(res) if res else None, R(c), None, ws, n)

    refused(lib, L.TFB200_EINVAL, "null descriptor", fn, *call(a=None))
    refused(lib, L.TFB200_EINVAL, "dtype", fn, *call(a=mat(4, 64, L.TFB200_BF16)))
    refused(lib, L.TFB200_EINVAL, "dtype", fn, *call(c=mat(4, 8, L.TFB200_I8)))
    refused(lib, L.TFB200_EINVAL, "shapes", fn, *call(b=mat(8, 63, L.TFB200_I8)))
    refused(lib, L.TFB200_EINVAL, "shapes", fn, *call(c=mat(4, 9, L.TFB200_BF16)))
    refused(lib, L.TFB200_EINVAL, "shapes", fn, *call(res=mat(4, 9, L.TFB200_BF16)))
    refused(lib, L.TFB200_EINVAL, "gelu_mode", fn, *call(gelu=3))
    refused(lib, L.TFB200_EINVAL, "null scales", fn, *call(sa=None))
    refused(lib, L.TFB200_EINVAL, "null scales", fn, *call(sb=None))
    refused(lib, L.TFB200_EINVAL, "b_scale: not aligned", fn, *call(sb=4098))
    refused(lib, L.TFB200_EINVAL, "not aligned", fn, *call(c=mat(4, 8, L.TFB200_F32, data=4098)))
    k = 131072
    refused(lib, L.TFB200_EUNSUPPORTED, "131071", fn, *call(a=mat(4, k, L.TFB200_I8), b=mat(8, k, L.TFB200_I8)))
    need = lib.tfb200_matmul_int8_workspace_size(4, 64, 8)
    if need:
        refused(lib, L.TFB200_EWORKSPACE, str(need), fn, *call(n=need - 1))
        refused(lib, L.TFB200_EWORKSPACE, str(need), fn, *call(ws=None))
        refused(lib, L.TFB200_EWORKSPACE, "aligned", fn, *call(ws=4096 + 128))
    assert lib.tfb200_matmul_int8(*call(b=mat(0, 64, L.TFB200_I8), c=mat(4, 0, L.TFB200_BF16), sb=None)) == 0


def test_fused_refusals(lib):
    x, y = mat(4, 64, L.TFB200_BF16), mat(4, 8, L.TFB200_BF16)
    w1, w2 = mat(32, 64, L.TFB200_I8), mat(8, 32, L.TFB200_I8)
    big = (None, 4096, 1 << 40)
    fn = "tfb200_fused_rmsnorm_matmul_int8"
    w = mat(8, 64, L.TFB200_I8)
    refused(lib, L.TFB200_EINVAL, "shapes", fn, R(x), 4096, R(w2), 4096, 1e-5, R(y), *big)
    refused(lib, L.TFB200_EINVAL, "null gamma", fn, R(x), None, R(w), 4096, 1e-5, R(y), *big)
    refused(lib, L.TFB200_EINVAL, "w_scale", fn, R(x), 4096, R(w), None, 1e-5, R(y), *big)
    need = lib.tfb200_fused_rmsnorm_matmul_int8_workspace_size(4, 64, 8)
    refused(lib, L.TFB200_EWORKSPACE, str(need), fn, R(x), 4096, R(w), 4096, 1e-5, R(y), None, 4096, need - 1)
    fn = "tfb200_fused_mlp_int8"

    def call(w1=w1, w2=w2, res=y, gelu=0, eps=1e-5, gamma=4096, ws=big):
        return (R(x), gamma, R(w1), 4096, None, R(w2), 4096, R(res), eps, gelu, R(y), *ws)

    refused(lib, L.TFB200_EINVAL, "shapes", fn, *call(w2=mat(8, 31, L.TFB200_I8)))
    refused(lib, L.TFB200_EINVAL, "shapes", fn, *call(res=x))
    refused(lib, L.TFB200_EINVAL, "gelu_mode", fn, *call(gelu=L.TFB200_GELU_NONE))
    refused(lib, L.TFB200_EINVAL, "eps", fn, *call(eps=-1.0))
    refused(lib, L.TFB200_EINVAL, "null gamma", fn, *call(gamma=None))
    refused(lib, L.TFB200_EUNSUPPORTED, "empty hidden", fn,
            *call(w1=mat(0, 64, L.TFB200_I8), w2=mat(8, 0, L.TFB200_I8)))
    need = lib.tfb200_fused_mlp_int8_workspace_size(4, 64, 32, 8)
    refused(lib, L.TFB200_EWORKSPACE, str(need), fn, *call(ws=(None, 4096, need - 1)))


def test_workspace_sizes(lib):
    big = 2 ** 64 - 1
    assert lib.tfb200_matmul_int8_workspace_size(0, 64, 64) == 0
    assert lib.tfb200_matmul_int8_workspace_size(1 << 40, 64, 64) == big
    assert lib.tfb200_fused_rmsnorm_matmul_int8_workspace_size(64, 1 << 40, 64) == big
    assert lib.tfb200_fused_mlp_int8_workspace_size(64, 64, 1 << 40, 64) == big
    assert lib.tfb200_fused_mlp_int8_workspace_size(64, 64, 0, 64) == 0
    for m in (1, 64, 65, 128, 129, 8192):
        one = lib.tfb200_fused_rmsnorm_matmul_int8_workspace_size(m, 4096, 6144)
        # the int8 rows and their scales, then the product's own region
        assert one >= m * 4096 + m * 4 + lib.tfb200_matmul_int8_workspace_size(m, 4096, 6144)
        mlp = lib.tfb200_fused_mlp_int8_workspace_size(m, 4096, 16384, 4096)
        assert mlp >= m * (4096 + 16384 * 3 + 8) and mlp % 256 == 0


def test_python_checks_need_no_device():
    torch = pytest.importorskip("torch")
    from tfb200 import ops

    x, q, s = torch.zeros(4, 64, dtype=torch.bfloat16), torch.zeros(4, 64, dtype=torch.int8), torch.zeros(4)
    for call in (lambda: ops.quantize_int8(x), lambda: ops.rmsnorm_int8(x, x[0]),
                 lambda: ops.matmul_int8(q, s, q, s), lambda: ops.fused_rmsnorm_matmul_int8(x, x[0], q, s),
                 lambda: ops.fused_mlp_int8(x, x[0], q, s, None, q, s, x)):
        with pytest.raises(TypeError, match="CUDA tensor"):
            call()
