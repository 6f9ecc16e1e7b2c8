"""The reference's operator interface on the B200 backend.

Same names, argument order and meaning as the reference golden
(tensixflow ``python/tensixflow/golden.py``): ``matmul(a, b)`` (:56-60),
``fused_rmsnorm_matmul(x, gamma, w, eps=1e-6)`` (:97-102) and
``fused_mlp(x, gamma, w1, b1, w2, residual, eps=1e-6)`` (:105-122), plus a
``gelu`` keyword ("erf", the reference's exact form, or "tanh").

Inputs are CUDA bf16 torch tensors, row-major; leading dimensions of ``x`` /
``a`` / ``residual`` are flattened into rows as the reference's lowering does
(``LowerToTTKernelPass.cpp:181-189``). The result is a bf16 tensor of shape
``[..., N]``. Every call runs the sm_100a kernels of libtfb200.so through its C
ABI; there is no other code path. Shape errors raise ``ValueError`` (numpy's
``@`` raises the same class in the reference); backend errors raise
``TFB200Error``.
"""

from __future__ import annotations

import ctypes
import math

import torch

from . import _lib as L

__all__ = ["matmul", "fused_rmsnorm_matmul", "fused_mlp", "fused_mlp_partial", "fused_mlp_tp", "residual_add",
           "mlp_workspace_bytes",
           "rmsnorm_matmul_workspace_bytes", "quantize_int8", "rmsnorm_int8", "matmul_int8",
           "fused_rmsnorm_matmul_int8", "fused_mlp_int8", "matmul_int8_workspace_bytes",
           "rmsnorm_matmul_int8_workspace_bytes", "mlp_int8_workspace_bytes", "mat", "stream_ptr"]


def stream_ptr(stream: torch.cuda.Stream | None = None) -> int:
    s = stream if stream is not None else torch.cuda.current_stream()
    return s.cuda_stream


def _rows2d(t: torch.Tensor, name: str) -> torch.Tensor:
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError(f"{name} must be a CUDA tensor")
    if t.dtype != torch.bfloat16:
        raise TypeError(f"{name} must be bfloat16 (got {t.dtype})")
    if t.dim() < 2:
        raise ValueError(f"{name} must have at least 2 dimensions")
    t2 = t.reshape(math.prod(t.shape[:-1]), t.shape[-1])
    if t2.stride(-1) != 1:
        t2 = t2.contiguous()
    return t2


def mat(t: torch.Tensor) -> L.Mat:
    """tfb200_mat view of a 2-D row-major tensor (unit column stride)."""
    assert t.dim() == 2 and (t.stride(1) == 1 or t.shape[1] <= 1)
    ld = t.stride(0) if t.shape[0] > 1 else max(t.shape[1], 1)
    return L.Mat(t.data_ptr(), t.shape[0], t.shape[1], max(ld, t.shape[1], 1), L.TFB200_BF16)


def _vec(t: torch.Tensor | None, n: int, name: str):
    if t is None:
        return None
    if not t.is_cuda or t.dtype != torch.bfloat16:
        raise TypeError(f"{name} must be a CUDA bfloat16 tensor")
    t = t.reshape(-1)
    if t.numel() != n:
        raise ValueError(f"{name} has {t.numel()} elements, expected {n}")
    return t.contiguous()


def matmul(a: torch.Tensor, b: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """``a @ b`` with fp32 accumulation and a bf16 result (golden.matmul)."""
    a2 = _rows2d(a, "a")
    b2 = _rows2d(b, "b")
    if a2.shape[1] != b2.shape[0]:
        raise ValueError(f"matmul: inner dimensions differ ({a2.shape[1]} vs {b2.shape[0]})")
    dev = _device_of(("a", a), ("b", b), ("out", out))
    y = out if out is not None else torch.empty(a2.shape[0], b2.shape[1], dtype=torch.bfloat16, device=a.device)
    with torch.cuda.device(dev):
        L.check(L.lib().tfb200_matmul(ctypes.byref(mat(a2)), ctypes.byref(mat(b2)), ctypes.byref(mat(y)),
                                      ctypes.c_void_p(stream_ptr())))
    return y.reshape(*a.shape[:-1], b2.shape[1]) if out is None else y


def rmsnorm_matmul_workspace_bytes(m: int, k: int, n: int) -> int:
    return int(L.lib().tfb200_fused_rmsnorm_matmul_workspace_size(m, k, n))


def _workspace(need: int, ws: torch.Tensor | None, device) -> torch.Tensor:
    """The caller's workspace, checked, or (when none is given) a new one. A workspace that is given but too small
    is an error, not a silent reallocation: callers pass one precisely to keep allocations out of their loop."""
    if ws is None:
        return torch.empty(max(need, 256), dtype=torch.uint8, device=device)
    if not ws.is_cuda or ws.device != device:
        raise ValueError(f"workspace must be on {device} (got {ws.device})")
    if not ws.is_contiguous():
        raise ValueError("workspace must be contiguous")
    if ws.numel() * ws.element_size() < need:
        raise ValueError(f"workspace holds {ws.numel() * ws.element_size()} bytes; this call needs {need}")
    return ws


def _device_of(*named) -> torch.device:
    """The one CUDA device of every operand given (name, tensor-or-None); the call then runs on that device's
    current stream."""
    dev = None
    for name, t in named:
        if t is None:
            continue
        if not isinstance(t, torch.Tensor) or not t.is_cuda:
            raise TypeError(f"{name} must be a CUDA tensor")
        if dev is None:
            dev = t.device
        elif t.device != dev:
            raise ValueError(f"{name} is on {t.device}; the other operands are on {dev}")
    return dev


def fused_rmsnorm_matmul(x: torch.Tensor, gamma: torch.Tensor, w: torch.Tensor, eps: float = 1e-6,
                         out: torch.Tensor | None = None, workspace: torch.Tensor | None = None) -> torch.Tensor:
    """``matmul(rmsnorm(x, gamma, eps), w)`` (golden.fused_rmsnorm_matmul)."""
    x2 = _rows2d(x, "x")
    w2 = _rows2d(w, "w")
    K = x2.shape[1]
    if w2.shape[0] != K:
        raise ValueError(f"fused_rmsnorm_matmul: x has K={K} but w has {w2.shape[0]} rows")
    g = _vec(gamma, K, "gamma")
    dev = _device_of(("x", x), ("gamma", gamma), ("w", w), ("out", out))
    y = out if out is not None else torch.empty(x2.shape[0], w2.shape[1], dtype=torch.bfloat16, device=x.device)
    ws = _workspace(rmsnorm_matmul_workspace_bytes(x2.shape[0], K, w2.shape[1]), workspace, dev)
    with torch.cuda.device(dev):
        L.check(L.lib().tfb200_fused_rmsnorm_matmul(ctypes.byref(mat(x2)), ctypes.c_void_p(g.data_ptr()),
                                                    ctypes.byref(mat(w2)), ctypes.c_float(eps), ctypes.byref(mat(y)),
                                                    ctypes.c_void_p(stream_ptr()), ctypes.c_void_p(ws.data_ptr()),
                                                    ctypes.c_size_t(ws.numel() * ws.element_size())))
    return y.reshape(*x.shape[:-1], w2.shape[1]) if out is None else y


def mlp_workspace_bytes(m: int, k: int, h: int, n: int) -> int:
    return int(L.lib().tfb200_fused_mlp_workspace_size(m, k, h, n))


_GELU = {"erf": L.TFB200_GELU_ERF, "tanh": L.TFB200_GELU_TANH}


def fused_mlp(x: torch.Tensor, gamma: torch.Tensor, w1: torch.Tensor, b1: torch.Tensor | None,
              w2: torch.Tensor, residual: torch.Tensor, eps: float = 1e-6, gelu: str = "erf",
              out: torch.Tensor | None = None, workspace: torch.Tensor | None = None) -> torch.Tensor:
    """``(gelu(rmsnorm(x) @ w1 + b1) @ w2) + residual`` (golden.fused_mlp).

    ``b1`` is the 1-D ``[H]`` bias the dialect's verifier accepts
    (TensixflowOps.cpp:329-335); a full-rank bias whose rows are all equal may be
    passed and is reduced to its first row.
    """
    x2 = _rows2d(x, "x")
    W1 = _rows2d(w1, "w1")
    W2 = _rows2d(w2, "w2")
    r2 = _rows2d(residual, "residual")
    M, K = x2.shape
    H = W1.shape[1]
    N = W2.shape[1]
    if W1.shape[0] != K or W2.shape[0] != H:
        raise ValueError("fused_mlp: shapes do not chain (x[M,K] @ w1[K,H] @ w2[H,N])")
    if r2.shape != (M, N):
        raise ValueError(f"fused_mlp: residual must be [{M},{N}] (got {tuple(r2.shape)})")
    if b1 is not None and b1.dim() > 1:
        b1 = b1.reshape(-1, b1.shape[-1])[0]
    b = _vec(b1, H, "b1")
    g = _vec(gamma, K, "gamma")
    if gelu not in _GELU:
        raise ValueError(f"gelu must be 'erf' or 'tanh' (got {gelu!r})")
    dev = _device_of(("x", x), ("gamma", gamma), ("w1", w1), ("b1", b1), ("w2", w2), ("residual", residual),
                     ("out", out))
    y = out if out is not None else torch.empty(M, N, dtype=torch.bfloat16, device=x.device)
    workspace = _workspace(mlp_workspace_bytes(M, K, H, N), workspace, dev)
    with torch.cuda.device(dev):
        L.check(L.lib().tfb200_fused_mlp(
            ctypes.byref(mat(x2)), ctypes.c_void_p(g.data_ptr()), ctypes.byref(mat(W1)),
            ctypes.c_void_p(b.data_ptr() if b is not None else None), ctypes.byref(mat(W2)), ctypes.byref(mat(r2)),
            ctypes.c_float(eps), ctypes.c_int(_GELU[gelu]), ctypes.byref(mat(y)), ctypes.c_void_p(stream_ptr()),
            ctypes.c_void_p(workspace.data_ptr()), ctypes.c_size_t(workspace.numel() * workspace.element_size())))
    return y.reshape(*x.shape[:-1], N) if out is None else y


def fused_mlp_partial(x: torch.Tensor, gamma: torch.Tensor, w1_shard: torch.Tensor, b1_shard: torch.Tensor | None,
                      w2_shard: torch.Tensor, eps: float = 1e-6, gelu: str = "erf",
                      out: torch.Tensor | None = None, workspace: torch.Tensor | None = None) -> torch.Tensor:
    """One GPU's share of a tensor-parallel MLP: fp32 ``gelu(rmsnorm(x) @ w1_shard + b1_shard) @ w2_shard``
    (W1 split by columns, W2 by rows). Sum over GPUs, then ``residual_add``."""
    x2 = _rows2d(x, "x")
    W1 = _rows2d(w1_shard, "w1_shard")
    W2 = _rows2d(w2_shard, "w2_shard")
    M, K = x2.shape
    H, N = W1.shape[1], W2.shape[1]
    if W1.shape[0] != K or W2.shape[0] != H:
        raise ValueError("fused_mlp_partial: shapes do not chain")
    b = _vec(b1_shard, H, "b1_shard")
    g = _vec(gamma, K, "gamma")
    if gelu not in _GELU:
        raise ValueError(f"gelu must be 'erf' or 'tanh' (got {gelu!r})")
    dev = _device_of(("x", x), ("gamma", gamma), ("w1_shard", w1_shard), ("b1_shard", b1_shard),
                     ("w2_shard", w2_shard), ("out", out))
    y = out if out is not None else torch.empty(M, N, dtype=torch.float32, device=x.device)
    ws = _workspace(int(L.lib().tfb200_fused_mlp_partial_workspace_size(M, K, H, N)), workspace, dev)
    with torch.cuda.device(dev):
        L.check(L.lib().tfb200_fused_mlp_partial(
            ctypes.byref(mat(x2)), ctypes.c_void_p(g.data_ptr()), ctypes.byref(mat(W1)),
            ctypes.c_void_p(b.data_ptr() if b is not None else None), ctypes.byref(mat(W2)), ctypes.c_float(eps),
            ctypes.c_int(_GELU[gelu]), ctypes.c_void_p(y.data_ptr()), ctypes.c_int64(y.stride(0)),
            ctypes.c_void_p(stream_ptr()), ctypes.c_void_p(ws.data_ptr()),
            ctypes.c_size_t(ws.numel() * ws.element_size())))
    return y


def fused_mlp_tp(x: torch.Tensor, gamma: torch.Tensor, w1_shard: torch.Tensor, b1_shard: torch.Tensor | None,
                 w2_shard: torch.Tensor, residual: torch.Tensor, comm: L.TpComm, eps: float = 1e-6,
                 gelu: str = "erf", workspace: torch.Tensor | None = None) -> None:
    """One rank's call of the tensor-parallel MLP whose all-reduce is fused into the down-projection kernel
    (``tfb200_fused_mlp_tp``). The result lands in every rank's ``comm.out`` buffer; ``tp.TPDecodeMLPFused``
    owns the buffers and the epoch."""
    x2 = _rows2d(x, "x")
    W1 = _rows2d(w1_shard, "w1_shard")
    W2 = _rows2d(w2_shard, "w2_shard")
    r2 = _rows2d(residual, "residual")
    M, K = x2.shape
    H, N = W1.shape[1], W2.shape[1]
    if W1.shape[0] != K or W2.shape[0] != H:
        raise ValueError("fused_mlp_tp: shapes do not chain")
    if tuple(r2.shape) != (M, N):
        raise ValueError(f"fused_mlp_tp: residual must be [{M},{N}] (got {tuple(r2.shape)})")
    if gelu not in _GELU:
        raise ValueError(f"gelu must be 'erf' or 'tanh' (got {gelu!r})")
    b = _vec(b1_shard, H, "b1_shard")
    g = _vec(gamma, K, "gamma")
    dev = _device_of(("x", x), ("gamma", gamma), ("w1_shard", w1_shard), ("b1_shard", b1_shard),
                     ("w2_shard", w2_shard), ("residual", residual))
    ws = _workspace(int(L.lib().tfb200_fused_mlp_partial_workspace_size(M, K, H, N)), workspace, dev)
    with torch.cuda.device(dev):
        L.check(L.lib().tfb200_fused_mlp_tp(
            ctypes.byref(mat(x2)), ctypes.c_void_p(g.data_ptr()), ctypes.byref(mat(W1)),
            ctypes.c_void_p(b.data_ptr() if b is not None else None), ctypes.byref(mat(W2)), ctypes.byref(mat(r2)),
            ctypes.c_float(eps), ctypes.c_int(_GELU[gelu]), ctypes.byref(comm), ctypes.c_void_p(stream_ptr()),
            ctypes.c_void_p(ws.data_ptr()), ctypes.c_size_t(ws.numel() * ws.element_size())))


def residual_add(partial: torch.Tensor, residual: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """``bf16(partial + residual)``: the tail of the tensor-parallel MLP."""
    if partial.dtype != torch.float32 or partial.dim() != 2 or partial.stride(1) != 1:
        raise TypeError("partial must be a row-major fp32 matrix")
    r2 = _rows2d(residual, "residual")
    if tuple(r2.shape) != tuple(partial.shape):
        raise ValueError("residual and partial shapes differ")
    dev = _device_of(("partial", partial), ("residual", residual), ("out", out))
    y = out if out is not None else torch.empty(r2.shape, dtype=torch.bfloat16, device=partial.device)
    with torch.cuda.device(dev):
        L.check(L.lib().tfb200_residual_add(ctypes.c_void_p(partial.data_ptr()), ctypes.c_int64(partial.stride(0)),
                                            ctypes.byref(mat(r2)), ctypes.byref(mat(y)),
                                            ctypes.c_void_p(stream_ptr())))
    return y


# ------------------------------------------------- 8-bit integer operators

_GELU_INT8 = {**_GELU, "none": L.TFB200_GELU_NONE, None: L.TFB200_GELU_NONE}
_DTYPES = {torch.bfloat16: L.TFB200_BF16, torch.float32: L.TFB200_F32, torch.int8: L.TFB200_I8}

# A decode step makes these calls while the GPU waits for them, so each looks at a tensor once, through the accessors
# that build no Python objects: ``_rows`` and ``_out`` return the operand's C descriptor beside its shape, devices are
# compared by index (25 us of host time a product with torch.cuda's accessors, 11 us without).
_Tensor = torch.Tensor
_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)  # absent from builds of torch without CUDA
_BF16, _F32, _I8 = torch.bfloat16, torch.float32, torch.int8


def _bad(t, name: str, dtype: torch.dtype, dev: int):
    if not isinstance(t, _Tensor) or not t.is_cuda:
        return TypeError(f"{name} must be a CUDA tensor")
    if t.dtype != dtype:
        return TypeError(f"{name} must be {dtype} (got {t.dtype})")
    return ValueError(f"{name} is on {t.device}; the other operands are on cuda:{dev}")


def _first(t, name: str) -> int:
    """The device index of a call's first operand."""
    if not isinstance(t, _Tensor) or not t.is_cuda:
        raise TypeError(f"{name} must be a CUDA tensor")
    return t.get_device()


def _rows(t: torch.Tensor, name: str, dtype: torch.dtype, dev: int, two_d: bool = False):
    """(rows, columns, tfb200_mat, tensor) of an operand: leading dimensions flattened, unit column stride, rows that
    do not overlap. A view that is not so is copied; the tensor keeps the memory alive."""
    if not isinstance(t, _Tensor) or t.dtype is not dtype or t.get_device() != dev:
        raise _bad(t, name, dtype, dev)
    n = t.dim()
    if n != 2:
        if n < 2 or two_d:
            raise ValueError(f"{name} must have {'' if two_d else 'at least '}2 dimensions (got {n})")
        t = t.reshape(math.prod(t.shape[:-1]), t.shape[-1])
    rows, cols = t.shape
    ld, unit = t.stride()
    if (unit != 1 and cols > 1) or (ld < cols and rows > 1):
        t = t.contiguous()
        ld = cols
    return rows, cols, L.Mat(t.data_ptr(), rows, cols, ld if rows > 1 and ld > 0 else cols or 1, _DTYPES[dtype]), t


def _rows_int8(t: torch.Tensor, name: str, dev: int, two_d: bool = False):
    """``_rows`` of a product's int8 operand. The tensor cores' copies need rows on 16-byte boundaries; an operand laid
    out otherwise is copied so, which takes a fraction of the time the product would take on it as it is."""
    r = _rows(t, name, _I8, dev, two_d)
    rows, cols, mat, t = r
    if rows and cols and ((mat.data & 15) or (rows > 1 and mat.ld & 15)):
        q, r = _new_int8((rows, cols), rows, t.device)
        q.copy_(t)
    return r


def _out(t: torch.Tensor, name: str, dtype: torch.dtype, shape, dev: int):
    """``_rows`` of a caller's output, which is written in place: nothing is copied."""
    if not isinstance(t, _Tensor) or t.dtype != dtype or t.get_device() != dev:
        raise _bad(t, name, dtype, dev)
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must be {list(shape)} (got {list(t.shape)})")
    if t.dim() > 2:
        try:
            t = t.view(math.prod(shape[:-1]), shape[-1])
        except RuntimeError:
            raise ValueError(f"{name}: the leading dimensions must flatten into rows without a copy") from None
    r = _rows(t, name, dtype, dev)
    if r[3].data_ptr() != t.data_ptr():
        raise ValueError(f"{name} must have unit column stride and rows that do not overlap")
    return r


def _out_scale(t: torch.Tensor, n: int, dev: int) -> int:
    if not isinstance(t, _Tensor) or t.dtype != _F32 or t.get_device() != dev:
        raise _bad(t, "scale", _F32, dev)
    if t.numel() != n or not t.is_contiguous():
        raise ValueError(f"scale must be contiguous and have {n} elements (got {list(t.shape)})")
    return t.data_ptr()


def _vec1(t, n: int, name: str, dtype: torch.dtype, dev: int):
    """(address, tensor) of a contiguous vector of n elements (any shape); (None, None) for None."""
    if t is None:
        return None, None
    if not isinstance(t, _Tensor) or t.dtype is not dtype or t.get_device() != dev:
        raise _bad(t, name, dtype, dev)
    if t.numel() != n:
        raise ValueError(f"{name} has {t.numel()} elements, expected {n}")
    if not t.is_contiguous():
        t = t.reshape(-1).contiguous()
    return t.data_ptr(), t


def _space(need: int, ws: torch.Tensor | None, x: torch.Tensor):
    """(tensor, address, bytes) of the workspace of a call on x's device that needs `need` bytes."""
    if ws is None:
        if need == 0:
            return None, None, 0
        ws = torch.empty(need, dtype=torch.uint8, device=x.device)
        return ws, ws.data_ptr(), need
    ws = _workspace(need, ws, x.device)
    return ws, ws.data_ptr(), ws.numel() * ws.element_size()


def _call(dev: int, fn, *args) -> None:
    """One C call with device ``dev`` current."""
    if torch._C._cuda_getDevice() == dev:
        rc = fn(*args)
    else:
        with torch.cuda.device(dev):
            rc = fn(*args)
    if rc:
        L.check(rc)


_byref = ctypes.byref


def _ref(r):
    return None if r is None else _byref(r[2])


def _new_int8(shape, rows: int, dev):
    """A new int8 tensor of ``shape``, and as ``_rows``: its rows start a multiple of 16 bytes apart, as the products
    read best."""
    k = shape[-1]
    ld = (k + 15) // 16 * 16
    q = torch.empty(rows, ld, dtype=_I8, device=dev)
    mat = L.Mat(q.data_ptr(), rows, k, ld or 1, L.TFB200_I8)
    if ld != k:
        q = q[:, :k]
    return (q if len(shape) == 2 else q.unflatten(0, shape[:-1])), (rows, k, mat, q)


def quantize_int8(x: torch.Tensor, out: tuple | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """``(q, scale)``: int8 ``q = round(x * 127 / amax)`` of ``x``'s shape and fp32 ``scale = amax / 127`` of its
    leading dimensions, ``amax`` the largest magnitude of each row (last dimension). ``q`` is the fp32 product
    ``x * ((1 / amax) * 127)`` rounded to an integer, halves of that product to even.

    A weight ``w [in, out]`` is laid out for the products once: ``w_q, w_scale = quantize_int8(w.t())``. The rows of
    a returned ``q`` start 16 bytes apart or a multiple of it (its row stride may exceed its width); the products copy
    an operand laid out otherwise on every call. ``out = (q, scale)`` takes the results in place.
    """
    dev = _first(x, "x")
    xr = _rows(x, "x", _BF16, dev)
    rows = xr[0]
    if out is None:
        device = x.device
        q, qr = _new_int8(x.shape, rows, device)
        scale = torch.empty(x.shape[:-1], dtype=_F32, device=device)
        sp = scale.data_ptr()
    else:
        q, scale = out
        qr, sp = _out(q, "q", _I8, x.shape, dev), _out_scale(scale, rows, dev)
    _call(dev, L.lib().tfb200_quantize_int8, _byref(xr[2]), _byref(qr[2]), sp, _stream(dev))
    return q, scale


def rmsnorm_int8(x: torch.Tensor, gamma: torch.Tensor, eps: float = 1e-6, residual: torch.Tensor | None = None,
                 out: tuple | None = None) -> tuple:
    """``(q, scale)`` of ``rmsnorm(x, gamma, eps)``, quantised as ``quantize_int8`` does; with a ``residual``,
    ``(q, scale, sum)`` of ``rmsnorm(x + residual, gamma, eps)`` and ``sum = bf16(x + residual)``. The norm and ``q``
    are taken from the unrounded sum. ``out`` takes the results in place; its ``sum`` may be ``x`` or ``residual``.
    """
    dev = _first(x, "x")
    xr = _rows(x, "x", _BF16, dev)
    rows, K = xr[:2]
    g, gk = _vec1(gamma, K, "gamma", _BF16, dev)
    rr = tr = total = None
    if residual is not None:
        rr = _rows(residual, "residual", _BF16, dev)
        if residual.shape != x.shape:
            raise ValueError(f"residual must have the shape of x (got {list(residual.shape)})")
    if out is None:
        device = x.device
        q, qr = _new_int8(x.shape, rows, device)
        scale = torch.empty(x.shape[:-1], dtype=_F32, device=device)
        sp = scale.data_ptr()
        if rr is not None:
            total = torch.empty(x.shape, dtype=_BF16, device=device)
            tr = (rows, K, L.Mat(total.data_ptr(), rows, K, K or 1, L.TFB200_BF16), total)
    else:
        if len(out) != (2 if residual is None else 3):
            raise ValueError("out must be (q, scale), and (q, scale, sum) with a residual")
        q, scale = out[:2]
        qr, sp = _out(q, "q", _I8, x.shape, dev), _out_scale(scale, rows, dev)
        if rr is not None:
            total = out[2]
            tr = _out(total, "sum", _BF16, x.shape, dev)
    _call(dev, L.lib().tfb200_rmsnorm_int8, _byref(xr[2]), _ref(rr), g, eps, _ref(tr), _byref(qr[2]), sp, _stream(dev))
    return (q, scale) if residual is None else (q, scale, total)


def _result(x: torch.Tensor, rows: int, n: int, dtype: torch.dtype, out: torch.Tensor | None, dev: int):
    """A product's output, [..., N] for an input [..., K] (a caller's may also be given as [rows, N])."""
    if out is None:
        y = torch.empty(rows, n, dtype=dtype, device=x.device)
        r = (rows, n, L.Mat(y.data_ptr(), rows, n, n or 1, _DTYPES[dtype]), y)
        return (y if x.dim() == 2 else y.view(*x.shape[:-1], n)), r
    return out, _out(out, "out", dtype, (rows, n) if out.dim() == 2 else (*x.shape[:-1], n), dev)


def matmul_int8_workspace_bytes(m: int, k: int, n: int) -> int:
    return L.lib().tfb200_matmul_int8_workspace_size(m, k, n)


def matmul_int8(a: torch.Tensor, a_scale: torch.Tensor, b: torch.Tensor, b_scale: torch.Tensor,
                bias: torch.Tensor | None = None, gelu: str | None = None, residual: torch.Tensor | None = None,
                out_dtype: torch.dtype = torch.bfloat16, out: torch.Tensor | None = None,
                workspace: torch.Tensor | None = None) -> torch.Tensor:
    """``gelu((a * a_scale) @ (b * b_scale).T + bias) + residual`` of int8 ``a [..., K]`` and ``b [N, K]``, one scale
    per row of each; exact integer sums, the rest in fp32 steps, the result rounded to ``out_dtype`` (bf16 or fp32).
    ``bias`` is bf16 ``[N]``, ``gelu`` "erf", "tanh" or None, ``residual`` bf16 ``[..., N]``. K is at most 131071.
    """
    dev = _first(a, "a")
    ar = _rows_int8(a, "a", dev)
    M, K = ar[:2]
    br = _rows_int8(b, "b", dev, True)
    N = br[0]
    if br[1] != K:
        raise ValueError(f"matmul_int8: a has K={K} but b has {br[1]} columns")
    if out_dtype is not _BF16 and out_dtype is not _F32:
        raise TypeError(f"out_dtype must be bfloat16 or float32 (got {out_dtype})")
    if gelu not in _GELU_INT8:
        raise ValueError(f"gelu must be 'erf', 'tanh' or None (got {gelu!r})")
    sa, sak = _vec1(a_scale, M, "a_scale", _F32, dev)
    sb, sbk = _vec1(b_scale, N, "b_scale", _F32, dev)
    bv, bvk = _vec1(bias, N, "bias", _BF16, dev)
    rr = None
    if residual is not None:
        rr = _rows(residual, "residual", _BF16, dev)
        if rr[0] != M or rr[1] != N:
            raise ValueError(f"residual must be [{M},{N}] (got {list(residual.shape)})")
    y, yr = _result(a, M, N, out_dtype, out, dev)
    lib = L.lib()
    ws, wp, wn = _space(lib.tfb200_matmul_int8_workspace_size(M, K, N), workspace, a)
    _call(dev, lib.tfb200_matmul_int8, _byref(ar[2]), sa, _byref(br[2]), sb, bv, _GELU_INT8[gelu], _ref(rr),
          _byref(yr[2]), _stream(dev), wp, wn)
    return y


def rmsnorm_matmul_int8_workspace_bytes(m: int, k: int, n: int) -> int:
    return L.lib().tfb200_fused_rmsnorm_matmul_int8_workspace_size(m, k, n)


def fused_rmsnorm_matmul_int8(x: torch.Tensor, gamma: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor,
                              eps: float = 1e-6, out: torch.Tensor | None = None,
                              workspace: torch.Tensor | None = None) -> torch.Tensor:
    """``rmsnorm(x, gamma, eps) @ w`` on int8 ``w [N, K]`` with ``w_scale [N]``: ``fused_rmsnorm_matmul`` with the
    normalised rows quantised per token (``rmsnorm_int8``, then ``matmul_int8``)."""
    dev = _first(x, "x")
    xr = _rows(x, "x", _BF16, dev)
    M, K = xr[:2]
    wr = _rows_int8(w, "w", dev, True)
    N = wr[0]
    if wr[1] != K:
        raise ValueError(f"fused_rmsnorm_matmul_int8: x has K={K} but w has {wr[1]} columns")
    g, gk = _vec1(gamma, K, "gamma", _BF16, dev)
    sw, swk = _vec1(w_scale, N, "w_scale", _F32, dev)
    y, yr = _result(x, M, N, _BF16, out, dev)
    lib = L.lib()
    ws, wp, wn = _space(lib.tfb200_fused_rmsnorm_matmul_int8_workspace_size(M, K, N), workspace, x)
    _call(dev, lib.tfb200_fused_rmsnorm_matmul_int8, _byref(xr[2]), g, _byref(wr[2]), sw, eps, _byref(yr[2]),
          _stream(dev), wp, wn)
    return y


def mlp_int8_workspace_bytes(m: int, k: int, h: int, n: int) -> int:
    return L.lib().tfb200_fused_mlp_int8_workspace_size(m, k, h, n)


def fused_mlp_int8(x: torch.Tensor, gamma: torch.Tensor, w1: torch.Tensor, w1_scale: torch.Tensor,
                   b1: torch.Tensor | None, w2: torch.Tensor, w2_scale: torch.Tensor, residual: torch.Tensor,
                   eps: float = 1e-6, gelu: str = "erf", out: torch.Tensor | None = None,
                   workspace: torch.Tensor | None = None) -> torch.Tensor:
    """``fused_mlp`` on int8 ``w1 [H, K]`` and ``w2 [N, H]`` with a scale per row: the normalised rows and the hidden
    block (fp32 until then) are quantised per token. ``b1`` is a bf16 ``[H]`` bias or None."""
    dev = _first(x, "x")
    xr = _rows(x, "x", _BF16, dev)
    M, K = xr[:2]
    w1r, w2r = _rows_int8(w1, "w1", dev, True), _rows_int8(w2, "w2", dev, True)
    H, N = w1r[0], w2r[0]
    if w1r[1] != K or w2r[1] != H:
        raise ValueError("fused_mlp_int8: shapes do not chain (x[M,K], w1[H,K], w2[N,H])")
    rr = _rows(residual, "residual", _BF16, dev)
    if rr[0] != M or rr[1] != N:
        raise ValueError(f"fused_mlp_int8: residual must be [{M},{N}] (got {list(residual.shape)})")
    if gelu not in _GELU:
        raise ValueError(f"gelu must be 'erf' or 'tanh' (got {gelu!r})")
    g, gk = _vec1(gamma, K, "gamma", _BF16, dev)
    b, bk = _vec1(b1, H, "b1", _BF16, dev)
    s1, s1k = _vec1(w1_scale, H, "w1_scale", _F32, dev)
    s2, s2k = _vec1(w2_scale, N, "w2_scale", _F32, dev)
    y, yr = _result(x, M, N, _BF16, out, dev)
    lib = L.lib()
    ws, wp, wn = _space(lib.tfb200_fused_mlp_int8_workspace_size(M, K, H, N), workspace, x)
    _call(dev, lib.tfb200_fused_mlp_int8, _byref(xr[2]), g, _byref(w1r[2]), s1, b, _byref(w2r[2]), s2, _byref(rr[2]),
          eps, _GELU[gelu], _byref(yr[2]), _stream(dev), wp, wn)
    return y
