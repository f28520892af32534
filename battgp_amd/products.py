"""Matrix products next to the exact-GP engine's own (``ExactGPEngine.gemm_nt_sub_device``: one pair of fp64 operands):
products grouped by expert with ragged sizes, their gradients, and products in 8-bit integers with one scale per row.

torch tensors on the GPU in and out, in fp64, fp32, bf16 and fp16.  Every function enqueues its kernels on the current
torch stream of the tensors' device and returns without waiting for them; nothing is kept between calls, so the calls can
be captured into a graph and come from several threads.  The kernels run in libbattgp_products.so
(``include/battgp_products.h``); there is no fallback.  An ordinary call goes there by way of ``_products_torch``
(``csrc/products/torch_calls.cpp``); whatever that does not take - an ``out``, a part of the gradients, a wrong argument - goes
through the checks below.  Like the engine's ``lml_grad``, gradients are calls of their own:
no function records an autograd graph, and inputs that ask for one, or that carry a forward-mode tangent, are refused.
"""

from __future__ import annotations

import torch
from torch.autograd.graph import increment_version  # a given output is written in place: autograd is to notice

from . import _lib
from .engine import EngineError

_lib.load_products()  # first: the module below is linked against it
try:
    from . import _products_torch as _calls
except ImportError as exc:
    raise ImportError(f"battgp_amd/_products_torch.so can not be loaded ({exc}): build it with `python -m battgp_amd.build`") from exc

DTYPES = {torch.float64: _lib.F64, torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}
INT8_MAX_K = _lib.INT8_MAX_K
MAX_GROUPS = _lib.MAX_GROUPS


FIRST_DEVICE = 0  # torch's index of the first device there is a kernel for; the CPU's is below it
_Tensor, _strided, _int64, _int8 = torch.Tensor, torch.strided, torch.int64, torch.int8  # looked up once: a call is a few us


def _call(name: str, like: torch.Tensor, *args) -> None:
    """A C entry that may ask for a workspace: torch's allocator gives it, on the stream that the call uses."""
    lib = _lib.load_products()
    entry = getattr(lib, name)
    rc = entry(*args, None, 0)
    if rc > 0:
        work = like.new_empty(rc, dtype=torch.uint8)
        rc = entry(*args, work.data_ptr(), rc)
    if rc != 0:
        raise EngineError(lib.bgp_products_last_error().decode())


def _gpu_tensor(name: str, t, dim: int, device: int | None = None) -> int:
    """the index of the device that ``t`` is on (checks are written for the call that passes: they cost a call its time)"""
    if not isinstance(t, _Tensor):
        raise TypeError(f"{name} is not a torch tensor")
    if t.layout is not _strided or t.is_neg():
        raise ValueError(f"{name} is not a dense tensor that holds its own values")
    if t.dim() != dim:
        raise ValueError(f"{name} has {t.dim()} dimensions, {dim} are wanted")
    at = t.get_device()
    if at != device:
        if at < FIRST_DEVICE:
            raise EngineError(f"{name} is on {t.device}: battgp_amd runs on MI355X only")
        if device is not None:
            raise ValueError(f"{name} is on {t.device}, the other operands are on device {device}")
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} requires a gradient: battgp_amd.products records no autograd graph; detach it and call the gradient's function")
    other = _calls.stands_for(t)
    if other == 1:  # inside vmap, jvp and grad, and wrappers, whose pointer may read as NULL
        raise ValueError(f"{name} is not a dense tensor that holds its own values")
    if other == 2:
        raise ValueError(f"{name} has a tangent: battgp_amd.products does not carry forward-mode gradients along")
    return at


def _float_type(name: str, dtype) -> int:
    code = DTYPES.get(dtype)
    if code is None:
        raise ValueError(f"{name}: {dtype} is not one of float64, float32, bfloat16, float16")
    return code


def _rows(name: str, t: torch.Tensor, m: int, n: int) -> int:
    """Leading dimension of t[m, n], whose rows are contiguous (a dimension of one element has no stride of its own)."""
    ld, inner = t.stride()
    if inner != 1 and n > 1:
        raise ValueError(f"{name}: the elements of a row have to be contiguous, strides are {t.stride()}")
    if m <= 1:
        return n or 1
    if ld < n:
        raise ValueError(f"{name}: rows overlap, strides are {t.stride()}")
    return ld or 1


def _weights(w: torch.Tensor, g: int, n: int, k: int) -> tuple[int, int, int]:
    """(stride of a group, leading dimension, 1 if the output axis is the contiguous one) of w[g, n, k]."""
    sg, sn, sk = w.stride()
    if g <= 1:
        sg = 0
    if (sk == 1 or k <= 1) and (sn >= (k or 1) or n <= 1):
        return sg, (sn if n > 1 else k or 1), 0
    if (sn == 1 or n <= 1) and (sk >= (n or 1) or k <= 1):
        return sg, (sk if k > 1 else n or 1), 1
    raise ValueError(f"w: either axis of a group's weights has to be contiguous, strides are {w.stride()}")


def _span(t: torch.Tensor) -> tuple[int, int]:
    if t.numel() == 0:
        return 0, 0
    last = sum((s - 1) * st for s, st in zip(t.shape, t.stride()))
    return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()


def _between_columns(out: torch.Tensor, t: torch.Tensor) -> bool:
    """Whether ``t`` lies beside the columns of ``out``: both in pieces that recur at the same distance in memory."""
    pitch, width, size = out.stride(0) * out.element_size(), 1, t.element_size()
    if pitch == 0:
        return False
    for n, stride in zip(t.shape, t.stride()):
        if n > 1 and stride == 1:
            width += n - 1
        elif n > 1 and stride * size % pitch:
            return False
    at = (t.data_ptr() - out.data_ptr()) % pitch
    return at >= out.shape[1] * out.element_size() and at + width * size <= pitch


def _output(out, name: str, shape, dtype, device: int, inputs, added=None) -> torch.Tensor:
    """``out``, checked; it may be ``added`` itself, and lies apart from everything else"""
    if _gpu_tensor(name, out, len(shape)) != device or out.dtype is not dtype or tuple(out.shape) != shape:
        raise ValueError(f"{name}: {shape} of {dtype} on device {device} is wanted, got {tuple(out.shape)} of {out.dtype} on {out.device}")
    if added is not None and not (added.data_ptr() == out.data_ptr() and added.stride() == out.stride()):
        inputs = (*inputs, added)
    lo, hi = _span(out)
    for t in inputs:
        a, b = _span(t)
        if a < hi and lo < b and not _between_columns(out, t):
            raise ValueError(f"{name} overlaps an input")
    return out


def _stream(device: int) -> int:
    return torch._C._cuda_getCurrentRawStream(device)  # current_stream(device).cuda_stream, without the objects around it


def _offsets(offsets, groups: int, device: int) -> None:
    _gpu_tensor("offsets", offsets, 1, device)
    if offsets.dtype is not _int64:
        raise ValueError(f"offsets are {offsets.dtype}, int64 is wanted")
    if offsets.numel() != groups + 1:
        raise ValueError(f"{offsets.numel()} offsets for {groups} groups, {groups + 1} are wanted")
    if groups > MAX_GROUPS:
        raise ValueError(f"{groups} groups, at most {MAX_GROUPS} are possible")
    if not offsets.is_contiguous():
        raise ValueError("offsets are not contiguous")


def _grouped(device, dtype, x, w, offsets, out, t, n, k, g):
    """out[t, :] = x[t, :] w_g^T; w may be any view of [G, N, K] that _weights takes"""
    sw, ldw, trans = _weights(w, g, n, k)
    ldx = _rows("x", x, t, k)
    if out is None:
        y, ldy = x.new_empty((t, n)), n or 1
    else:
        y = _output(out, "out", (t, n), x.dtype, device, (x, w, offsets))
        ldy = _rows("out", y, t, n)
        increment_version(y)
    _call(
        "bgp_grouped_gemm", x, device, _stream(device), dtype, t, n, k, g, x.data_ptr(), ldx, w.data_ptr(), sw, ldw, trans,
        offsets.data_ptr(), y.data_ptr(), ldy, out is None,
    )
    return y


def grouped_matmul(x: torch.Tensor, w: torch.Tensor, offsets: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """``y[t] = w[g] @ x[t]`` for the rows ``offsets[g] <= t < offsets[g + 1]`` of every group ``g``.

    ``x [T, K]`` with contiguous rows, sorted by group; ``w [G, N, K]`` with either of its last two axes contiguous
    (``w.transpose(1, 2)`` of stored ``[G, K, N]`` weights is taken as it is; ``expand`` shares weights); ``offsets
    [G + 1]`` int64 on the device, ascending, within ``[0, T]`` - they are never read on the host.  Groups may be empty.
    Rows in no group are 0 in a new output and left as they are in a given ``out``.  Sums are held in fp32 (fp64 for
    fp64) and rounded once."""
    if out is None:
        y = _calls.grouped(x, w, offsets)
        if y is not None:
            return y
    device = _gpu_tensor("x", x, 2)
    _gpu_tensor("w", w, 3, device)
    dtype = _float_type("x", x.dtype)
    if w.dtype is not x.dtype:
        raise ValueError(f"x is {x.dtype}, w is {w.dtype}")
    t, k = x.shape
    g, n, wk = w.shape
    if wk != k:
        raise ValueError(f"x has {k} columns, w has {wk}")
    _offsets(offsets, g, device)
    return _grouped(device, dtype, x, w, offsets, out, t, n, k, g)


def grouped_matmul_grad(dy: torch.Tensor, x: torch.Tensor, w: torch.Tensor, offsets: torch.Tensor, need_dx: bool = True, need_dw: bool = True):
    """Gradients of :func:`grouped_matmul` for ``dy [T, N]``: ``(dx [T, K], dw [G, N, K])``, ``None`` for one that is not
    needed.  ``dx`` is 0 in rows of no group, ``dw`` is 0 for an empty group; both are new and contiguous, and for shared
    weights (``expand``) ``dw`` still holds each group's own share."""
    if need_dx and need_dw:
        both = _calls.grouped_grad(dy, x, w, offsets)
        if both is not None:
            return both
    device = _gpu_tensor("x", x, 2)
    _gpu_tensor("dy", dy, 2, device)
    _gpu_tensor("w", w, 3, device)
    dtype = _float_type("x", x.dtype)
    if w.dtype is not x.dtype or dy.dtype is not x.dtype:
        raise ValueError(f"x is {x.dtype}, w is {w.dtype}, dy is {dy.dtype}")
    t, k = x.shape
    g, n, wk = w.shape
    if wk != k or tuple(dy.shape) != (t, n):
        raise ValueError(f"dy {tuple(dy.shape)}, x {tuple(x.shape)} and w {tuple(w.shape)} do not belong together")
    _offsets(offsets, g, device)
    lddy, ldx = _rows("dy", dy, t, n), _rows("x", x, t, k)
    dx = dw = None
    if need_dx:
        dx = _grouped(device, dtype, dy, w.transpose(1, 2), offsets, None, t, k, n, g)
    if need_dw:
        dw = x.new_empty((g, n, k))
        _call(
            "bgp_grouped_gemm_dw", x, device, _stream(device), dtype, t, n, k, g, dy.data_ptr(), lddy, x.data_ptr(), ldx,
            offsets.data_ptr(), dw.data_ptr(), n * (k or 1), k or 1,
        )
    return dx, dw


def _scale_type(dtype):
    return torch.float64 if dtype is torch.float64 else torch.float32


def quantize_rows(x: torch.Tensor, pow2: bool = False, residual: bool = False):
    """``(q, scale)`` or ``(q, scale, rest)``: 8-bit codes of the rows of ``x [M, K]``, one scale each, ``x ~ scale * q``.

    ``scale = max |row| / 127`` (fp64 for fp64, else fp32), or with ``pow2`` the smallest power of two ``p`` with
    ``max |row| <= 127 p``; at least the smallest normal number.  ``q`` is rounded to the nearest, ties to even.
    ``rest = x - scale * q``, exact with ``pow2``: quantising it again gives the next slice of the row.  A row with an
    infinity or a NaN has that for its scale, and codes 0."""
    made = _calls.quantize(x, pow2, residual)
    if made is not None:
        return made
    device = _gpu_tensor("x", x, 2)
    dtype = _float_type("x", x.dtype)
    m, k = x.shape
    ldx = _rows("x", x, m, k)
    q = x.new_empty((m, k), dtype=torch.int8)
    scale = x.new_empty(m, dtype=_scale_type(x.dtype))
    rest = x.new_empty((m, k)) if residual else None
    lib = _lib.load_products()
    rc = lib.bgp_quantize_rows(
        device, _stream(device), dtype, m, k, x.data_ptr(), ldx, q.data_ptr(), k or 1, scale.data_ptr(), bool(pow2), rest.data_ptr() if residual else None,
        k or 1,
    )
    if rc != 0:
        raise EngineError(lib.bgp_products_last_error().decode())
    return (q, scale, rest) if residual else (q, scale)


def _scale(name: str, s, rows: int, dtype, device: int) -> None:
    _gpu_tensor(name, s, 1, device)
    if s.dtype is not dtype or s.numel() != rows or not s.is_contiguous():
        raise ValueError(f"{name}: {rows} contiguous values of {dtype} are wanted for this result")


def int8_matmul(
    a: torch.Tensor, b: torch.Tensor, a_scale: torch.Tensor, b_scale: torch.Tensor, c: torch.Tensor | None = None,
    dtype: torch.dtype = torch.bfloat16, out: torch.Tensor | None = None,
) -> torch.Tensor:
    """``y[i, j] = (c[i, j] +) a_scale[i] * b_scale[j] * sum_k a[i, k] b[j, k]`` in ``dtype``.

    ``a [M, K]`` and ``b [N, K]`` int8 with contiguous rows, ``K <= 131071`` (the sum is exact in 32 bits);
    scales fp64 for a fp64 result, else fp32; ``c`` and ``out`` of the result's type, ``out`` may be ``c`` itself.  The
    scaling and the sum with ``c`` are computed in fp64 and rounded once."""
    if out is None:
        y = _calls.int8(a, b, a_scale, b_scale, c, DTYPES.get(dtype, -1))
        if y is not None:
            return y
    device = _gpu_tensor("a", a, 2)
    _gpu_tensor("b", b, 2, device)
    code = _float_type("dtype", dtype)
    if a.dtype is not _int8 or b.dtype is not _int8:
        raise ValueError(f"a is {a.dtype}, b is {b.dtype}: int8 is wanted")
    m, k = a.shape
    n, bk = b.shape
    if bk != k:
        raise ValueError(f"a has {k} columns, b has {bk}")
    if k > INT8_MAX_K:
        raise ValueError(f"{k} columns: a sum over more than {INT8_MAX_K} can pass 32 bits")
    stype = _scale_type(dtype)
    _scale("a_scale", a_scale, m, stype, device)
    _scale("b_scale", b_scale, n, stype, device)
    cp, ldc = None, 0
    if c is not None:
        _gpu_tensor("c", c, 2, device)
        if c.dtype is not dtype or tuple(c.shape) != (m, n):
            raise ValueError(f"c: {(m, n)} of {dtype} is wanted, got {tuple(c.shape)} of {c.dtype}")
        cp, ldc = c.data_ptr(), _rows("c", c, m, n)
    lda, ldb = _rows("a", a, m, k), _rows("b", b, n, k)
    if out is None:
        y, ldy = a.new_empty((m, n), dtype=dtype), n or 1
    else:
        y = _output(out, "out", (m, n), dtype, device, (a, b, a_scale, b_scale), c)
        ldy = _rows("out", y, m, n)
        increment_version(y)
    _call(
        "bgp_int8_gemm", a, device, _stream(device), code, m, n, k, a.data_ptr(), lda, b.data_ptr(), ldb, a_scale.data_ptr(),
        b_scale.data_ptr(), cp, ldc, y.data_ptr(), ldy,
    )
    return y
