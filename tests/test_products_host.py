"""CPU tests of the grouped and 8-bit products: the library exports its header, wrong calls are refused before anything
reaches a GPU (the C entries by their own checks, the Python functions by theirs), and the Python functions hand the C
entries the sizes, strides and flags that the header asks for."""

import ctypes as C
import os
import re

import pytest
import torch

from battgp_amd import _lib, products
from battgp_amd.engine import EngineError

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_library_exports_every_declared_symbol():
    text = open(os.path.join(ROOT, "include", "battgp_products.h")).read()
    code = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    declared = sorted(set(re.findall(r"\b(bgp_[a-z_0-9]+)\s*\(", code)))
    lib = _lib.load_products()
    assert declared == sorted(_lib.PRODUCTS_SIGNATURES)
    for name in declared:
        assert hasattr(lib, name)
        args = re.search(name + r"\s*\((.*?)\);", code, flags=re.S).group(1).split(",")
        assert len(_lib.PRODUCTS_SIGNATURES[name][1]) == (0 if args == ["void"] else len(args)), name
    for name, val in (("BGP_F64", _lib.F64), ("BGP_F32", _lib.F32), ("BGP_BF16", _lib.BF16), ("BGP_F16", _lib.F16)):
        assert int(re.search(rf"{name}\s*=\s*(\d+)", code).group(1)) == val
    assert int(re.search(r"BGP_MAX_GROUPS\s+(\d+)", code).group(1)) == _lib.MAX_GROUPS
    assert int(re.search(r"BGP_INT8_MAX_K\s+(\d+)", code).group(1)) == _lib.INT8_MAX_K


P = C.c_void_p(4096)  # an address: none of these calls may follow it
GEMM = dict(device=0, stream=None, dtype=1, T=8, N=4, K=4, G=2, X=P, ldx=4, W=P, sW=16, ldw=4, trans=0, off=P, Y=P, ldy=4, zero=1, ws=None, wsb=0)
DW = dict(device=0, stream=None, dtype=1, T=8, N=4, K=4, G=2, dY=P, lddy=4, X=P, ldx=4, off=P, dW=P, sW=16, ldw=4, ws=None, wsb=0)
QUANT = dict(device=0, stream=None, dtype=1, M=4, K=8, x=P, ldx=8, q=P, ldq=8, scale=P, pow2=0, rest=None, ldr=8)
INT8 = dict(device=0, stream=None, dtype=1, M=4, N=4, K=8, A=P, lda=8, B=P, ldb=8, sa=P, sb=P, C=None, ldc=0, Y=P, ldy=4, ws=None, wsb=0)


@pytest.mark.parametrize(
    "name, base, change, text",
    [
        ("bgp_grouped_gemm", GEMM, dict(dtype=9), "type"),
        ("bgp_grouped_gemm", GEMM, dict(dtype=-1), "type"),
        ("bgp_grouped_gemm", GEMM, dict(T=-1), "sizes"),
        ("bgp_grouped_gemm", GEMM, dict(G=65536), "sizes"),
        ("bgp_grouped_gemm", GEMM, dict(off=None), "offsets"),
        ("bgp_grouped_gemm", GEMM, dict(X=None), "null"),
        ("bgp_grouped_gemm", GEMM, dict(Y=None), "null"),
        ("bgp_grouped_gemm", GEMM, dict(ldx=3), "strides"),
        ("bgp_grouped_gemm", GEMM, dict(ldw=3), "strides"),
        ("bgp_grouped_gemm", GEMM, dict(N=8, ldy=8, trans=1), "strides"),
        ("bgp_grouped_gemm", GEMM, dict(ldy=3), "strides"),
        ("bgp_grouped_gemm", GEMM, dict(sW=-1), "strides"),
        ("bgp_grouped_gemm", GEMM, dict(T=1 << 40, N=1 << 20, ldy=1 << 20), "launch"),
        ("bgp_grouped_gemm_dw", DW, dict(dtype=4), "type"),
        ("bgp_grouped_gemm_dw", DW, dict(N=-1), "sizes"),
        ("bgp_grouped_gemm_dw", DW, dict(off=None), "offsets"),
        ("bgp_grouped_gemm_dw", DW, dict(dW=None), "null"),
        ("bgp_grouped_gemm_dw", DW, dict(dY=None), "null"),
        ("bgp_grouped_gemm_dw", DW, dict(sW=15), "strides"),
        ("bgp_grouped_gemm_dw", DW, dict(lddy=3), "strides"),
        ("bgp_grouped_gemm_dw", DW, dict(N=1 << 20, K=1 << 20, lddy=1 << 20, ldx=1 << 20, ldw=1 << 20, sW=1 << 40), "launch"),
        ("bgp_quantize_rows", QUANT, dict(dtype=7), "type"),
        ("bgp_quantize_rows", QUANT, dict(K=-1), "sizes"),
        ("bgp_quantize_rows", QUANT, dict(scale=None), "null"),
        ("bgp_quantize_rows", QUANT, dict(q=None), "null"),
        ("bgp_quantize_rows", QUANT, dict(ldq=7), "strides"),
        ("bgp_quantize_rows", QUANT, dict(rest=P, ldr=7), "strides"),
        ("bgp_int8_gemm", INT8, dict(dtype=7), "type"),
        ("bgp_int8_gemm", INT8, dict(K=131072, lda=131072, ldb=131072), "32 bits"),
        ("bgp_int8_gemm", INT8, dict(sb=None), "null"),
        ("bgp_int8_gemm", INT8, dict(lda=7), "strides"),
        ("bgp_int8_gemm", INT8, dict(C=P, ldc=3), "strides"),
    ],
)
def test_c_entries_refuse_bad_arguments(name, base, change, text):
    lib = _lib.load_products()
    args = {**base, **change}
    rc = getattr(lib, name)(*args.values())
    err = lib.bgp_products_last_error().decode()
    if text == "launch":  # a first call may ask for workspace; without a GPU the device's selection fails first
        if rc > 0:
            rc = getattr(lib, name)(*{**args, "ws": P, "wsb": rc}.values())
        assert rc in (-1, -2)
    else:
        assert rc == -1 and text in err and name in err, (rc, err)


@pytest.mark.parametrize("name, base, change", [
    ("bgp_grouped_gemm", GEMM, dict(T=0)), ("bgp_grouped_gemm", GEMM, dict(N=0, ldy=0)), ("bgp_grouped_gemm_dw", DW, dict(G=0, off=None)),
    ("bgp_quantize_rows", QUANT, dict(M=0)), ("bgp_int8_gemm", INT8, dict(M=0)), ("bgp_int8_gemm", INT8, dict(N=0)),
])
def test_nothing_to_do_is_no_error(name, base, change):
    assert getattr(_lib.load_products(), name)(*{**base, **change}.values()) == 0


MANY = 1 << 40


@pytest.mark.parametrize("name, base, change", [
    ("bgp_grouped_gemm", GEMM, dict(T=MANY)),
    ("bgp_grouped_gemm", GEMM, dict(T=MANY, X=C.c_void_p(4098), ldx=5)),  # operands that would be copied first
    ("bgp_grouped_gemm", GEMM, dict(N=MANY, ldy=MANY, sW=4 * MANY)),
    ("bgp_grouped_gemm_dw", DW, dict(N=1 << 20, K=1 << 20, lddy=1 << 20, ldx=1 << 20, ldw=1 << 20, sW=MANY)),
    ("bgp_grouped_gemm_dw", DW, dict(G=65535, N=1 << 12, K=1 << 12, lddy=1 << 12, ldx=1 << 12, ldw=1 << 12, sW=1 << 24)),
    ("bgp_int8_gemm", INT8, dict(M=MANY)),
    ("bgp_int8_gemm", INT8, dict(M=MANY, N=MANY, ldy=MANY)),
])
def test_more_tiles_than_a_launch_holds_are_refused_before_anything_is_enqueued(name, base, change):
    lib = _lib.load_products()
    assert getattr(lib, name)(*{**base, **change}.values()) == -1
    assert "launch" in lib.bgp_products_last_error().decode()


def test_many_tiles_that_a_launch_holds_are_taken():
    """2e8 rows of 16 numbers to 16: too many tiles of 16 rows, which the sizes would ask for, but not of 64 or 128"""
    lib = _lib.load_products()
    rc = lib.bgp_grouped_gemm(*{**GEMM, "T": 200_000_000, "N": 16, "K": 16, "ldx": 16, "ldw": 16, "ldy": 16, "sW": 256, "device": 4095}.values())
    assert rc == -2  # it got as far as the device


@pytest.mark.parametrize("name, base, change", [
    # operands off the 16-byte chunks and long enough to be copied
    ("bgp_grouped_gemm", GEMM, dict(dtype=2, T=8192, N=2049, K=2049, X=C.c_void_p(4098), ldx=2049, ldw=2049, sW=2049 * 2049, ldy=2049)),
    ("bgp_int8_gemm", INT8, dict(M=4097, N=4097, K=4097, A=C.c_void_p(4097), lda=4097, ldb=4097, ldy=4097)),
])
def test_workspaces_off_their_alignment_are_refused(name, base, change):
    lib = _lib.load_products()
    args = {**base, **change}
    need = getattr(lib, name)(*args.values())
    assert need > 0 and getattr(lib, name)(*{**args, "ws": P, "wsb": need - 1}.values()) == need
    assert getattr(lib, name)(*{**args, "ws": C.c_void_p(4104), "wsb": need}.values()) == -1
    assert "workspace" in lib.bgp_products_last_error().decode()


def test_added_in_place_with_another_leading_dimension_is_refused():
    lib = _lib.load_products()
    assert lib.bgp_int8_gemm(*{**INT8, "C": P, "ldc": 5}.values()) == -1
    assert "strides" in lib.bgp_products_last_error().decode()


@pytest.mark.parametrize("call", [
    lambda t: products.grouped_matmul(t, torch.ones(1, 4, 3), torch.tensor([0, 6])),
    lambda t: products.quantize_rows(t),
])
def test_lazily_negated_tensors_are_refused(recorder, call):
    """the imaginary part of a conjugate: its memory holds the opposite of its values"""
    t = torch.complex(torch.ones(6, 3), torch.ones(6, 3)).conj().imag
    assert t.is_neg()
    with pytest.raises(ValueError, match="own values"):
        call(t)
    assert not recorder.calls


class Recorder:
    """Stands for the library on the CPU: keeps the last call's arguments by the header's names."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        keys = {"bgp_grouped_gemm": GEMM, "bgp_grouped_gemm_dw": DW, "bgp_quantize_rows": QUANT, "bgp_int8_gemm": INT8}[name]

        def call(*args):
            assert len(args) == len(keys)
            self.calls.append((name, dict(zip(keys, args))))
            return 0

        return call


@pytest.fixture
def recorder(monkeypatch):
    rec = Recorder()
    monkeypatch.setattr(products, "FIRST_DEVICE", -1)
    monkeypatch.setattr(products, "_stream", lambda device: None)
    monkeypatch.setattr(_lib, "load_products", lambda: rec)
    return rec


def test_cpu_tensors_are_refused():
    x, w, o = torch.ones(2, 3), torch.ones(1, 4, 3), torch.tensor([0, 2])
    with pytest.raises(EngineError, match="MI355X only"):
        products.grouped_matmul(x, w, o)
    with pytest.raises(EngineError, match="MI355X only"):
        products.quantize_rows(x)


def _case(t=6, n=4, k=3, g=2, dtype=torch.float32):
    return torch.ones(t, k, dtype=dtype), torch.ones(g, n, k, dtype=dtype), torch.tensor([0] + [t] * g)


@pytest.mark.parametrize("change, error, text", [
    (lambda x, w, o: (x.numpy(), w, o), TypeError, "x is not"),
    (lambda x, w, o: (x[0], w, o), ValueError, "x has 1 dim"),
    (lambda x, w, o: (x, w[0], o), ValueError, "w has 2 dim"),
    (lambda x, w, o: (x.int(), w, o), ValueError, "not one of"),
    (lambda x, w, o: (x, w.double(), o), ValueError, "float64"),
    (lambda x, w, o: (x[:, :2], w, o), ValueError, "columns"),
    (lambda x, w, o: (torch.ones(3, 6).t(), w, o), ValueError, "contiguous"),
    (lambda x, w, o: (torch.ones(1, 3).expand(6, 3), w, o), ValueError, "overlap"),
    (lambda x, w, o: (x, torch.ones(2, 8, 6)[:, ::2, ::2], o), ValueError, "either axis"),
    (lambda x, w, o: (x, torch.ones(2, 1, 3).expand(2, 4, 3), o), ValueError, "either axis"),
    (lambda x, w, o: (x, w, o.int()), ValueError, "int64"),
    (lambda x, w, o: (x, w, o[:2]), ValueError, "3 are wanted"),
    (lambda x, w, o: (x, w, torch.zeros(6, dtype=torch.int64)[::2]), ValueError, "not contiguous"),
    (lambda x, w, o: (x.requires_grad_(), w, o), ValueError, "autograd"),
    (lambda x, w, o: (x.to_sparse(), w, o), ValueError, "dense"),
])
def test_grouped_matmul_refuses(recorder, change, error, text):
    with pytest.raises(error, match=text):
        products.grouped_matmul(*change(*_case()))
    assert not recorder.calls


def test_grouped_matmul_refuses_outputs(recorder):
    x, w, o = _case(n=3)
    for bad in (torch.empty(6, 4), torch.empty(5, 3), torch.empty(6, 3, dtype=torch.float64), torch.empty(3, 6).t()):
        with pytest.raises(ValueError):
            products.grouped_matmul(x, w, o, out=bad)
    with pytest.raises(ValueError, match="overlaps"):
        products.grouped_matmul(x, w, o, out=x)
    with pytest.raises(ValueError, match="overlaps"):
        products.grouped_matmul(x, torch.ones(2, 3, 3), o, out=x)
    with pytest.raises(ValueError, match="dy"):
        products.grouped_matmul_grad(torch.ones(6, 5), x, w, o)
    assert not recorder.calls


def test_grouped_matmul_arguments(recorder):
    x = torch.ones(6, 8)[:, :3]
    w, o = torch.ones(2, 4, 3), torch.tensor([0, 2, 6])
    y = products.grouped_matmul(x, w, o)
    name, a = recorder.calls[-1]
    assert y.shape == (6, 4) and (a["T"], a["N"], a["K"], a["G"]) == (6, 4, 3, 2)
    assert (a["ldx"], a["sW"], a["ldw"], a["trans"], a["ldy"], a["zero"]) == (8, 12, 3, 0, 4, 1)
    out = torch.empty(6, 10)[:, 2:6]
    assert products.grouped_matmul(x, torch.ones(2, 3, 4).transpose(1, 2), o, out=out) is out
    a = recorder.calls[-1][1]
    assert (a["sW"], a["ldw"], a["trans"], a["ldy"], a["zero"]) == (12, 4, 1, 10, 0)
    products.grouped_matmul(x, w[:1].expand(2, 4, 3), o)
    assert recorder.calls[-1][1]["sW"] == 0
    # one row, one column, one output: the stride of such an axis says nothing
    products.grouped_matmul(torch.as_strided(torch.ones(9), (1, 3), (1, 1)), w, o)
    assert recorder.calls.pop()[1]["ldx"] == 3
    products.grouped_matmul(torch.ones(6, 1), torch.ones(2, 4, 1), o)
    products.grouped_matmul(torch.ones(0, 3), w, o)
    products.grouped_matmul(torch.ones(4, 3), torch.ones(0, 4, 3), torch.zeros(1, dtype=torch.int64))
    assert recorder.calls[-1][1]["G"] == 0


def test_grouped_matmul_grad_arguments(recorder):
    x, w, o = _case()
    dy = torch.ones(6, 4)
    dx, dw = products.grouped_matmul_grad(dy, x, w, o)
    (n1, a), (n2, b) = recorder.calls
    # dX is the product of dY with the weights read along their other axis
    assert n1 == "bgp_grouped_gemm" and (a["N"], a["K"], a["trans"], a["ldw"], a["X"]) == (3, 4, 1, 3, dy.data_ptr())
    assert n2 == "bgp_grouped_gemm_dw" and (b["N"], b["K"], b["sW"], b["ldw"]) == (4, 3, 12, 3)
    assert dx.shape == x.shape and dw.shape == w.shape and dw.is_contiguous()
    assert products.grouped_matmul_grad(dy, x, w, o, need_dx=False)[0] is None
    assert products.grouped_matmul_grad(dy, x, w, o, need_dw=False)[1] is None
    products.grouped_matmul_grad(dy, x, torch.ones(2, 3, 4).transpose(1, 2), o, need_dw=False)
    assert recorder.calls[-1][1]["trans"] == 0


def test_int8_functions_refuse_and_pass_on(recorder):
    a, b = torch.ones(4, 8, dtype=torch.int8), torch.ones(5, 8, dtype=torch.int8)
    sa, sb = torch.ones(4), torch.ones(5)
    for args, text in (
        ((a.float(), b, sa, sb), "int8"), ((a, b[:, :7], sa, sb), "columns"), ((a, b, sa.double(), sb), "a_scale"), ((a, b, sa, sb[:4]), "b_scale"),
        ((a, b, sa, torch.ones(10)[::2]), "b_scale"), ((a, b, sa[:, None], sb), "dimensions"), ((a, b, sa, sb, torch.ones(4, 5)), "c:"),
        ((torch.ones(1, 131072, dtype=torch.int8), torch.ones(5, 131072, dtype=torch.int8), sa[:1], sb), "32 bits"),
    ):
        with pytest.raises(ValueError, match=text):
            products.int8_matmul(*args)
    with pytest.raises(ValueError, match="int32"):
        products.int8_matmul(a, b, sa, sb, dtype=torch.int32)
    with pytest.raises(ValueError, match="a_scale"):  # fp64 results take fp64 scales
        products.int8_matmul(a, b, sa, sb, dtype=torch.float64)
    c = torch.zeros(5, 6)[:4, :5]
    with pytest.raises(ValueError, match="overlaps"):  # neither c itself nor apart from it
        products.int8_matmul(a, b, sa, sb, c=c, dtype=torch.float32, out=torch.as_strided(c, (4, 5), (6, 1), 1))
    assert not recorder.calls
    assert products.int8_matmul(a, b, sa, sb).dtype == torch.bfloat16
    assert products.int8_matmul(a, b, sa, sb, c=c, dtype=torch.float32, out=c) is c
    call = recorder.calls[-1][1]
    assert call["C"] == call["Y"] == c.data_ptr() and call["ldc"] == call["ldy"] == 6
    with pytest.raises(ValueError, match="not one of"):
        products.quantize_rows(a)
    q, s = products.quantize_rows(torch.ones(4, 9)[:, :8])
    assert q.dtype == torch.int8 and s.dtype == torch.float32 and recorder.calls[-1][1]["ldx"] == 9 and recorder.calls[-1][1]["rest"] is None
    q, s, r = products.quantize_rows(torch.ones(4, 8, dtype=torch.float64), pow2=True, residual=True)
    assert s.dtype == r.dtype == torch.float64 and recorder.calls[-1][1]["pow2"] == 1


# ---- calls without groups ----


@pytest.mark.parametrize("dtype, t, n, k", [(_lib.BF16, 8192, 2049, 2049), (_lib.F16, 4096, 4096, 4001), (_lib.F32, 3001, 2999, 2001), (_lib.F64, 2700, 1000, 1001)])
@pytest.mark.parametrize("trans", [0, 1])
@pytest.mark.parametrize("x", [None, C.c_void_p(4096 + 8)])
def test_without_groups_no_operand_is_copied(dtype, t, n, k, trans, x):
    """an empty tensor's pointer is NULL: of rows and weights off the 16-byte chunks nothing may be read for aligned copies"""
    lib = _lib.load_products()
    args = {**GEMM, "device": 4095, "dtype": dtype, "T": t, "N": n, "K": k, "G": 0, "X": x, "ldx": k, "W": None, "sW": 0, "ldw": n if trans else k, "trans": trans,
            "ldy": n}
    assert lib.bgp_grouped_gemm(*args.values()) == -2  # no workspace is asked for: it got as far as the device
    assert lib.bgp_grouped_gemm(*{**args, "ws": P, "wsb": 1 << 40}.values()) == -2
    assert lib.bgp_grouped_gemm(*{**args, "zero": 0}.values()) == 0  # nothing to do at all


# ---- outputs that are given ----


def _given_outputs():
    x, w, o = _case(n=3)
    a, sa = torch.ones(4, 8, dtype=torch.int8), torch.ones(4)
    yield torch.zeros(6, 3), lambda out: products.grouped_matmul(x, w, o, out=out)
    yield torch.zeros(4, 4), lambda out: products.int8_matmul(a, a, sa, sa, dtype=torch.float32, out=out)
    yield torch.zeros(4, 4), lambda out: products.int8_matmul(a, a, sa, sa, c=out, dtype=torch.float32, out=out)


@pytest.mark.parametrize("case", range(3))
def test_autograd_notices_a_given_output(recorder, case):
    """what was saved for a backward pass and is then written over raises there, as after torch's own operations in place"""
    out, call = list(_given_outputs())[case]
    p = torch.ones_like(out).requires_grad_()
    z = p * out  # keeps out for p's gradient
    assert call(out) is out and recorder.calls
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.sum().backward()
    (p * out).sum().backward()
    view = out.view(-1)
    call(out)
    assert view._version == out._version == 2
    with torch.inference_mode():  # keeps no versions
        fresh = torch.zeros_like(out)
        assert call(fresh) is fresh
    wrong = torch.zeros(1, 1)
    with pytest.raises(ValueError):
        call(wrong)
    assert wrong._version == 0


# ---- tensors that stand for something else than the numbers in their memory ----


class Wrapped(torch.Tensor):
    """a wrapper without memory of its own"""

    @staticmethod
    def __new__(cls, inner):
        return torch.Tensor._make_wrapper_subclass(cls, inner.shape, dtype=inner.dtype, device=inner.device)

    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        raise NotImplementedError


def _operands():
    """every call with its floating point operands"""
    x, w, o = _case(n=3)
    yield lambda x, w: products.grouped_matmul(x, w, o), (x, w)
    yield lambda x, w, out: products.grouped_matmul(x, w, o, out=out), (x, w, torch.zeros(6, 3))
    yield lambda dy, x, w: products.grouped_matmul_grad(dy, x, w, o), (torch.ones(6, 3), x, w)
    yield lambda x: products.quantize_rows(x), (x,)
    a = torch.ones(6, 3, dtype=torch.int8)
    yield lambda sa, sb, c: products.int8_matmul(a, a, sa, sb, c=c, dtype=torch.float32), (torch.ones(6), torch.ones(6), torch.zeros(6, 6))


CALLS = [(i, j) for i, (_, operands) in enumerate(_operands()) for j in range(len(operands))]


@pytest.mark.parametrize("i, j", CALLS)
def test_operands_with_tangents_are_refused(recorder, i, j):
    import torch.autograd.forward_ad as fw

    call, operands = list(_operands())[i]
    with fw.dual_level():
        dual = fw.make_dual(operands[j], torch.ones_like(operands[j]))
        with pytest.raises(ValueError, match="tangent"):
            call(*operands[:j], dual, *operands[j + 1:])
        with torch.no_grad(), pytest.raises(ValueError, match="tangent"):  # does not turn forward mode off
            call(*operands[:j], dual, *operands[j + 1:])
        assert not recorder.calls
        call(*operands)
    assert recorder.calls


@pytest.mark.parametrize("i, j", CALLS)
def test_operands_without_memory_are_refused(recorder, i, j):
    call, operands = list(_operands())[i]

    def with_one(t):
        return call(*operands[:j], t, *operands[j + 1:])

    with pytest.raises(ValueError, match="own values"):
        with_one(Wrapped(operands[j]))
    with pytest.raises(ValueError, match="own values"):
        torch.func.vmap(with_one)(operands[j][None])
    with pytest.raises(ValueError, match="own values|tangent"):
        torch.func.jvp(with_one, (operands[j],), (operands[j],))
    with pytest.raises(ValueError, match="gradient"):
        torch.func.grad(lambda t: with_one(t)[0].sum())(operands[j])
    assert not recorder.calls


@pytest.mark.parametrize("m, ldr, fits", [(4, 9, False), (4, 8, True), (1, 9, True)])
def test_rest_in_place_with_another_leading_dimension_is_refused(m, ldr, fits):
    """a row of the rest would lie over rows of x that are still to be read; with one row there is no other"""
    lib = _lib.load_products()
    rc = lib.bgp_quantize_rows(*{**QUANT, "device": 4095, "M": m, "rest": P, "ldr": ldr}.values())
    assert rc == (-2 if fits else -1)  # -2: it got as far as the device
    if not fits:
        assert "strides" in lib.bgp_products_last_error().decode()
    assert lib.bgp_quantize_rows(*{**QUANT, "device": 4095, "M": m, "K": 0, "x": None, "q": None, "ldr": ldr}.values()) == -2  # no rest, and nothing to read


def test_outputs_that_are_no_tensors_are_refused_as_such(recorder):
    a, s, c = torch.ones(4, 8, dtype=torch.int8), torch.ones(4), torch.zeros(4, 4)
    for bad in (c.numpy(), [0.0]):
        with pytest.raises(TypeError, match="out is not a torch tensor"):
            products.int8_matmul(a, a, s, s, c=c, dtype=torch.float32, out=bad)
        with pytest.raises(TypeError, match="out is not a torch tensor"):
            products.int8_matmul(a, a, s, s, dtype=torch.float32, out=bad)
    with pytest.raises(ValueError, match="own values"):  # nor one that has no memory
        products.int8_matmul(a, a, s, s, c=c, dtype=torch.float32, out=Wrapped(c))
    assert not recorder.calls


def test_outputs_between_the_columns_of_an_input(recorder):
    """columns of one wide matrix are apart, though each reaches over the other's rows"""
    buf, o = torch.zeros(6, 12), torch.tensor([0, 2, 6])
    x, w = buf[:, 2:5], torch.ones(2, 4, 3)
    for at in (5, 8):
        out = buf[:, at:at + 4]
        assert products.grouped_matmul(x, w, o, out=out) is out
    out = torch.as_strided(buf, (5, 4), (12, 1), 10)  # the last two columns and the next row's first two
    assert products.grouped_matmul(buf[:5, 2:5], w, o, out=out) is out
    assert len(recorder.calls) == 3
    for bad in (buf[:, 1:5], buf[:, 4:8], torch.as_strided(buf, (5, 4), (12, 1), 11), torch.as_strided(buf, (6, 4), (11, 1), 5)):
        t = bad.shape[0]
        with pytest.raises(ValueError, match="overlaps"):
            products.grouped_matmul(x[:t], w, o, out=bad)
    # weights between the columns of the output, in either order of their axes; scales in its last one
    big = torch.zeros(24, 12)
    out = big[:6, :4]
    assert products.grouped_matmul(torch.ones(6, 3), torch.as_strided(big, (2, 4, 3), (48, 12, 1), 4), o, out=out) is out
    assert products.grouped_matmul(torch.ones(6, 3), torch.as_strided(big, (2, 4, 3), (36, 1, 12), 4), o, out=out) is out
    with pytest.raises(ValueError, match="overlaps"):
        products.grouped_matmul(torch.ones(6, 3), torch.as_strided(big, (2, 4, 3), (48, 12, 1), 3), o, out=out)
    with pytest.raises(ValueError, match="overlaps"):
        products.grouped_matmul(torch.ones(6, 3), torch.as_strided(big, (2, 4, 3), (50, 12, 1), 4), o, out=out)
    a = torch.ones(6, 8, dtype=torch.int8)
    assert products.int8_matmul(a, a[:4], torch.ones(6), big[0, 4:8], dtype=torch.float32, out=out) is out
    with pytest.raises(ValueError, match="overlaps"):
        products.int8_matmul(a, a[:4], torch.ones(6), big[0, 3:7], dtype=torch.float32, out=out)
    one = torch.zeros(24)  # a single row, whose stride says nothing
    for stride in (0, 2, 24):
        out = torch.as_strided(one, (1, 4), (stride, 1))
        with pytest.raises(ValueError, match="overlaps"):
            products.grouped_matmul(one[None, 3:6], w, o, out=out)
        assert products.grouped_matmul(one[None, 4:7], w, o, out=out) is out
    with pytest.raises(ValueError, match="overlaps"):  # both axes of the weights next to each other
        products.grouped_matmul(torch.ones(6, 3), torch.as_strided(big, (2, 4, 3), (48, 12, 1), 4)[:, :, :], o, out=big[:6, 1:5])


def test_the_libraries_are_built_without_torch(monkeypatch, tmp_path, capsys):
    """a program that calls the C entries needs hipcc only; the compiled calls from torch tensors are left out, in words"""
    import sys

    from battgp_amd import build

    made = []
    monkeypatch.setattr(build, "_compile", lambda folder, sources, flags, suffix, lib, verbose: made.append(lib))
    monkeypatch.setattr(build, "LIB_TORCH_CALLS", str(tmp_path / "calls.so"))
    monkeypatch.setattr(build.subprocess, "check_call", lambda cmd: pytest.fail("nothing to compile against"))
    monkeypatch.setitem(sys.modules, "torch", None)
    assert build.build_products(force=True, verbose=False) == build.LIB_PRODUCTS and made == [build.LIB_PRODUCTS]
    assert "torch" in capsys.readouterr().err
