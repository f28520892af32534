"""Every way through the products' library that the model chooses (tests/products_plans.py), on the GPU: whole numbers within
+-2, whose sums every accumulator holds exactly (4 * 20000 < 2^24), compared for equality with the sum in 64 bits rounded once."""

import pytest
import torch
from products_plans import DW, INT8, ROWS, ROWS_TURNED, counts

pytestmark = [pytest.mark.gpu, pytest.mark.gpu_sized]  # matrix instructions that the CPU build of the sources does not have

TYPES = {2: (torch.bfloat16, torch.float16), 4: (torch.float32,), 8: (torch.float64,)}


@pytest.fixture(scope="module")
def products():
    from battgp_amd import products

    return products


def whole(shape, seed, dtype):
    return torch.randint(-2, 3, shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)).to(dtype)


def bounds(t, g):
    off = [0]
    for c in counts(t, g):
        off.append(off[-1] + c)
    return off


def rounded(ref, dtype):
    return ref.float().to(dtype) if dtype == torch.float16 else ref.to(dtype)  # sums past 65504 are infinities


def name(case):
    return "-".join(str(v) for v in case)


@pytest.mark.parametrize("case", ROWS, ids=name)
def test_rows(products, case):
    check_rows(products, case, False)


@pytest.mark.parametrize("case", ROWS_TURNED, ids=name)
def test_rows_against_turned_weights(products, case):
    check_rows(products, case, True)


def check_rows(products, case, turned):
    size, t, n, k, g = case[:5]
    off = bounds(t, g)
    for dtype in TYPES[size]:
        x, w = whole((t, k), 1, dtype), whole((g, k, n) if turned else (g, n, k), 2, dtype)
        w = w.transpose(1, 2) if turned else w
        y = products.grouped_matmul(x, w, torch.tensor(off, device="cuda"))
        for i, (a, b) in enumerate(zip(off, off[1:])):
            assert torch.equal(y[a:b], rounded(x[a:b].double() @ w[i].double().T, dtype)), (dtype, i)


@pytest.mark.parametrize("case", DW, ids=name)
def test_weight_gradients(products, case):
    size, t, n, k, g = case[:5]
    off = bounds(t, g)
    for dtype in TYPES[size]:
        dy, x = whole((t, n), 1, dtype), whole((t, k), 2, dtype)
        w = torch.empty((1, n, k), dtype=dtype, device="cuda").expand(g, n, k)  # its values do not matter
        _, dw = products.grouped_matmul_grad(dy, x, w, torch.tensor(off, device="cuda"), need_dx=False)
        for i, (a, b) in enumerate(zip(off, off[1:])):
            assert torch.equal(dw[i], rounded(dy[a:b].double().T @ x[a:b].double(), dtype)), (dtype, i)


@pytest.mark.parametrize("case", INT8, ids=name)
def test_8_bit_products(products, case):
    out_bytes, m, n, k = case[:4]
    dtype = {2: torch.bfloat16, 4: torch.float32, 8: torch.float64, 16: torch.float64}[out_bytes]
    gen = torch.Generator(device="cuda").manual_seed(3)
    a, b = (torch.randint(-128, 128, s, device="cuda", generator=gen, dtype=torch.int8) for s in ((m, k), (n, k)))
    one = torch.ones(max(m, n), device="cuda", dtype=torch.float64 if dtype == torch.float64 else torch.float32)
    c = whole((m, n), 4, dtype) if out_bytes == 16 else None
    y = products.int8_matmul(a, b, one[:m], one[:n], c=c, dtype=dtype)
    ref = a.double() @ b.double().T  # below 2^31: exact
    ref = ref if c is None else ref + c
    half = 0.0 if dtype == torch.float64 else torch.finfo(dtype).eps / 2
    assert ((y.double() - ref).abs() <= half * ref.abs()).all()
