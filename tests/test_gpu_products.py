"""GPU tests of the grouped and 8-bit products (battgp_amd/products.py) against their formulas in 64 bits on the CPU.

Most cases take small whole numbers, whose products and sums every type's accumulator holds exactly (|x|, |w| <= 4:
|sum| <= 16 K < 2^24): the result is the exact sum rounded once to the output's type, and is compared for equality.
Cases with ordinary numbers allow for the rounding of each of the K additions in fp32 (K 2^-23 of the sum of the products'
magnitudes: whole steps, since the matrix unit's inner order and rounding are its own) and half a step of the output's
type; fp64 likewise with 2^-52."""

import numpy as np
import pytest
import torch

pytestmark = [pytest.mark.gpu, pytest.mark.gpu_sized]  # matrix instructions that the CPU build of the sources does not have

ALL = [torch.float64, torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def products():
    from battgp_amd import products

    return products


def whole(shape, seed, most=4, dtype=torch.float64):
    return torch.randint(-most, most + 1, shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def guarded(shape, dtype, pad=3):
    """A view of `shape` with a rim of 7s around it, and a check that the rim is whole."""
    buf = torch.full((shape[0] + 2, shape[1] + 2 * pad), 7.0, dtype=dtype, device="cuda")
    view = buf[1:-1, pad:pad + shape[1]]

    def check():
        seen = buf.clone()
        seen[1:-1, pad:pad + shape[1]] = 7.0
        assert (seen == 7.0).all(), "written outside the output"

    return view, check


def rows_of(offsets):
    return [(int(a), int(b)) for a, b in zip(offsets, offsets[1:])]


def grouped_ref(x, w, offsets, y=None):
    y = torch.zeros(x.shape[0], w.shape[1], dtype=torch.float64) if y is None else y
    for g, (a, b) in enumerate(rows_of(offsets)):
        y[a:b] = x[a:b] @ w[g].T
    return y


SHAPES = [  # offsets, rows in all, n, k
    ([0, 1], 1, 1, 1),
    ([0, 1], 1, 130, 70),
    ([0, 3, 3, 3, 8], 8, 64, 64),
    ([0, 0, 0], 0, 8, 8),
    ([0, 0, 5], 5, 33, 0),
    ([2, 130, 130, 259, 260], 263, 257, 129),
    ([0, 128, 256], 256, 128, 128),
    ([0, 127, 254, 511], 511, 256, 192),
    ([0] * 70 + [200], 200, 72, 40),
    (list(range(0, 141, 2)), 150, 16, 513),
    ([0, 300, 600, 900], 900, 100, 100),
    ([0, 700], 700, 300, 24),
]


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("wt", [False, True])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"T{s[1]}G{len(s[0]) - 1}n{s[2]}k{s[3]}")
def test_grouped_matmul_is_the_rounded_exact_sum(products, dtype, wt, shape):
    off, t, n, k = shape
    g = len(off) - 1
    x, w = whole((t, k), 1), whole((g, n, k), 2)
    ref = grouped_ref(x, w, off).to(dtype)
    xd, od = x.to(dtype).cuda(), torch.tensor(off, device="cuda")
    wd = w.transpose(1, 2).contiguous().to(dtype).cuda().transpose(1, 2) if wt else w.to(dtype).cuda()
    y = products.grouped_matmul(xd, wd, od)
    assert y.dtype == dtype and torch.equal(y.cpu(), ref)
    # a given output keeps the rows of no group, and nothing around it is touched
    out, rim = guarded((t, n), dtype)
    out.fill_(5.0)
    assert products.grouped_matmul(xd, wd, od, out=out) is out
    kept = torch.full((t, n), 5.0, dtype=torch.float64)
    assert torch.equal(out.cpu(), grouped_ref(x, w, off, kept).to(dtype))
    rim()


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("wt", [False, True])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"T{s[1]}G{len(s[0]) - 1}n{s[2]}k{s[3]}")
def test_grouped_matmul_grad_is_the_rounded_exact_sum(products, dtype, wt, shape):
    off, t, n, k = shape
    g = len(off) - 1
    x, w, dy = whole((t, k), 3), whole((g, n, k), 4), whole((t, n), 5)
    dx_ref = grouped_ref(dy, w.transpose(1, 2), off)
    dw_ref = torch.stack([dy[a:b].T @ x[a:b] for a, b in rows_of(off)]) if g else torch.zeros(0, n, k)
    wd = w.transpose(1, 2).contiguous().to(dtype).cuda().transpose(1, 2) if wt else w.to(dtype).cuda()
    dx, dw = products.grouped_matmul_grad(dy.to(dtype).cuda(), x.to(dtype).cuda(), wd, torch.tensor(off, device="cuda"))
    assert torch.equal(dx.cpu(), dx_ref.to(dtype))
    assert torch.equal(dw.cpu(), dw_ref.to(dtype))


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("t, n, k, g", [(517, 200, 304, 4), (40, 130, 250, 3), (6, 520, 1000, 5)])
def test_ordinary_numbers(products, dtype, t, n, k, g):
    gen = torch.Generator().manual_seed(t)
    x, w, dy = (torch.randn(*s, generator=gen, dtype=torch.float64).to(dtype) for s in ((t, k), (g, n, k), (t, n)))
    off = [0] + sorted(torch.randint(0, t + 1, (g - 1,), generator=gen).tolist()) + [t]
    xd, wd, dyd, od = x.cuda(), w.cuda(), dy.cuda(), torch.tensor(off, device="cuda")
    step = 2.0 ** -52 if dtype == torch.float64 else 2.0 ** -23
    half = 0.0 if dtype == torch.float64 else torch.finfo(dtype).eps / 2
    # below the smallest normal number the step stops shrinking with the value: fp16 has steps of 2^-24 below 2^-14, so a
    # rounding there is off by up to 2^-25 whatever the value is
    least = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
    x, w, dy = x.double(), w.double(), dy.double()

    def near(got, ref, mags, terms):
        # half a step of the sum as rounded; the sums' own error moves it by at most as much again
        bound = terms * step * mags
        assert ((got.cpu().double() - ref).abs() <= bound + half * (ref.abs() + bound) + least).all()

    near(products.grouped_matmul(xd, wd, od), grouped_ref(x, w, off), grouped_ref(x.abs(), w.abs(), off), k)
    dx, dw = products.grouped_matmul_grad(dyd, xd, wd, od)
    wt = w.transpose(1, 2)
    near(dx, grouped_ref(dy, wt, off), grouped_ref(dy.abs(), wt.abs(), off), n)
    for i, (a, b) in enumerate(rows_of(off)):
        near(dw[i], dy[a:b].T @ x[a:b], dy[a:b].abs().T @ x[a:b].abs(), max(b - a, 1))


def test_gradients_against_differences(products):
    gen = torch.Generator(device="cuda").manual_seed(3)
    x, w, dy = (torch.randn(*s, generator=gen, device="cuda", dtype=torch.float64) for s in ((50, 20), (3, 30, 20), (50, 30)))
    off = torch.tensor([0, 17, 17, 50], device="cuda")
    dx, dw = products.grouped_matmul_grad(dy, x, w, off)
    for _ in range(3):
        px, pw = (torch.randn(t.shape, generator=gen, device="cuda", dtype=torch.float64) for t in (x, w))
        h = 0.5  # the product is bilinear: the central difference has no error of its own along one operand
        fx = ((products.grouped_matmul(x + h * px, w, off) - products.grouped_matmul(x - h * px, w, off)) * dy).sum() / (2 * h)
        fw = ((products.grouped_matmul(x, w + h * pw, off) - products.grouped_matmul(x, w - h * pw, off)) * dy).sum() / (2 * h)
        # sums of 50 * 30 * 20 products of size 1 at 2^-53 each, twice
        assert abs(fx - (dx * px).sum()) < 1e-9 and abs(fw - (dw * pw).sum()) < 1e-9


@pytest.mark.parametrize("dtype", ALL)
def test_rows_and_weights_of_others_do_not_leak(products, dtype):
    """NaN in rows of no group, in another group's rows, in an unused group's weights and behind the last column."""
    off, t, n, k = [1, 40, 40, 77], 80, 70, 50
    x, w, dy = whole((t, k + 6), 1), whole((3, n, k + 6), 2), whole((t, n + 6), 3)
    for m in (x, w):
        m[..., k:] = float("nan")
    dy[:, n:] = float("nan")
    for m in (x, dy):
        m[0] = m[77:] = float("nan")
    w[1] = float("nan")
    xs, ws, dys = (m.to(dtype).cuda() for m in (x, w, dy))
    xs, ws, dys, od = xs[:, :k], ws[:, :, :k], dys[:, :n], torch.tensor(off, device="cuda")
    x, w, dy = x[:, :k], w[:, :, :k], dy[:, :n]
    assert torch.equal(products.grouped_matmul(xs, ws, od).cpu(), grouped_ref(x, w, off).to(dtype))
    dx, dw = products.grouped_matmul_grad(dys, xs, ws, od)
    assert torch.equal(dx.cpu(), grouped_ref(dy, w.transpose(1, 2), off).to(dtype))
    assert torch.equal(dw.cpu(), torch.stack([dy[a:b].T @ x[a:b] for a, b in rows_of(off)]).to(dtype))
    xs[45] = float("nan")  # a row of the last group: its own row of y and its group's dw
    y = products.grouped_matmul(xs, ws, od)
    assert y[45].isnan().all() and not y[torch.arange(t) != 45].isnan().any()


def test_shared_weights_and_offsets_out_of_range(products):
    x, w = whole((90, 24), 1), whole((1, 40, 24), 2)
    xd, wd = x.cuda(), w.cuda().expand(3, 40, 24)
    y = products.grouped_matmul(xd, wd, torch.tensor([0, 20, 21, 90], device="cuda"))
    assert torch.equal(y.cpu(), x @ w[0].T)
    # offsets are clamped into the matrix
    wrong = torch.tensor([-5, 20, 2 ** 40, 2 ** 62], device="cuda")
    out, rim = guarded((90, 40), torch.float64)
    products.grouped_matmul(xd, wd, wrong, out=out)
    assert torch.equal(out.cpu(), x @ w[0].T)
    rim()
    dx, dw = products.grouped_matmul_grad(out, xd, wd, wrong)
    assert torch.equal(dw[2].cpu(), torch.zeros(40, 24, dtype=torch.float64))


def test_many_groups(products):
    g = 3000
    counts = torch.randint(0, 4, (g,), generator=torch.Generator().manual_seed(1))
    off = torch.cat((torch.zeros(1, dtype=torch.int64), counts.cumsum(0)))
    t = int(off[-1])
    x, w = whole((t, 32), 1), whole((g, 48, 32), 2)
    y = products.grouped_matmul(x.float().cuda(), w.float().cuda(), off.cuda())
    dx, dw = products.grouped_matmul_grad(y, x.float().cuda(), w.float().cuda(), off.cuda())
    group = torch.repeat_interleave(torch.arange(g), counts)
    ref = torch.bmm(w[group], x[:, :, None])[:, :, 0]
    assert torch.equal(y.cpu().double(), ref)
    dwr = torch.zeros(g, 48, 32, dtype=torch.float64).index_add_(0, group, ref[:, :, None] * x[:, None, :])
    assert torch.equal(dw.cpu().double(), dwr)  # |sums| <= 3 * 512 * 4: whole numbers below 2^24


# ---- 8-bit integers ----

def quantize_ref(x, pow2):
    """The definition, in numpy's 64 bits."""
    v = x.double().numpy()
    top = np.abs(v).max(axis=1) if v.shape[1] else np.zeros(v.shape[0])
    stype = np.float64 if x.dtype == torch.float64 else np.float32
    if pow2:
        scale = np.zeros(v.shape[0])
        for i, m in enumerate(top):
            p = -1080
            while m > 0 and np.isfinite(m) and p < 1018 and m > np.ldexp(127.0, p):  # 127 * 2^1018 is past the largest number
                p += 1
            scale[i] = np.ldexp(1.0, p) if m > 0 else 0.0
    else:
        scale = (top / 127.0).astype(stype).astype(np.float64)
    bad = ~np.isfinite(top)
    scale = np.where(bad, top, np.maximum(scale, np.finfo(stype).tiny))
    with np.errstate(all="ignore"):
        q = np.where(bad[:, None], 0.0, np.clip(np.rint(v / scale[:, None]), -127, 127))
        rest = v - q * scale[:, None]
    return q.astype(np.int8), scale.astype(stype), rest


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("pow2", [False, True])
@pytest.mark.parametrize("m, k, pad", [(1, 1, 0), (3, 8, 0), (5, 127, 0), (7, 1000, 3), (130, 257, 0), (2, 8192, 0), (2, 20011, 5), (0, 5, 0), (4, 0, 0)])
def test_quantize_rows(products, dtype, pow2, m, k, pad):
    gen = torch.Generator().manual_seed(m + k)
    x = (torch.randn(m, k + pad, generator=gen, dtype=torch.float64) * torch.exp(3 * torch.randn(m, 1, generator=gen, dtype=torch.float64))).to(dtype)
    x = x[:, :k]
    xd = x.cuda() if pad == 0 else torch.as_strided(torch.nn.functional.pad(x, (0, pad), value=float("nan")).cuda(), (m, k), (k + pad, 1))
    q, s, r = products.quantize_rows(xd, pow2=pow2, residual=True)
    qr, sr, rr = quantize_ref(x, pow2)
    assert np.array_equal(s.cpu().numpy(), sr)
    assert np.array_equal(q.cpu().numpy(), qr)
    if pow2:
        assert torch.equal(r.cpu(), torch.from_numpy(rr).to(dtype)) and np.array_equal(r.cpu().double().numpy(), rr)
    else:  # x - s q is formed in 64 bits and rounded: half a step of the type (not less than half of its
        # smallest number, the step below the normal ones), one of 64 bits of x
        least = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
        assert (np.abs(r.cpu().double().numpy() - rr) <= least + torch.finfo(dtype).eps / 2 * np.abs(rr) + 2.0 ** -52 * np.abs(x.double().numpy())).all()
    q2, s2 = products.quantize_rows(xd, pow2=pow2)
    assert torch.equal(q2, q) and torch.equal(s2, s)


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("pow2", [False, True])
def test_quantize_rows_of_odd_values(products, dtype, pow2):
    fi = torch.finfo(dtype)
    rows = [
        [0.0] * 8, [-0.0, 0.0] * 4, [fi.tiny] * 8, [fi.smallest_normal, -fi.smallest_normal] + [0.0] * 6, [fi.max, -fi.max, 1.0, 0.0] * 2,
        [127.0, 0.5, 1.5, 2.5, -0.5, -1.5, -2.5, 126.5],  # scale 1: ties to even
        [128.0, 1.0, 3.0, 5.0, -1.0, -3.0, -5.0, 127.0], [float("inf"), 1.0] * 4, [float("nan"), 1.0] * 4, [float("inf"), float("nan")] * 4,
        [1.0, float("-inf")] + [0.0] * 6,
    ]
    x = torch.tensor(rows, dtype=torch.float64).to(dtype)
    q, s = products.quantize_rows(x.cuda(), pow2=pow2)
    qr, sr, _ = quantize_ref(x, pow2)
    assert np.array_equal(s.cpu().numpy(), sr, equal_nan=True)
    assert np.array_equal(q.cpu().numpy(), qr)


INT8_SHAPES = [(1, 1, 1), (1, 130, 64), (2, 5, 131071), (3, 17, 1001), (64, 64, 128), (128, 128, 256), (129, 255, 130), (300, 1001, 500), (17, 33, 0), (257, 512, 1024)]


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("m, n, k", INT8_SHAPES)
def test_int8_matmul(products, dtype, m, n, k):
    gen = torch.Generator().manual_seed(m * n + k)
    a = torch.randint(-128, 128, (m, k), generator=gen, dtype=torch.int8)
    b = torch.randint(-128, 128, (n, k), generator=gen, dtype=torch.int8)
    if k == 131071:
        a[0] = -128  # the largest sum there is: 128 * 128 * 131071 < 2^31
        b[0] = -128
    stype = torch.float64 if dtype == torch.float64 else torch.float32
    sa, sb = (torch.rand(r, generator=gen, dtype=torch.float64).add(0.5).to(stype) / 128 for r in (m, n))
    c = torch.randn(m, n, generator=gen, dtype=torch.float64).to(dtype)
    acc = a.double() @ b.double().T
    ref = acc * (sa.double()[:, None] * sb.double()[None, :])
    ref_c = ref + c.double()
    dev = [t.cuda() for t in (a, b, sa, sb)]
    y = products.int8_matmul(*dev, dtype=dtype)
    if dtype in (torch.bfloat16, torch.float16):
        # one rounding, of a value that 64 bits hold to 2^-52: the reference's own rounding, but for ties it may tip
        lim = torch.finfo(dtype).eps / 2 * ref.abs() + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
        got = y.cpu().double()
        assert (((got - ref).abs() <= lim * (1 + 1e-12)) | (got.isinf() & (ref.abs() >= torch.finfo(dtype).max))).all()
    else:
        half = torch.finfo(dtype).eps / 2
        assert ((y.cpu().double() - ref).abs() <= half * ref.abs() + 2.0 ** -51 * ref.abs()).all()
    # added to what is there, in place, inside a larger matrix
    out, rim = guarded((m, n), dtype)
    out.copy_(c)
    assert products.int8_matmul(*dev, c=out, dtype=dtype, out=out) is out
    mags = ref.abs() + c.double().abs()
    got = out.cpu().double()
    lim = torch.finfo(dtype).eps / 2 * ref_c.abs() + 2.0 ** -51 * mags + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    assert (((got - ref_c).abs() <= lim * (1 + 1e-12)) | (got.isinf() & (ref_c.abs() >= torch.finfo(dtype).max))).all()
    rim()
    if k:
        # operands inside larger ones, off the 16-byte grid, with other columns around them
        ap, bp = (torch.nn.functional.pad(t, (3, 2), value=99).cuda()[:, 3:3 + k] for t in (a, b))
        assert torch.equal(products.int8_matmul(ap, bp, dev[2], dev[3], dtype=dtype), y)


def test_a_64_bit_product_out_of_8_bit_slices(products):
    """Slices of both operands, each pair's product added to a 64-bit matrix: the run of the two operators together."""
    gen = torch.Generator().manual_seed(5)
    m, n, k = 100, 75, 260
    a = torch.randn(m, k, generator=gen, dtype=torch.float64)
    b = torch.randn(n, k, generator=gen, dtype=torch.float64)

    def slices(x, count):
        out, rest = [], x.cuda()
        for _ in range(count):
            q, s, rest = products.quantize_rows(rest, pow2=True, residual=True)
            out.append((q, s))
        return out, rest

    sa, ra = slices(a, 8)
    sb, rb = slices(b, 8)
    # each slice leaves at most half of the next power of two below 1/127 of what was there: 8 slices, 2^-53 and less
    assert float(ra.abs().max()) <= float(a.abs().max()) * 2.0 ** -53 and float(rb.abs().max()) <= float(b.abs().max()) * 2.0 ** -53
    y = torch.zeros(m, n, dtype=torch.float64, device="cuda")
    for i in reversed(range(8)):
        for j in reversed(range(8)):
            products.int8_matmul(sa[i][0], sb[j][0], sa[i][1], sb[j][1], c=y, dtype=torch.float64, out=y)
    exact = a.to(torch.float64) @ b.T
    mags = a.abs() @ b.abs().T
    # the rests: 2^-53 of each operand's largest entry against the other's row; 64 additions and the reference's k, 2^-52 each
    lost = 2.0 ** -53 * (a.abs().amax(1, keepdim=True) * b.abs().sum(1)[None, :] + a.abs().sum(1, keepdim=True) * b.abs().amax(1)[None, :])
    assert ((y.cpu() - exact).abs() <= lost * (1 + 1e-6) + (64 + k) * 2.0 ** -52 * mags).all()


def test_a_quantised_expert_layer_end_to_end(products):
    """Grouped product, its rows quantised, a second layer in 8 bits: as a model would call them, against 64 bits."""
    x, w = whole((70, 64), 1), whole((4, 96, 64), 2)
    off = [0, 20, 20, 45, 70]
    h = products.grouped_matmul(x.to(torch.bfloat16).cuda(), w.to(torch.bfloat16).cuda(), torch.tensor(off, device="cuda"))
    href = grouped_ref(x, w, off).to(torch.bfloat16)
    q, s = products.quantize_rows(h)
    qr, sr, _ = quantize_ref(href, False)
    assert np.array_equal(q.cpu().numpy(), qr) and np.array_equal(s.cpu().numpy(), sr)
    wq, ws = products.quantize_rows(whole((33, 96), 3, most=100, dtype=torch.float32).cuda())
    y = products.int8_matmul(q, wq, s, ws, dtype=torch.float32)
    ref = (q.cpu().double() @ wq.cpu().double().T) * (s.cpu().double()[:, None] * ws.cpu().double()[None, :])
    assert ((y.cpu().double() - ref).abs() <= 2.0 ** -24 * (1 + 1e-6) * ref.abs()).all()


# ---- streams, graphs, threads ----

def test_runs_on_the_current_stream(products):
    x, w, off = whole((600, 256), 1).float().cuda(), whole((3, 256, 256), 2).float().cuda(), torch.tensor([0, 100, 350, 600], device="cuda")
    ref = products.grouped_matmul(x, w, off)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        buf = x * 2
        y = products.grouped_matmul(buf, w, off)
        z = products.quantize_rows(y)[1]
    st.synchronize()
    # the quotient in 64 bits, rounded: a tensor divided by a number is multiplied by its rounded reciprocal on the GPU
    assert torch.equal(y, ref * 2) and torch.equal(z.cpu(), ((ref * 2).abs().amax(1).double().cpu() / 127).float())


def test_graph_replays(products):
    t, n, k, g = 333, 130, 200, 5
    x, w, dy = (whole(s, i).float().cuda() for i, s in enumerate(((t, k), (g, n, k), (t, n))))
    off = torch.tensor([0, 50, 50, 120, 300, 333], device="cuda")

    def step():
        y = products.grouped_matmul(x, w, off)
        dx, dw = products.grouped_matmul_grad(dy, x, w, off)
        q, s, r = products.quantize_rows(y, pow2=True, residual=True)
        z = products.int8_matmul(q, q, s, s, dtype=torch.float32)
        return y, dx, dw, q, s, r, z

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for i in range(4):
        x.copy_(whole((t, k), 10 + i))
        w.copy_(whole((g, n, k), 20 + i))
        cuts = torch.sort(torch.randint(0, t + 1, (g - 1,), generator=torch.Generator().manual_seed(i)))[0]
        off[1:g].copy_(cuts)
        graph.replay()
        torch.cuda.synchronize()
        kept = [o.clone() for o in outs]
        for a, b in zip(kept, step()):
            assert torch.equal(a, b)
        torch.cuda.synchronize()


def test_calls_from_two_threads(products):
    from concurrent.futures import ThreadPoolExecutor

    def work(seed):
        st = torch.cuda.Stream()
        with torch.cuda.stream(st):
            x, w = whole((200, 100), seed).cuda(), whole((2, 150, 100), seed + 1).cuda()
            off = torch.tensor([0, 90, 200], device="cuda")
            for _ in range(10):
                y = products.grouped_matmul(x, w, off)
            st.synchronize()
            return torch.equal(y.cpu(), grouped_ref(x.cpu(), w.cpu(), [0, 90, 200]))

    with ThreadPoolExecutor(2) as pool:
        assert all(pool.map(work, [1, 50]))


def test_results_do_not_change_from_run_to_run(products):
    gen = torch.Generator(device="cuda").manual_seed(1)
    for dtype in ALL:
        x, w, dy = (torch.randn(*s, generator=gen, device="cuda").to(dtype) for s in ((900, 320), (3, 200, 320), (900, 200)))
        off = torch.tensor([0, 10, 700, 900], device="cuda")
        first = (products.grouped_matmul(x, w, off), *products.grouped_matmul_grad(dy, x, w, off))
        for _ in range(3):
            again = (products.grouped_matmul(x, w, off), *products.grouped_matmul_grad(dy, x, w, off))
            assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_offsets_past_32_bits(products):
    """A matrix of more than 2^31 elements (and bytes past 2^32), read and written at its far end."""
    if torch.cuda.mem_get_info()[0] < 40 * 2 ** 30:
        pytest.skip("needs 40 GiB of free memory")
    t, k, n = 2 ** 22 + 5, 520, 520
    x = torch.zeros(t, k, dtype=torch.bfloat16, device="cuda")
    tail = whole((300, k), 1)
    x[-300:] = tail.to(torch.bfloat16).cuda()
    w = whole((2, n, k), 2)
    off = torch.tensor([0, t - 200, t], device="cuda")
    y = products.grouped_matmul(x, w.to(torch.bfloat16).cuda(), off)
    assert torch.equal(y[-200:].cpu(), (tail[100:] @ w[1].T).to(torch.bfloat16))
    assert torch.equal(y[-300:-200].cpu(), (tail[:100] @ w[0].T).to(torch.bfloat16))
    dx, dw = products.grouped_matmul_grad(y, x, w.to(torch.bfloat16).cuda(), off)
    dyt = y[-300:].cpu().double()
    assert torch.equal(dx[-300:-200].cpu(), (dyt[:100] @ w[0]).to(torch.bfloat16)) or (
        (dx[-300:-200].cpu().double() - dyt[:100] @ w[0]).abs() <= 2.0 ** -8 * (dyt[:100] @ w[0]).abs() + n * 2.0 ** -23 * (dyt[:100].abs() @ w[0].abs())).all()
    ref = dyt[100:].T @ tail[100:]
    assert ((dw[1].cpu().double() - ref).abs() <= 2.0 ** -8 * (ref.abs() + 1e-3) + 200 * 2.0 ** -23 * (dyt[100:].abs().T @ tail[100:].abs())).all()
    del x, y, dx
    a = torch.zeros(2 ** 22 + 3, 1040, dtype=torch.int8, device="cuda")
    a[-1] = 3
    z = products.int8_matmul(a, a[-2:], torch.ones(a.shape[0], device="cuda"), torch.ones(2, device="cuda"))
    assert z[-1].tolist() == [0.0, float(torch.tensor(9360.0).bfloat16())] and not z[:-1].any()


# ---- sizes and strides that take the other ways through the library ----

def gpu_whole(shape, seed, dtype, most=4):
    return torch.randint(-most, most + 1, shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)).to(dtype)


def gpu_grouped_ref(x, w, off):
    """in 64 bits on the GPU, one group at a time"""
    y = torch.zeros(x.shape[0], w.shape[1], dtype=torch.float64, device="cuda")
    for g, (a, b) in enumerate(rows_of(off)):
        if b > a:
            y[a:b] = x[a:b].double() @ w[g].double().T
    return y


def in_rows_of(t, ld, at=0):
    """t[.., m, n] inside rows of ld elements, from column `at` on, NaN (99) around it"""
    buf = torch.full((*t.shape[:-1], ld), 99 if t.dtype == torch.int8 else float("nan"), dtype=t.dtype, device="cuda")
    buf[..., at:at + t.shape[-1]] = t
    return buf[..., at:at + t.shape[-1]]


CUTS = [  # rows of the groups, n, k: many tiles, a last round of few, long k with few tiles, long groups with few tiles
    ([1500, 3, 0, 700, 2600], 1500, 70),
    ([4000, 260, 1], 4300, 200),
    ([9000], 2100, 24),
    ([3], 96, 4100),
    ([17, 0, 30], 130, 2600),
    ([6000, 0, 2500], 70, 90),
    ([20000], 33, 40),
]


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("counts, n, k", CUTS, ids=lambda v: str(v).replace(" ", ""))
@pytest.mark.parametrize("layout", ["contiguous", "aligned rows", "words", "odd"])
def test_larger_products_and_layouts(products, dtype, counts, n, k, layout):
    """exact whole numbers again: |x|, |w|, |dy| <= 2, so that sums of 20000 products stay below 2^24"""
    off = np.concatenate(([0], np.cumsum(counts))).tolist()
    t, g = off[-1], len(counts)
    x, w, dy = gpu_whole((t, k), 1, dtype, 2), gpu_whole((g, n, k), 2, dtype, 2), gpu_whole((t, n), 3, dtype, 2)
    yr, dxr = gpu_grouped_ref(x, w, off), gpu_grouped_ref(dy, w.transpose(1, 2), off)
    dwr = torch.stack([dy[a:b].double().T @ x[a:b].double() for a, b in rows_of(off)])
    if layout != "contiguous":
        size = dtype.itemsize
        unit = {"aligned rows": 16, "words": max(4, size), "odd": size}[layout] // size
        at = {"aligned rows": 0, "words": unit, "odd": 1}[layout]
        x, w, dy = (in_rows_of(m, (m.shape[-1] + at) // unit * unit + 2 * unit, at) for m in (x, w, dy))
    od = torch.tensor(off, device="cuda")
    assert torch.equal(products.grouped_matmul(x, w, od), yr.to(dtype))
    dx, dw = products.grouped_matmul_grad(dy, x, w, od)
    assert torch.equal(dx, dxr.to(dtype))
    if dtype == torch.float16:  # sums past 65504 are infinities in both
        assert torch.equal(dw, dwr.float().to(dtype))
    else:
        assert torch.equal(dw, dwr.to(dtype))
    wt = w.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(products.grouped_matmul(x, wt, od), yr.to(dtype))
    dx, _ = products.grouped_matmul_grad(dy, x, wt, od)
    assert torch.equal(dx, dxr.to(dtype))


@pytest.mark.parametrize("m, n, k", [(3000, 5000, 300), (2600, 2700, 33), (1, 300, 9000), (70, 50, 8000), (9000, 20, 100)])
@pytest.mark.parametrize("layout", ["contiguous", "aligned rows", "words", "odd"])
def test_larger_int8_products_and_layouts(products, m, n, k, layout):
    gen = torch.Generator(device="cuda").manual_seed(m)
    a, b = (torch.randint(-128, 128, s, device="cuda", generator=gen, dtype=torch.int8) for s in ((m, k), (n, k)))
    ref = a.double() @ b.double().T  # below 2^53: exact
    if layout != "contiguous":
        unit, at = {"aligned rows": (16, 0), "words": (4, 4), "odd": (1, 1)}[layout]
        a, b = (in_rows_of(t, (k + at) // unit * unit + 2 * unit, at) for t in (a, b))
    one = torch.ones(max(m, n), device="cuda", dtype=torch.float64)
    assert torch.equal(products.int8_matmul(a, b, one[:m], one[:n], dtype=torch.float64), ref)
    half = torch.full((max(m, n),), 0.5, device="cuda")
    got = products.int8_matmul(a, b, half[:m], half[:n], dtype=torch.bfloat16)
    # a quarter of a whole number below 2^53: its rounding to bf16 by way of fp32 could round twice; by way of whole steps not
    step = torch.exp2(torch.floor(torch.log2((ref / 4).abs().clamp_min(1e-30))) - 7)
    assert torch.equal(got.double(), torch.where(ref == 0, ref, torch.round(ref / 4 / step) * step))


def test_offsets_that_do_not_ascend_stay_inside(products):
    """what they select is up to the call, but nothing outside the output is written and the call ends"""
    x, w = gpu_whole((300, 64), 1, torch.float32), gpu_whole((5, 70, 64), 2, torch.float32)
    for off in ([0, 300, 0, 300, 0, 300], [300, 200, 100, 50, 20, 0], [-9, 2 ** 60, -2 ** 60, 7, 3, 2 ** 40]):
        out, rim = guarded((300, 70), torch.float32)
        od = torch.tensor(off, device="cuda")
        products.grouped_matmul(x, w, od, out=out)
        products.grouped_matmul_grad(out, x, w, od)
        torch.cuda.synchronize()
        rim()
    many = torch.tensor([0, 300] * 2000 + [0], device="cuda")
    products.grouped_matmul(x, w[:1].expand(4000, 70, 64), many)
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_numbers_below_the_normal_ones(products, dtype):
    fi = torch.finfo(dtype)
    least = fi.smallest_normal * fi.eps  # the smallest number above 0
    x = torch.tensor([[least, 3 * least, -5 * least, fi.smallest_normal] + [0.0] * 12], dtype=torch.float64)
    w = torch.eye(16, dtype=torch.float64)[None] * 64.0
    y = products.grouped_matmul(x.to(dtype).cuda(), w.to(dtype).cuda(), torch.tensor([0, 1], device="cuda"))
    assert torch.equal(y.cpu().double(), x * 64.0)


def test_infinities_stay_in_their_rows(products):
    for dtype in ALL:
        x, w = whole((40, 100), 1).to(dtype).cuda(), whole((2, 50, 100), 2).to(dtype).cuda()
        off = torch.tensor([0, 25, 40], device="cuda")
        clean = products.grouped_matmul(x, w, off)
        x[7, 3], w[1, 9, 99] = float("inf"), float("-inf")
        y = products.grouped_matmul(x, w, off)
        hit = torch.zeros(40, 50, dtype=torch.bool, device="cuda")
        hit[7] = True
        hit[25:, 9] = True
        assert torch.equal(y[~hit], clean[~hit]) and not y[hit].isfinite().any()


def test_rest_in_the_place_of_the_input(products):
    """the C entry lets the rest overwrite what was quantised: in rows that are kept in registers and in longer ones"""
    import ctypes as C

    from battgp_amd import _lib

    lib = _lib.load_products()
    st = C.c_void_p(torch.cuda.current_stream().cuda_stream)
    for k in (50, 3000, 8000, 30000):
        x = torch.randn(5, k, device="cuda", dtype=torch.float64)
        q, s, r = products.quantize_rows(x, pow2=True, residual=True)
        q2, s2 = torch.empty_like(q), torch.empty_like(s)
        assert lib.bgp_quantize_rows(0, st, _lib.F64, 5, k, x.data_ptr(), k, q2.data_ptr(), k, s2.data_ptr(), 1, x.data_ptr(), k) == 0
        torch.cuda.synchronize()
        assert torch.equal(x, r) and torch.equal(q2, q) and torch.equal(s2, s)


def test_workspaces_are_asked_for_and_fewer_bytes_refused(products):
    import ctypes as C

    from battgp_amd import _lib

    lib = _lib.load_products()
    st = C.c_void_p(torch.cuda.current_stream().cuda_stream)
    t, n, k = 2, 64, 8192  # few tiles and a long k along rows: k is cut
    x, w, off = gpu_whole((t, k), 1, torch.bfloat16, 1), gpu_whole((1, k, n), 2, torch.bfloat16, 1), torch.tensor([0, t], device="cuda")
    y = torch.full((t, n), 7.0, dtype=torch.bfloat16, device="cuda")
    args = (0, st, _lib.BF16, t, n, k, 1, x.data_ptr(), k, w.data_ptr(), n * k, n, 1, off.data_ptr(), y.data_ptr(), n, 0)
    need = lib.bgp_grouped_gemm(*args, None, 0)
    assert need > 0
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    assert lib.bgp_grouped_gemm(*args, ws.data_ptr(), need - 1) == need
    torch.cuda.synchronize()
    assert (y == 7.0).all()  # nothing was enqueued
    assert lib.bgp_grouped_gemm(*args, ws.data_ptr(), need) == 0
    assert torch.equal(y, (x.double() @ w[0].double()).to(torch.bfloat16))


def test_graph_replays_with_workspaces(products):
    """two graphs that cut k and copy operands, replayed in turn with eager work between"""
    off = torch.tensor([0, 3], device="cuda")
    w = gpu_whole((1, 4100, 96), 2, torch.bfloat16, 1).transpose(1, 2)
    a, b = (torch.randint(-99, 99, s, device="cuda", dtype=torch.int8) for s in ((2100, 2047), (2200, 2047)))
    one = torch.ones(2200, device="cuda")
    x = gpu_whole((3, 4100), 3, torch.bfloat16, 1)

    def first():
        return products.grouped_matmul(x, w, off)

    def second():
        return products.int8_matmul(a, b, one[:2100], one, dtype=torch.float32)

    first(), second()
    torch.cuda.synchronize()
    graphs = []
    for f in (first, second):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = f()
        graphs.append((g, out))
    for i in range(4):
        x.copy_(gpu_whole((3, 4100), 10 + i, torch.bfloat16, 1))
        a.copy_(torch.randint(-99, 99, a.shape, device="cuda", dtype=torch.int8))
        for g, _ in graphs:
            g.replay()
        eager = (first(), second())
        torch.cuda.synchronize()
        assert torch.equal(graphs[0][1], eager[0]) and torch.equal(graphs[1][1], eager[1])


def test_rows_of_more_than_one_launch_are_quantised(products):
    """67 million rows of one number: the code is 127 or -127, the scale the number's 127th part.  (The quotient in 64 bits
    is not rounded across an fp32 midpoint m: a / 127 - m is a whole multiple of m's last place / 254, or 0.)"""
    m = 4 * ((1 << 24) - 1) + 5
    x = torch.randint(-64, 65, (m, 1), device="cuda", generator=torch.Generator("cuda").manual_seed(5), dtype=torch.int8).to(torch.bfloat16)
    q, scale = products.quantize_rows(x)
    assert torch.equal(q[:, 0], torch.sign(x[:, 0]).to(torch.int8) * 127)
    want = (x[:, 0].double().abs() / 127).float().clamp_min(torch.finfo(torch.float32).tiny)
    assert torch.equal(scale, want)


def test_more_row_tiles_than_the_smallest_cut_could_launch(products):
    t, n, k = 150_000_001, 8, 8
    x = torch.randint(-4, 5, (t, k), device="cuda", generator=torch.Generator("cuda").manual_seed(6), dtype=torch.int8).to(torch.bfloat16)
    w = whole((2, n, k), 7, dtype=torch.bfloat16).cuda()
    cut = 75_000_005
    y = products.grouped_matmul(x, w, torch.tensor([0, cut, t - 3], device="cuda"))
    for a, b, g in ((0, cut, 0), (cut, t - 3, 1)):
        for i in range(a, b, 25_000_000):
            j = min(i + 25_000_000, b)  # sums of 8 products up to 16: exact in bf16 (128 < 256)
            assert torch.equal(y[i:j], (x[i:j].float() @ w[g].float().T).to(torch.bfloat16))
    assert not y[t - 3:].any()


# ---- few tiles of long k, whose k two sets of waves may halve: one stage, two, odd numbers of them, parts of one, ragged edges ----


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("k", [64, 72, 128, 136, 192, 200, 264, 1048, 2056, 4104])
@pytest.mark.parametrize("counts, n", [([70, 0, 3, 64], 200), ([300], 1000), ([1], 264), ([65, 129], 72)])
def test_few_tiles_of_long_k(products, dtype, k, counts, n):
    """whole numbers again: |sums| <= 4 * 4104 < 2^24"""
    off = np.concatenate(([0], np.cumsum(counts))).tolist()
    t, g = off[-1], len(counts)
    x, w = gpu_whole((t, k), 1, dtype, 2), gpu_whole((g, n, k), 2, dtype, 2)
    ref, od = gpu_grouped_ref(x, w, off).to(dtype), torch.tensor(off, device="cuda")
    assert torch.equal(products.grouped_matmul(x, w, od), ref)
    assert torch.equal(products.grouped_matmul(x, w.transpose(1, 2).contiguous().transpose(1, 2), od), ref)
    out, rim = guarded((t, n), dtype)
    products.grouped_matmul(x, w.transpose(1, 2).contiguous().transpose(1, 2), od, out=out)
    assert torch.equal(out, ref)
    rim()


@pytest.mark.parametrize("counts", [[1], [64], [65, 0, 128], [200, 1], [1000], [63, 2000]])
@pytest.mark.parametrize("n, k", [(200, 136), (512, 520), (72, 64)])
def test_weight_gradients_of_few_tiles(products, counts, n, k):
    off = np.concatenate(([0], np.cumsum(counts))).tolist()
    dy, x = gpu_whole((off[-1], n), 1, torch.bfloat16, 2), gpu_whole((off[-1], k), 2, torch.bfloat16, 2)
    _, dw = products.grouped_matmul_grad(dy, x, gpu_whole((len(counts), n, k), 3, torch.bfloat16), torch.tensor(off, device="cuda"), need_dx=False)
    want = torch.stack([dy[a:b].double().T @ x[a:b].double() for a, b in rows_of(off)])
    assert torch.equal(dw, want.to(torch.bfloat16))


@pytest.mark.parametrize("k", [128, 144, 256, 400, 2000, 4112, 8016])
@pytest.mark.parametrize("m, n", [(300, 1000), (65, 130), (500, 900)])
@pytest.mark.parametrize("dtype", ALL)
def test_few_tiles_of_long_k_in_8_bits(products, m, n, k, dtype):
    gen = torch.Generator(device="cuda").manual_seed(k)
    a, b = (torch.randint(-128, 128, s, device="cuda", generator=gen, dtype=torch.int8) for s in ((m, k), (n, k)))
    small = torch.full((max(m, n),), 2.0 ** -7, device="cuda", dtype=torch.float64 if dtype == torch.float64 else torch.float32)
    ref = a.double() @ b.double().T * 2.0 ** -14  # exact; its magnitude is below 8016 and above 2^-14: normal in every type
    got = products.int8_matmul(a, b, small[:m], small[:n], dtype=dtype)
    assert ((got.double() - ref).abs() <= (torch.finfo(dtype).eps / 2 if dtype != torch.float64 else 0) * ref.abs()).all()


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("wt", [False, True])
@pytest.mark.parametrize("t, n, k", [(1500, 1201, 1301), (5, 7, 9), (1, 8, 0)])
def test_without_groups_all_rows_are_zero(products, dtype, wt, t, n, k):
    """sizes and rows off the 16-byte chunks, whose operands would be copied if there were any"""
    x, dy = gpu_whole((t, k), 1, dtype), gpu_whole((t, n), 2, dtype)
    w = torch.empty((0, k, n) if wt else (0, n, k), dtype=dtype, device="cuda")
    w, off = w.transpose(1, 2) if wt else w, torch.zeros(1, dtype=torch.int64, device="cuda")
    y = products.grouped_matmul(x, w, off)
    assert y.shape == (t, n) and not y.any()
    dx, dw = products.grouped_matmul_grad(dy, x, w, off)
    assert dx.shape == (t, k) and not dx.any() and dw.shape == (0, n, k)
    out, rim = guarded((t, n), dtype)
    out.fill_(5.0)
    products.grouped_matmul(x, w, off, out=out)
    assert (out == 5.0).all()
    rim()


def operands_of_every_call(products):
    """ordinary calls, as the compiled way takes them, with their floating point operands"""
    x, w, dy, off = gpu_whole((6, 3), 1, torch.float32), gpu_whole((2, 4, 3), 2, torch.float32), gpu_whole((6, 4), 3, torch.float32), torch.tensor([0, 2, 6], device="cuda")
    a, s, c = gpu_whole((6, 3), 4, torch.int8), gpu_whole((6,), 5, torch.float32), gpu_whole((6, 6), 6, torch.float32)
    return [
        (lambda x, w: products.grouped_matmul(x, w, off), (x, w)),
        (lambda dy, x, w: products.grouped_matmul_grad(dy, x, w, off), (dy, x, w)),
        (lambda x: products.quantize_rows(x), (x,)),
        (lambda sa, sb, c: products.int8_matmul(a, a, sa, sb, c=c, dtype=torch.float32), (s, s, c)),
    ]


@pytest.mark.parametrize("i", range(4))
def test_tangents_are_refused(products, i):
    import torch.autograd.forward_ad as fw

    call, operands = operands_of_every_call(products)[i]
    for j, t in enumerate(operands):
        with fw.dual_level():
            with pytest.raises(ValueError, match="tangent"):
                call(*operands[:j], fw.make_dual(t, torch.ones_like(t)), *operands[j + 1:])
            call(*operands)


@pytest.mark.parametrize("i", range(4))
def test_transformed_operands_are_refused(products, i):
    call, operands = operands_of_every_call(products)[i]
    for j, t in enumerate(operands):
        def with_one(v):
            return call(*operands[:j], v, *operands[j + 1:])

        with pytest.raises(ValueError, match="own values"):
            torch.func.vmap(with_one)(t[None])
        with pytest.raises(ValueError, match="own values|tangent"):
            torch.func.jvp(with_one, (t,), (t,))
        with pytest.raises(ValueError, match="gradient"):
            torch.func.grad(lambda v: with_one(v)[0].sum())(t)


def test_fp64_codes_next_to_a_half(products):
    """quotients that 64 bits round to a half which they are not: the code is the nearest to the quotient itself"""
    from fractions import Fraction

    rng = np.random.default_rng(3)
    rows, want = [], []
    while len(rows) < 60:
        top = float(rng.uniform(0.5, 2.0) * 2.0 ** rng.integers(-40, 40))
        scale = top / 127.0
        row, codes = [top], [127]
        for half in np.arange(0.5, 127.0):
            for x in (half * scale, float(np.nextafter(half * scale, 0.0)), float(np.nextafter(half * scale, np.inf))):
                exact = Fraction(x) / Fraction(scale)
                if x / scale == half and exact != Fraction(half):
                    nearest = int(half) + (exact > Fraction(half))
                    if nearest != int(np.rint(half)):
                        row += [x, -x]
                        codes += [nearest, -nearest]
        if len(row) > 1:
            rows.append(row[:9] + [0.0] * (9 - len(row)))
            want.append(codes[:9] + [0] * (9 - len(codes)))
    x = torch.tensor(rows, dtype=torch.float64)
    q, s, r = products.quantize_rows(x.cuda(), residual=True)
    assert torch.equal(s.cpu(), x[:, 0] / 127.0)
    assert torch.equal(q.cpu(), torch.tensor(want, dtype=torch.int8))
    for xi, qi, si, ri in zip(x.tolist(), q.tolist(), s.tolist(), r.tolist()):
        for a, b, c in zip(xi, qi, ri):  # what is left over is a number of 64 bits: exact
            assert Fraction(c) == Fraction(a) - b * Fraction(si)


@pytest.mark.parametrize("dtype", ALL)
def test_outputs_beside_their_inputs(products, dtype):
    """blocks of columns of one matrix, off the 16-byte chunks: the input stays as it was, and autograd notices the output"""
    t, n, k = 300, 70, 53
    buf, off = gpu_whole((t, 1 + k + 2 + n + 1), 1, dtype), torch.tensor([0, 100, 100, 290], device="cuda")
    w, before = gpu_whole((3, n, k), 2, dtype), buf.clone()
    x, out = buf[:, 1:1 + k], buf[:, k + 3:k + 3 + n]
    z = torch.ones(t, n, dtype=dtype, device="cuda", requires_grad=True) * out
    assert products.grouped_matmul(x, w, off, out=out) is out
    want = before.clone()
    want[:290, k + 3:k + 3 + n] = gpu_grouped_ref(before[:, 1:1 + k], w, [0, 100, 100, 290])[:290].to(dtype)
    assert torch.equal(buf, want)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.sum().backward()
