"""Block-scaled 8-bit operators on the GPU against their definitions in 64 bits (oracle/lowbit_oracle.py).

Tolerances.  The quantiser is exact: values and scales are compared to the bit.  A product of quantised operands adds K exact
products (4 + 4 significant bits) in fp32 in some order: off by at most K * 2^-24 * sum_k |a_k b_k|, plus half a step of the output
type (2^-24 / 2^-8 of the value).  `check_product` and the tests before "operands and sums" allow bf16 outputs 7 * 2^-13 *
sum_k |a_k b_k| more, what the 8-bit matrix instructions would lose; the tests behind it do not: sums are fp32 for every type."""
import numpy as np
import pytest
import torch

from conv1d_text_vae_amd import _lib as L
from oracle import lowbit_oracle as O

pytestmark = pytest.mark.gpu
KIND = {'f32': torch.float32, 'bf16': torch.bfloat16}


@pytest.fixture(scope='module')
def fp8():
    from conv1d_text_vae_amd import fp8 as m
    return m


def data(rows, cols, kind, seed, gap=0):
    """Rows of different magnitude, large single values, zero rows, denormal and huge blocks."""
    rng = np.random.RandomState(seed)
    x = rng.standard_normal((rows, cols)) * np.exp(rng.standard_normal((rows, 1)))
    x[rng.rand(rows, cols) < 0.01] *= 50
    if rows > 2:
        x[1] = 0.0
    if rows > 6:
        x[3] *= 1e-40
        x[4] *= 1e30
        x[5] = -0.0
    t = torch.from_numpy(x.astype(np.float32)).to(KIND[kind])
    if not gap:
        return t.cuda()
    wide = torch.full((rows, cols + gap), float('nan'), dtype=t.dtype)
    wide[:, :cols] = t
    return wide.cuda()[:, :cols]


def f64(t):
    return t.detach().float().cpu().numpy().astype(np.float64)


def check_rows(q, x):
    """An Fp8Rows against the oracle's quantisation of x [R, K] (float64)."""
    want, e = O.quantize(x)
    got = f64(q.data)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    np.testing.assert_array_equal(np.nan_to_num(got), np.nan_to_num(want))
    s = q.scale.cpu().numpy().astype(np.int64)
    np.testing.assert_array_equal(s[:, :x.shape[0]].T - 127, e)
    assert (s[:, x.shape[0]:] == 127).all()
    assert (q.rows, q.cols) == x.shape


@pytest.mark.parametrize('kind', ['f32', 'bf16'])
@pytest.mark.parametrize('rows,cols,gap', [(1, 1, 0), (1, 128, 0), (3, 127, 5), (16, 129, 0), (17, 300, 1), (127, 64, 0), (128, 256, 0),
                                           (129, 131, 3), (260, 1000, 0), (1000, 7, 1)])
def test_quantiser_is_exact(fp8, kind, rows, cols, gap):
    x = data(rows, cols, kind, rows * 7 + cols, gap)
    ref = f64(x)
    check_rows(fp8.quantize_rows(x), ref)
    check_rows(fp8.quantize_cols(x), ref.T)
    a, b = fp8.quantize_both(x)
    check_rows(a, ref)
    check_rows(b, ref.T)
    np.testing.assert_array_equal(f64(fp8.quantize_rows(x).dequantize()), O.quantized(ref))


def test_quantiser_keeps_what_is_no_number(fp8):
    x = data(140, 200, 'f32', 1)
    x[0, 3], x[0, 150], x[7, 0], x[139, 199] = float('nan'), float('inf'), float('-inf'), float('nan')
    x[20] = float('inf')
    a, b = fp8.quantize_both(x)
    check_rows(a, f64(x))
    check_rows(b, f64(x).T)
    check_rows(fp8.quantize_rows(x), f64(x))
    check_rows(fp8.quantize_rows(x.to(torch.bfloat16)), f64(x.to(torch.bfloat16)))


def test_quantiser_at_the_borders_of_a_scale(fp8):
    """amax exactly 448 * 2^k keeps the smaller scale, the next float32 above takes the larger one."""
    x = torch.zeros(8, 128, device='cuda')
    x[0, 0], x[1, 0] = 448.0, float(np.nextafter(np.float32(448.0), np.float32(1e9)))
    x[2, 5], x[3, 5] = -448.0 * 2.0 ** 60, 448.0 * 2.0 ** -111
    x[4, 0], x[5, 0], x[6, 0] = 3.4e38, 1.2e-38, 1e-45
    check_rows(fp8.quantize_rows(x), f64(x))
    check_rows(fp8.quantize_cols(x.t().contiguous()), f64(x))


def test_quantiser_takes_any_strides(fp8):
    x = data(40, 200, 'f32', 3)
    check_rows(fp8.quantize_rows(x.t()), f64(x).T)
    check_rows(fp8.quantize_rows(x[::2]), f64(x)[::2])
    check_rows(fp8.quantize_cols(x[:, 1:150]), f64(x)[:, 1:150].T)
    check_rows(fp8.quantize_rows(x[:1].expand(5, 200)), f64(x[:1].expand(5, 200)))
    check_rows(fp8.quantize_rows(x[:, ::3]), f64(x)[:, ::3])


def check_product(got, a, b, bias=None, relu=False, k=None):
    """a [m, k], b [n, k]: the operands' values in float64"""
    want = a @ b.T + (0.0 if bias is None else bias)
    size = np.abs(a) @ np.abs(b).T + (0.0 if bias is None else np.abs(bias))
    if relu:
        want = np.maximum(want, 0.0)
    half = 2.0 ** -24 if got.dtype == torch.float32 else 2.0 ** -8
    g = f64(got)
    assert g.shape == want.shape
    per = (a.shape[1] + 2) * 2.0 ** -24 + (7 * 2.0 ** -13 if got.dtype == torch.bfloat16 else 0.0)
    err = np.abs(g - want) - half * np.abs(want) - per * size * (1 + half)
    assert (err <= 0).all(), (err.max(), np.unravel_index(err.argmax(), err.shape))


SHAPES = [(1, 1, 1), (1, 1024, 1024), (2, 17, 300), (16, 130, 257), (17, 16, 128), (33, 65, 129), (64, 64, 640), (100, 1000, 64), (1000, 40, 1100), (256, 1024, 2048), (272, 1024, 300),
          (255, 257, 384), (256, 512, 1920), (300, 70, 4200), (2000, 1030, 300), (3000, 4200, 140),
          (4096, 4352, 300), (4100, 4400, 600), (6000, 5000, 1000)]


@pytest.mark.parametrize('kind', ['f32', 'bf16'])
@pytest.mark.parametrize('m,n,k', SHAPES)
def test_product_and_dense(fp8, kind, m, n, k):
    x = data(m, k, 'f32', m + n, 0)
    x = torch.where(torch.isfinite(x) & (x.abs() < 1e20), x, 0).to(KIND[kind])
    w = data(n, k, 'f32', m + n + k).clamp(-1e3, 1e3)
    bias = torch.linspace(-2, 2, n, device='cuda')
    qx, qw = fp8.quantize_rows(x), fp8.quantize_rows(w)
    a, b = O.quantized(f64(x)), O.quantized(f64(w))
    got = fp8.product(qx, qw, out_dtype=KIND[kind])
    check_product(got, a, b)
    assert torch.equal(got, fp8.product(qx, qw, out_dtype=KIND[kind]))                      # reproducible
    check_product(fp8.dense(x, qw, bias, relu=True), a, b, f64(bias), True)
    check_product(fp8.dense(x, qw, out_dtype=torch.float32), a, b)


@pytest.mark.parametrize('kind', ['f32', 'bf16'])
@pytest.mark.parametrize('m,n,k', [(5, 1301, 200), (40, 77, 200), (700, 333, 200), (2050, 1301, 200), (2048, 1312, 200), (4100, 4401, 330), (4352, 4100, 330), (66, 130, 4300)])
def test_bias_and_relu_in_every_form(fp8, kind, m, n, k):
    """Small, medium and large tiles, rows on and off 16-byte boundaries, a K cut into runs; the 64-bit product on the GPU."""
    a, b = fp8.quantize_rows(data(m, k, 'f32', m).clamp(-30, 30)), fp8.quantize_rows(data(n, k, 'f32', n + 1).clamp(-30, 30))
    A, B = a.dequantize().double(), b.dequantize().double()
    sums, size = A @ B.t(), A.abs() @ B.abs().t()
    bias = torch.linspace(-20, 20, n, device='cuda')
    per = (k + 2) * 2.0 ** -24 + (7 * 2.0 ** -13 if kind == 'bf16' else 0.0)
    half = 2.0 ** -24 if kind == 'f32' else 2.0 ** -8
    for with_bias in (False, True):
        for relu in (False, True):
            got = fp8.product(a, b, bias if with_bias else None, relu, KIND[kind]).double()
            want, most = (sums + bias.double(), size + bias.double().abs()) if with_bias else (sums, size)
            want = want.clamp(min=0.0) if relu else want
            assert ((got - want).abs() <= half * want.abs() + per * most * (1 + half)).all()


@pytest.mark.parametrize('m', [5, 40])
def test_dense_takes_slices_and_leading_dimensions(fp8, m):
    x = data(m, 302, 'bf16', 5, gap=3).clamp(-1e4, 1e4)
    wide = torch.full((m, 305), float('nan'), dtype=torch.bfloat16, device='cuda')
    wide[:, :302] = x
    w = fp8.quantize_cols(data(302, 75, 'f32', 6).clamp(-10, 10))
    a = O.quantized(f64(x))
    got = fp8.dense(wide[:, :302], w)
    check_product(got, a, f64(w.dequantize()))
    assert torch.equal(fp8.dense(x.reshape(1, m, 1, 302), w), got.view(1, m, 1, 75))
    assert torch.equal(fp8.dense(x.float(), w), fp8.dense(x, w, out_dtype=torch.float32))
    assert fp8.dense(x[:0], w).shape == (0, 75)


@pytest.mark.parametrize('m', [4, 70])
def test_a_value_that_is_no_number_stays_in_its_row(fp8, m):
    x = data(m, 300, 'f32', 7).clamp(-10, 10)
    x[2, 140] = float('inf')
    w = fp8.quantize_rows(data(33, 300, 'f32', 8).clamp(-1, 1))
    y = fp8.dense(x, w, relu=True)
    assert torch.isnan(y[2]).all() and torch.isfinite(y[torch.arange(m) != 2]).all()


def test_small_and_large_batches_agree(fp8):
    """The one-launch form for up to 16 rows quantises as the quantiser does: same operands, the same sums but for their order."""
    x = data(40, 1100, 'bf16', 9).clamp(-1e4, 1e4)
    w = fp8.quantize_rows(data(200, 1100, 'f32', 10).clamp(-1, 1))
    whole = fp8.dense(x, w, out_dtype=torch.float32)
    for i in range(0, 40, 13):
        part = fp8.dense(x[i:i + 13], w, out_dtype=torch.float32)
        check_product(part, O.quantized(f64(x[i:i + 13])), f64(w.dequantize()))
        check_product(whole[i:i + 13], O.quantized(f64(x[i:i + 13])), f64(w.dequantize()))


@pytest.mark.parametrize('kind', ['f32', 'bf16'])
@pytest.mark.parametrize('rows,k,n', [(1, 5, 3), (50, 130, 64), (128, 128, 128), (300, 302, 190)])
def test_linear_and_its_gradients(fp8, kind, rows, k, n):
    x = data(rows, k, 'f32', rows).clamp(-100, 100).to(KIND[kind]).requires_grad_(True)
    kernel = (data(k, n, 'f32', k + 1).clamp(-3, 3)).requires_grad_(True)
    bias = torch.linspace(-1, 1, n, device='cuda').requires_grad_(True)
    dy = data(rows, n, 'f32', n + 2).clamp(-5, 5).to(KIND[kind])
    y = fp8.linear(x, kernel, bias)
    dx, dk, db = torch.autograd.grad(y, (x, kernel, bias), dy)
    X, W, D = f64(x), f64(kernel), f64(dy)
    check_product(y, O.quantized(X), O.quantized(W.T), f64(bias))
    check_product(dx, O.quantized(D), O.quantized(W))
    check_product(dk, O.quantized(X.T), O.quantized(D.T))
    assert (np.abs(f64(db) - D.sum(0)) <= rows * 2.0 ** -24 * np.abs(D).sum(0)).all()
    assert (y.dtype, dx.dtype, dk.dtype, db.dtype) == (x.dtype, x.dtype, torch.float32, torch.float32)


def test_linear_gradient_against_differences(fp8):
    """On operands that the quantiser leaves as they are (small whole numbers), the layer is linear and its gradient is the
    difference quotient of  sum(y * c)  itself."""
    rng = np.random.RandomState(0)
    x = torch.from_numpy(rng.randint(-4, 5, (20, 30)).astype(np.float32)).cuda().requires_grad_(True)
    k = torch.from_numpy(rng.randint(-4, 5, (30, 10)).astype(np.float32)).cuda().requires_grad_(True)
    c = torch.from_numpy(rng.randint(-4, 5, (20, 10)).astype(np.float32)).cuda()
    (fp8.linear(x, k) * c).sum().backward()
    with torch.no_grad():
        for i, j in ((0, 0), (7, 29), (19, 3)):
            d = torch.zeros_like(x)
            d[i, j] = 1.0
            assert float(((fp8.linear(x + d, k) - fp8.linear(x - d, k)) * c).sum() / 2) == float(x.grad[i, j])
        for i, j in ((0, 0), (29, 9), (11, 4)):
            d = torch.zeros_like(k)
            d[i, j] = 1.0
            assert float(((fp8.linear(x, k + d) - fp8.linear(x, k - d)) * c).sum() / 2) == float(k.grad[i, j])


def test_linear_gradients_that_are_asked_for(fp8):
    x, k = data(30, 200, 'f32', 1).clamp(-3, 3), data(200, 40, 'f32', 2).clamp(-3, 3)
    b = torch.zeros(40, device='cuda')
    full = [t.clone().requires_grad_(True) for t in (x, k, b)]
    fp8.linear(*full).sum().backward()                                   # the gradient arrives as an expanded scalar
    for only in range(3):
        part = [t.clone().requires_grad_(i == only) for i, t in enumerate((x, k, b))]
        fp8.linear(*part).sum().backward()
        for i, t in enumerate(part):
            assert (t.grad is None) if i != only else torch.equal(t.grad, full[i].grad)
    twice = x.clone().requires_grad_(True)
    (fp8.linear(twice, k) + fp8.linear(twice, k)).sum().backward()
    assert torch.equal(twice.grad, 2 * full[0].grad)
    y = fp8.linear(x.view(2, 3, 5, 200), k)
    assert y.shape == (2, 3, 5, 40) and torch.equal(y.view(30, 40), fp8.linear(x, k))
    e = torch.zeros(0, 200, device='cuda', requires_grad=True)
    w = k.clone().requires_grad_(True)
    y = fp8.linear(e, w, b)
    y.sum().backward()
    assert y.shape == (0, 40) and not w.grad.any() and e.grad.shape == (0, 200)


@pytest.mark.parametrize('xk', ['f32', 'bf16'])
@pytest.mark.parametrize('kk', ['f32', 'bf16'])
@pytest.mark.parametrize('rows,k,n', [(2300, 130, 70), (129, 1000, 333)])
def test_linear_gradients_do_not_depend_on_which_are_asked_for(fp8, xk, kk, rows, k, n):
    """All three gradients together (two products and the sums in one launch where the layer is small) and each by itself."""
    x, w = data(rows, k, xk, 1).clamp(-3, 3), data(k, n, kk, 2).clamp(-3, 3)
    b, dy = torch.randn(n, device='cuda'), data(rows, n, xk, 3).clamp(-3, 3)
    args = [t.clone().requires_grad_(True) for t in (x, w, b)]
    every = torch.autograd.grad(fp8.linear(*args), args, dy)
    for i in range(3):
        one = [t.clone().requires_grad_(j == i) for j, t in enumerate((x, w, b))]
        assert torch.equal(torch.autograd.grad(fp8.linear(*one), one[i], dy)[0], every[i])
    a = fp8.quantize_both(dy)
    assert torch.equal(every[0], fp8.product(a[0], fp8.quantize_rows(w), out_dtype=x.dtype))
    assert torch.equal(every[1], fp8.product(fp8.quantize_cols(x), a[1], out_dtype=w.dtype))


def test_captured_product_and_training_pass_replay(fp8):
    """dense (both forms) and a forward + backward pass captured once and replayed, eager work and other inputs between."""
    x, k = data(40, 300, 'f32', 1).clamp(-3, 3), data(300, 50, 'f32', 2).clamp(-3, 3)
    w = fp8.quantize_cols(k)
    xs, ks = x.clone().requires_grad_(True), k.clone().requires_grad_(True)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        torch.autograd.grad(fp8.linear(xs, ks), (xs, ks), torch.ones(40, 50, device='cuda'))
        fp8.dense(xs.detach()[:3], w), fp8.dense(xs.detach(), w)
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    one = torch.ones(40, 50, device='cuda')
    with torch.cuda.graph(g):
        few, many = fp8.dense(xs.detach()[:3], w), fp8.dense(xs.detach(), w)
        y = fp8.linear(xs, ks)
        dx, dk = torch.autograd.grad(y, (xs, ks), one)
    for i in range(3):
        with torch.no_grad():
            xs.copy_(x * (i + 1))
        g.replay()
        torch.cuda.synchronize()
        xe, ke = (x * (i + 1)).requires_grad_(True), k.clone().requires_grad_(True)
        ye = fp8.linear(xe, ke)
        de = torch.autograd.grad(ye, (xe, ke), one)
        assert torch.equal(y, ye) and torch.equal(dx, de[0]) and torch.equal(dk, de[1])
        assert torch.equal(few, fp8.dense(xe.detach()[:3], w)) and torch.equal(many, fp8.dense(xe.detach(), w))


def test_offsets_beyond_32_bits(fp8):
    """4.6 G values: the last rows and columns as if they were quantised and multiplied alone."""
    n, k = 70016, 65536
    src = torch.empty((n, k), dtype=torch.bfloat16, device='cuda').normal_(generator=torch.Generator('cuda').manual_seed(1))
    w, tail = fp8.quantize_rows(src), fp8.quantize_rows(src[-128:])
    assert torch.equal(w.data[-128:].view(torch.uint8), tail.data.view(torch.uint8)) and torch.equal(w.scale[:, -128:], tail.scale)
    x = torch.randn(300, k, generator=torch.Generator('cuda').manual_seed(2), device='cuda')
    for rows in (3, 300):
        a, b = fp8.dense(x[:rows], w)[:, -128:], fp8.dense(x[:rows], tail)
        # the same exact products in another order: on either side K additions, each off by 2^-24 of a partial sum, which for
        # independent terms is no larger in norm than the whole sum
        assert float((a - b).norm()) <= 2 * k * 2.0 ** -24 * float(b.norm())
    del w
    t, last = fp8.quantize_cols(src), fp8.quantize_cols(src[:, -64:])
    assert torch.equal(t.data[-64:].view(torch.uint8), last.data.view(torch.uint8)) and torch.equal(t.scale[:, -64:], last.scale)


def test_work_on_another_stream(fp8):
    x, w = data(100, 2000, 'f32', 1).clamp(-3, 3), fp8.quantize_rows(data(300, 2000, 'f32', 2).clamp(-3, 3))
    want = fp8.dense(x, w)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = [fp8.dense(x, w) for _ in range(3)] + [fp8.dense(x[:5], w)]
    s.synchronize()
    assert all(torch.equal(g, want) for g in got[:3])
    assert torch.equal(got[3], fp8.dense(x[:5], w))


def test_refusals(fp8):
    x = torch.zeros(4, 130, device='cuda')
    w = fp8.quantize_rows(torch.ones(8, 130, device='cuda'))
    for bad in (lambda: fp8.dense(x[:, :129], w), lambda: fp8.dense(x.half(), w), lambda: fp8.dense(x, w, torch.zeros(7, device='cuda')),
                lambda: fp8.dense(x, w, torch.zeros(8, device='cuda').double()), lambda: fp8.dense(x, w, out_dtype=torch.float16),
                lambda: fp8.product(w, fp8.quantize_rows(x[:, :100])), lambda: fp8.linear(x, torch.zeros(131, 4, device='cuda')),
                lambda: fp8.Fp8Rows(w.data, w.scale[:1], 130), lambda: fp8.Fp8Rows(w.data, w.scale, 100)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(L.C1VError):
        fp8.quantize_rows(torch.zeros(3, 4))


# ---------------------------------------------------------------------------------------------------------------
# operands and sums
# ---------------------------------------------------------------------------------------------------------------
def cancelling(m, n, k, seed):
    """Whole numbers a [m, k], b [n, k] that the quantiser leaves as they are (blocks whose largest value is 448, or 3 at most): in
    every block of 128 two columns hold 448 * 448 and -448 * 448, which cancel, and the others products of at most 9.  Every
    partial sum, in any order, is a whole number below 64 * 448^2 < 2^24 for k <= 8192 (or within half of that, 2 * 9 * k, of
    it), so that fp32 sums are exact; a sum in fewer than 18 bits loses what is left."""
    rng = np.random.RandomState(seed)
    a, b = rng.randint(-3, 4, (m, k)).astype(np.float32), rng.randint(-3, 4, (n, k)).astype(np.float32)
    for kb in range(0, k, 128):
        w = min(128, k - kb)
        if w > 1:
            i, j = kb + rng.choice(w, 2, replace=False)
            a[:, i] = a[:, j] = 448.0
            b[:, i], b[:, j] = 448.0, -448.0
    want = (a.astype(np.float64) @ b.astype(np.float64).T) if m * n * k < 1 << 31 else None
    a, b = torch.from_numpy(a).cuda(), torch.from_numpy(b).cuda()
    return a, b, a.double() @ b.double().t() if want is None else torch.from_numpy(want).cuda()


@pytest.mark.parametrize('kind', ['f32', 'bf16'])
@pytest.mark.parametrize('n', [1288, 1304, 1336, 1400, 4104, 4232, 4312])
def test_right_edges_that_part_the_waves_of_a_workgroup(fp8, kind, n):
    """Rows on 16-byte boundaries whose last tile some waves cover whole, some in part and some not at all (128 x 128 and
    256 x 256 tiles); nothing is written behind the last row."""
    m, k = (2048 if n < 4000 else 4300), 140
    a, b, want = cancelling(m, n, k, n)
    assert torch.equal(fp8.product(fp8.quantize_rows(a), fp8.quantize_rows(b), out_dtype=torch.float32), want.float())
    y = torch.zeros(m + 1, n, dtype=KIND[kind], device='cuda')
    qa, qb = fp8.quantize_rows(torch.ones(m, k, device='cuda')), fp8.quantize_rows(torch.ones(n, k, device='cuda'))
    fp8._call('c1v_fp8_gemm', fp8._PRODUCT(qa.data.data_ptr(), qa.scale.data_ptr(), qb.data.data_ptr(), qb.scale.data_ptr(), m, n, 256, 0, 0,
                                           fp8._CODE[KIND[kind]], y.data_ptr(), n, 0, 0), 0)
    assert (y[:m] == k).all() and not y[m].any()


# up to 16 rows (one and two column fragments a workgroup), short batches (one, two, four), 64 x 64 tiles, a K in runs, 128 x 128
# and 256 x 256 tiles on and off 16-byte boundaries
SUMS = [(1, 1024, 1024), (13, 8192, 1024), (64, 512, 1920), (256, 512, 1920), (512, 512, 512), (1999, 1021, 302), (1024, 1024, 1024),
        (512, 512, 8192), (66, 130, 4352), (2048, 2048, 640), (2050, 1301, 300), (4352, 4096, 384), (4100, 4401, 330)]


@pytest.mark.parametrize('kind', ['f32', 'bf16'])
@pytest.mark.parametrize('m,n,k', SUMS)
def test_sums_are_fp32_whatever_the_output_type(fp8, kind, m, n, k):
    a, b, want = cancelling(m, n, k, m + n)
    want = want.float().to(KIND[kind])
    qa, qb = fp8.quantize_rows(a), fp8.quantize_rows(b)
    assert torch.equal(qa.dequantize(), a) and torch.equal(qb.dequantize(), b)
    assert torch.equal(fp8.product(qa, qb, out_dtype=KIND[kind]), want)
    for x in (a, a.bfloat16()):
        assert torch.equal(fp8.dense(x, qb, out_dtype=KIND[kind]), want)


@pytest.mark.parametrize('kind', ['f32', 'bf16'])
@pytest.mark.parametrize('m,n,k', [(300, 200, 140), (130, 66, 4300), (2050, 1301, 300), (4352, 4096, 384)])
def test_sums_of_a_layer_and_its_gradients_are_fp32(fp8, kind, m, n, k):
    """Each of the three products by itself as the one that cancels (in a small layer both gradients share a launch)."""
    a, b, want = cancelling(m, n, k, m + n + 1)
    t = KIND[kind]
    want = want.float().to(t)
    a, b = a.to(t), b.to(t)
    with torch.no_grad():
        assert torch.equal(fp8.linear(a, b.t()), want)                                          # y = x W
    for other in (False, True):
        x, w = torch.ones(m, n, dtype=t, device='cuda').requires_grad_(True), b.t().contiguous().t().requires_grad_(other)
        dx = torch.autograd.grad(fp8.linear(x, w), x, a, retain_graph=True)[0]                   # dx = dy W^T
        assert torch.equal(dx, want)
        x, w = a.t().contiguous().requires_grad_(other), torch.ones(m, n, dtype=t, device='cuda').requires_grad_(True)
        dw = torch.autograd.grad(fp8.linear(x, w), w, b.t().contiguous())[0]                     # dW = x^T dy
        assert torch.equal(dw, want)


@pytest.mark.parametrize('kind', ['f32', 'bf16'])
@pytest.mark.parametrize('rows,k,n', [(4100, 60, 4200), (2304, 1408, 1900), (4500, 4400, 520)])
def test_linear_of_large_layers(fp8, kind, rows, k, n):
    """Both gradients with a K in runs (one workspace), and through the larger tiles, against 64 bits: K * 2^-24 of the sum of
    magnitudes and half a step of the output type."""
    x, w = data(rows, k, kind, 1).clamp(-3, 3).requires_grad_(True), data(k, n, 'f32', 2).clamp(-3, 3).requires_grad_(True)
    bias = torch.linspace(-1, 1, n, device='cuda').requires_grad_(True)
    dy = data(rows, n, kind, 3).clamp(-3, 3)
    y = fp8.linear(x, w, bias)
    dx, dw, db = torch.autograd.grad(y, (x, w, bias), dy)
    x, w, bias = x.detach(), w.detach(), bias.detach().double()
    deq = lambda q: q.dequantize().double()
    for got, a, b, add in ((y, fp8.quantize_rows(x), fp8.quantize_cols(w), bias), (dx, fp8.quantize_rows(dy), fp8.quantize_rows(w), None),
                           (dw, fp8.quantize_cols(x), fp8.quantize_cols(dy), None)):
        A, B = deq(a), deq(b)
        want, size = A @ B.t(), A.abs() @ B.abs().t()
        if add is not None:
            want, size = want + add, size + add.abs()
        half = 2.0 ** -24 if got.dtype == torch.float32 else 2.0 ** -8
        assert ((got.double() - want).abs() <= half * want.abs() + (A.shape[1] + 2) * 2.0 ** -24 * size * (1 + half)).all()
    D = dy.double()
    assert ((db.double() - D.sum(0)).abs() <= rows * 2.0 ** -24 * D.abs().sum(0)).all()


def test_operands_at_any_strides(fp8):
    """Values and scales as a transposition or a slice leaves them: the constructor lays them out once."""
    x = data(32, 300, 'f32', 1).clamp(-3, 3)
    w = fp8.quantize_rows(data(48, 300, 'f32', 2).clamp(-3, 3))
    want = fp8.dense(x, w)
    scale = w.scale.t().contiguous().t()
    wide = torch.zeros(48, 400, dtype=torch.uint8, device='cuda')
    wide[:, :384] = w.data.view(torch.uint8)
    values = wide.view(torch.float8_e4m3fn)[:, :384]
    assert not scale.is_contiguous() and not values.is_contiguous()
    for v in (fp8.Fp8Rows(w.data, scale, 300), fp8.Fp8Rows(values, w.scale, 300), fp8.Fp8Rows(values, scale, 300)):
        assert torch.equal(fp8.dense(x, v), want) and torch.equal(fp8.dense(x[:3], v), fp8.dense(x[:3], w))
        assert torch.equal(fp8.product(fp8.quantize_rows(x), v), fp8.product(fp8.quantize_rows(x), w))
        assert torch.equal(v.dequantize(), w.dequantize())


def test_products_without_a_gradient_are_refused_where_one_is_asked_for(fp8):
    x, w, b = torch.randn(5, 130, device='cuda'), fp8.quantize_rows(torch.randn(8, 130, device='cuda')), torch.zeros(8, device='cuda')
    xg, bg = x.clone().requires_grad_(True), b.clone().requires_grad_(True)
    for bad in (lambda: fp8.dense(xg, w), lambda: fp8.dense(x, w, bg), lambda: fp8.product(fp8.quantize_rows(x), w, bg)):
        with pytest.raises(ValueError, match='gradient'):
            bad()
    with torch.no_grad():
        assert torch.equal(fp8.dense(xg, w, bg), fp8.dense(x, w, b))
    assert torch.equal(fp8.dense(xg.detach(), w, bg.detach()), fp8.dense(x, w, b))


@pytest.mark.parametrize('m', [1, 16, 33])
@pytest.mark.parametrize('n', [1360, 1376, 2736, 4096, 4097, 8192, 8200])
def test_column_fragments_of_a_served_product(fp8, m, n):
    """One, two and four fragments a workgroup on both sides of their borders, with bias, at a K whose last block is not whole."""
    a, b, want = cancelling(m, n, 300, m + n)
    bias = torch.from_numpy(np.random.RandomState(n).randint(-9, 10, n).astype(np.float32)).cuda()
    for x in (a, a.bfloat16()):
        assert torch.equal(fp8.dense(x, fp8.quantize_rows(b), bias, out_dtype=torch.float32), (want + bias).float())


@pytest.mark.parametrize('m,n,k', [(512, 512, 3968), (512, 512, 4096), (66, 130, 3970), (640, 770, 3968), (640, 770, 4096), (640, 900, 4096)])
def test_a_k_in_runs_on_both_sides_of_its_borders(fp8, m, n, k):
    a, b, want = cancelling(m, n, k, m + k)
    qa, qb = fp8.quantize_rows(a), fp8.quantize_rows(b)
    for t in KIND.values():
        assert torch.equal(fp8.product(qa, qb, out_dtype=t), want.float().to(t))


@pytest.mark.parametrize('m,n', [(5, 300), (100, 200), (700, 900), (2050, 1300), (4352, 4096)])
def test_sums_hold_24_bits(fp8, m, n):
    """One block of K: 448 * 448 and -448 * 448 beside products that are multiples of 2^-6.  Every partial sum, in any order, is a
    multiple of 2^-6 below 2^18, 24 bits, so fp32 sums are exact and anything shorter is not."""
    rng = np.random.RandomState(m)
    a, b = rng.randint(-3, 4, (m, 128)) / 8.0, rng.randint(-3, 4, (n, 128)) / 8.0
    i, j = rng.choice(128, 2, replace=False)
    a[:, i] = a[:, j] = b[:, i] = 448.0
    b[:, j] = -448.0
    a, b = torch.from_numpy(a.astype(np.float32)).cuda(), torch.from_numpy(b.astype(np.float32)).cuda()
    want = (a.double() @ b.double().t()).float()
    qa, qb = fp8.quantize_rows(a), fp8.quantize_rows(b)
    assert torch.equal(qa.dequantize(), a) and torch.equal(qb.dequantize(), b)
    assert torch.equal(fp8.product(qa, qb), want) and torch.equal(fp8.dense(a, qb), want)
    assert torch.equal(fp8.product(qa, qb, out_dtype=torch.bfloat16), want.bfloat16())
