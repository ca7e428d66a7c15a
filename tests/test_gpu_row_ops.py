"""GPU: the row operators against their 64-bit forms (tests/row_reference.py): gradient norm and
clip over many tensors, RMS norm with residual (forward, backward, 8-bit output), 8-bit rows with
block scales and their product.  Tolerances count roundings: half a step of the stored type for each
store, 2^-24 for each fp32 operation on the longest chain that a result goes through."""
import math

import pytest
import torch

import row_reference as ref
from objectdetection_amd import ops

pytestmark = pytest.mark.gpu

F32 = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
E4M3, E5M2 = torch.float8_e4m3fn, torch.float8_e5m2


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _rows(seed, r, c, dtype=torch.float32, size=1.0):
    g = _gen(seed)
    x = torch.randn((r, c), generator=g) * torch.exp(torch.randn((1, c), generator=g)) * size
    return (x * (torch.rand((r, c), generator=g) > 0.1)).to(dtype)


def _within(got, want, bound, what=""):
    """|got - want| <= bound, elementwise (64 bits), with equal NaN and infinities."""
    got, want = got.detach().double().cpu(), want.double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    odd = ~torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    assert torch.equal(got[odd & ~torch.isnan(want)], want[odd & ~torch.isnan(want)]), what
    over = ((got - want).abs() - bound)[~odd]
    assert over.numel() == 0 or over.max() <= 0, (what, over.max().item(), (got - want)[~odd].abs().max().item())


# ------------------------------------------------------------------ 8-bit rows

QSHAPES = [(1, 1), (1, 128), (3, 5), (7, 16), (5, 31), (2, 33), (130, 64), (127, 127), (128, 128), (129, 257),
           (1, 4096), (300, 1000), (16, 777)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", QSHAPES)
def test_f8_forms_equal_their_definition(cuda, shape, dtype):
    x = _rows(1, *shape, dtype)
    d = x.to(cuda)
    for f8 in (E4M3, E5M2):
        want = ref.quantise(x, f8)
        want_t = ref.quantise(x.t(), f8)
        for got, (q, e) in zip((ops.f8_rows(d, f8), ops.f8_cols(d, f8), *ops.f8_rows_cols(d, f8)),
                               (want, want_t, want, want_t)):
            assert got.data.dtype == f8 and got.data.shape == q.shape
            assert torch.equal(got.data.cpu().double(), q)
            assert torch.equal(got.scale.cpu().view(torch.uint8).int() - 127, e.int())
        q, e = ref.quantise(x, f8, 128)
        for got, (q, e) in ((ops.f8_weight_image(d, dtype=f8), (q, e)),
                            (ops.f8_weight_image(d, True, f8), (q.t(), e.t()))):
            assert torch.equal(got.data.cpu().double(), q)
            assert torch.equal(got.scale.cpu().view(torch.uint8).int() - 127, e.int())


def test_f8_padding_is_zero_and_rows_start_on_borders(cuda):
    x = _rows(2, 9, 150).to(cuda)
    for got in (ops.f8_rows(x), ops.f8_cols(x), ops.f8_weight_image(x)):
        ld, lds = got.data.stride(0), got.scale.stride(0)
        assert ld % 16 == 0 and lds % 4 == 0 and got.data.data_ptr() % 16 == 0
        R, C = got.data.shape
        whole = got.data.view(torch.uint8).as_strided((R, ld), (ld, 1))
        assert int(whole[:, C:].sum()) == 0
        s = got.scale.view(torch.uint8).as_strided((got.scale.shape[0], lds), (lds, 1))
        assert int(s[:, got.scale.shape[1]:].sum()) == 0


def test_f8_extremes(cuda):
    """Zero blocks, the smallest and largest magnitudes, exact format limits, infinities, NaN."""
    inf, nan = float("inf"), float("nan")
    rows = [[0.0] * 6, [1e-45, 1e-40, 2e-38, 0.0, -1e-44, 1e-45], [3.4e38, -3.4e38, 1.0, 0.0, 1e30, 2e38],
            [448.0, -448.0, 17.0, 18.0, 19.0, 2.0 ** -9], [448.5, 1.0, 0.1, 3.0, 5.0, 7.0],
            [inf, 1.0, -2.0, nan, 0.5, -inf], [nan] * 6, [57344.0, 57345.0, 1.0, 2.0, 3.0, 4.0]]
    x = torch.tensor(rows, dtype=torch.float32)
    for f8 in (E4M3, E5M2):
        q, e = ref.quantise(x, f8)
        got = ops.f8_rows(x.to(cuda), f8)
        assert torch.equal(got.scale.cpu().view(torch.uint8).int() - 127, e.int())
        g = got.data.cpu().double()
        assert torch.equal(torch.isnan(g), torch.isnan(q))
        assert torch.equal(g.nan_to_num(0.0), q.nan_to_num(0.0))


def test_f8_takes_strided_rows(cuda):
    big = _rows(3, 40, 300).to(cuda)
    for x in (big[:, 7:140], big[::2, 1:100], big.t()[3:50], big[5:6, ::2]):
        got = ops.f8_rows(x)
        want = ops.f8_rows(x.contiguous())
        assert torch.equal(got.data.view(torch.uint8), want.data.view(torch.uint8))
        assert torch.equal(got.scale.view(torch.uint8), want.scale.view(torch.uint8))


# ------------------------------------------------------------------ product

def _product_bound(qa, qb, K, y, out_dtype):
    """K products, each exact in fp32, summed in fp32: every addition is off by at most one unit
    (2 * 2^-24; the matrix core need not round to nearest) of what is summed, then one rounding.
    For 16-bit outputs the 8-bit instruction drops what lies 13 bits below the largest of eight
    products: 8 * 2^-13 of that largest one, at most 2^-10 of the sum of magnitudes."""
    low = 0.0 if out_dtype == torch.float32 else 2.0 ** -10
    return (2 * (K + 4) * F32 + low) * (qa.abs() @ qb.abs().t()) + half_step(out_dtype) * y.abs() + 1e-30


half_step = ref.half_step

MSHAPES = [(1, 1, 1), (1, 17, 16), (3, 128, 128), (16, 64, 256), (17, 65, 129), (5, 300, 777), (128, 128, 512),
           (129, 130, 1000), (257, 64, 64), (200, 256, 16), (64, 1000, 31), (2, 2048, 4096), (33, 24, 5000),
           (300, 257, 640), (1000, 16, 100)]


@pytest.mark.parametrize("shape", MSHAPES)
def test_f8_matmul(cuda, shape):
    M, N, K = shape
    a, b = _rows(4, M, K), _rows(5, N, K, size=K ** -0.5)
    for fa, fb, square, out in ((E4M3, E4M3, True, torch.float32), (E4M3, E4M3, False, torch.bfloat16),
                                (E5M2, E4M3, True, torch.float16), (E4M3, E5M2, False, torch.float32),
                                (E5M2, E5M2, False, torch.float32)):
        qa = ref.value(*ref.quantise(a, fa))
        qb = ref.value(*ref.quantise(b, fb, 128 if square else 1), 128 if square else 1)
        want = qa @ qb.t()
        xb = ops.f8_weight_image(b.to(cuda), dtype=fb) if square else ops.f8_rows(b.to(cuda), fb)
        got = ops.f8_matmul(ops.f8_rows(a.to(cuda), fa), xb, out_dtype=out)
        assert got.dtype == out
        _within(got, want, _product_bound(qa, qb, K, want, out), (shape, fa, fb, square))


@pytest.mark.parametrize("shape", [(4096, 1, 16), (4100, 64, 64), (5001, 256, 100), (4097, 130, 256), (4200, 200, 512),
                                   (9000, 65, 129), (4096, 256, 300), (3600, 3500, 330), (3585, 3600, 128)])
def test_f8_matmul_many_rows(cuda, shape):
    """Thin layers over many rows, and outputs of many tiles; a linear layer's one launch gives the
    bits of the two calls."""
    M, N, K = shape
    a, b = _rows(4, M, K), _rows(5, N, K, size=K ** -0.5)
    for fa, fb, square, out in ((E4M3, E4M3, True, torch.float32), (E4M3, E4M3, False, torch.bfloat16),
                                (E5M2, E5M2, True, torch.float16)):
        qa = ref.value(*ref.quantise(a, fa))
        qb = ref.value(*ref.quantise(b, fb, 128 if square else 1), 128 if square else 1)
        want = qa @ qb.t()
        xb = ops.f8_weight_image(b.to(cuda), dtype=fb) if square else ops.f8_rows(b.to(cuda), fb)
        got = ops.f8_matmul(ops.f8_rows(a.to(cuda), fa), xb, out_dtype=out)
        _within(got, want, _product_bound(qa, qb, K, want, out), (shape, fa, fb, square))
    w = ops.f8_weight_image(b.to(cuda))
    shift = torch.randn((N,), generator=_gen(6)).to(cuda)
    for dtype in DTYPES:
        x = torch.nn.functional.pad(a.to(dtype).to(cuda), (1, 2))[:, 1:1 + K]
        want = ops.f8_matmul(ops.f8_rows(x), w, shift=shift, relu=True, out_dtype=dtype)
        assert torch.equal(ops.f8_product(x, w, shift=shift, relu=True), want)


def test_f8_matmul_epilogue_and_out(cuda):
    M, N, K = 70, 150, 200
    a, b = _rows(6, M, K), _rows(7, N, K, size=0.1)
    scale, shift = torch.rand((N,), generator=_gen(8)) + 0.5, torch.randn((N,), generator=_gen(9))
    xa, xb = ops.f8_rows(a.to(cuda)), ops.f8_weight_image(b.to(cuda))
    qa, qb = ref.value(*ref.quantise(a)), ref.value(*ref.quantise(b, h=128), 128)
    y = qa @ qb.t()
    room = torch.full((M, 200), 7.0, device=cuda)
    for s, t, relu in ((scale, shift, True), (None, shift, False), (scale, None, False), (None, None, True)):
        want = y * (1.0 if s is None else s.double()) + (0.0 if t is None else t.double())
        size = y.abs() * (1.0 if s is None else s.double()) + (0.0 if t is None else t.abs().double())
        bound = 2 * _product_bound(qa, qb, K, y, torch.float32) + 3 * F32 * size
        if relu:
            want = want.clamp(min=0.0)
        out = room[:, 20:20 + N]
        got = ops.f8_matmul(xa, xb, None if s is None else s.to(cuda), None if t is None else t.to(cuda), relu,
                            out=out)
        assert got.data_ptr() == out.data_ptr()
        _within(got, want, bound)
        assert bool((room[:, :20] == 7).all()) and bool((room[:, 20 + N:] == 7).all())


@pytest.mark.parametrize("M", [40, 100])
def test_f8_matmul_split_sum_is_repeatable_and_joined(cuda, M):
    """A long sum split over the waves of a workgroup (few rows) and over workgroups (a workspace)."""
    N, K = 64, 70000
    a, b = _rows(10, M, K), _rows(11, N, K)
    assert (ops._lib.lib().lcf_f8_gemm_workspace_bytes(M, N, K, 0) > 0) == (M > 64)
    xa, xb = ops.f8_rows(a.to(cuda)), ops.f8_rows(b.to(cuda))
    qa, qb = ref.value(*ref.quantise(a)), ref.value(*ref.quantise(b))
    bias = torch.randn((N,), generator=_gen(12)).to(cuda)
    got = [ops.f8_matmul(xa, xb, shift=bias, relu=True) for _ in range(3)]
    want = (qa @ qb.t() + bias.double().cpu()).clamp(min=0)
    _within(got[0], want, 2 * (K + 4) * F32 * (qa.abs() @ qb.abs().t()))
    assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(100, 64, 9000), (100, 300, 6000), (70, 20, 5005), (300, 40, 4100)])
def test_f8_matmul_split_sums_of_every_type(cuda, shape, dtype):
    M, N, K = shape
    assert ops._lib.lib().lcf_f8_gemm_workspace_bytes(M, N, K, ops._TYPE_CODE[dtype]) > 0
    a, b = _rows(13, M, K), _rows(14, N, K, size=K ** -0.5)
    scale, shift = torch.rand((N,), generator=_gen(15)) + 0.5, torch.randn((N,), generator=_gen(16))
    qa, qb = ref.value(*ref.quantise(a)), ref.value(*ref.quantise(b, h=128), 128)
    y = qa @ qb.t()
    got = ops.f8_matmul(ops.f8_rows(a.to(cuda)), ops.f8_weight_image(b.to(cuda)), scale.to(cuda), shift.to(cuda), True,
                        dtype)
    want = (y * scale.double() + shift.double()).clamp(min=0)
    bound = scale.double() * _product_bound(qa, qb, K, y, torch.float32 if dtype == torch.float32 else dtype)
    _within(got, want, bound + 4 * F32 * (y.abs() * scale.double() + shift.double().abs())
            + half_step(dtype) * want * 1.01 + tiny(dtype))


def test_f8_matmul_empty_sizes(cuda):
    a = ops.f8_rows(torch.zeros((0, 40), device=cuda))
    b = ops.f8_weight_image(_rows(13, 8, 40).to(cuda))
    assert ops.f8_matmul(a, b).shape == (0, 8)
    a, b = ops.f8_rows(torch.zeros((3, 0), device=cuda)), ops.f8_weight_image(torch.zeros((8, 0), device=cuda))
    shift = torch.arange(8.0, device=cuda) - 4
    assert torch.equal(ops.f8_matmul(a, b, shift=shift, relu=True), shift.clamp(min=0).expand(3, 8))
    assert ops.f8_matmul(ops.f8_rows(_rows(14, 3, 40).to(cuda)),
                         ops.f8_weight_image(torch.zeros((0, 40), device=cuda))).shape == (3, 0)


def test_f8_matmul_ignores_what_lies_behind_the_last_column(cuda):
    """Views into wider 8-bit matrices, with NaN bytes right behind the columns that take part."""
    M, N, K = 20, 30, 100
    a, b = _rows(15, M, K), _rows(16, N, K)
    xa, xb = ops.f8_rows(a.to(cuda)), ops.f8_rows(b.to(cuda))
    want = ops.f8_matmul(xa, xb)
    wide = []
    for x in (xa, xb):
        room = torch.full((x.data.shape[0], 256), 0x7F, dtype=torch.uint8, device=cuda)
        room[:, :K] = x.data.view(torch.uint8)
        wide.append(ops.F8Rows(room.view(E4M3)[:, :K], x.scale))
    assert torch.equal(ops.f8_matmul(*wide), want)
    # rows and scales of a caller's own making: tight, odd strides, any start
    tight = [ops.F8Rows(x.data.contiguous().clone(), x.scale.contiguous().view(torch.uint8)) for x in (xa, xb)]
    assert torch.equal(ops.f8_matmul(*tight), want)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 16, 16), (50, 64, 256), (700, 256, 64), (300, 100, 37), (129, 1, 130),
                                   (4500, 256, 64), (4099, 64, 200), (4200, 300, 520)])
def test_f8_linear_forward_and_gradients(cuda, shape, dtype):
    M, N, K = shape
    x = _rows(17, M, K, dtype).to(cuda).requires_grad_(True)
    w = _rows(18, N, K, size=K ** -0.5).to(cuda).requires_grad_(True)
    bias = torch.randn((N,), generator=_gen(19)).to(cuda).requires_grad_(True)
    dy = _rows(20, M, N, dtype, 1e-2)
    y = ops.f8_linear(x, w, bias)
    dx, dw, db = torch.autograd.grad(y, (x, w, bias), dy.to(cuda))
    x8 = ref.value(*ref.quantise(x.detach()))
    w8 = ref.value(*ref.quantise(w.detach(), h=128), 128)
    want = x8 @ w8.t()
    _within(y, want + bias.detach().double().cpu(), 2 * _product_bound(x8, w8, K, want, dtype)
            + 2 * half_step(dtype) * (bias.detach().double().cpu().abs() + want.abs()) + tiny(dtype), "y")
    d8 = ref.value(*ref.quantise(dy))
    want = d8 @ w8
    _within(dx, want, _product_bound(d8, w8.t(), N, want, dtype) + tiny(dtype), "dx")
    dt, xt = ref.value(*ref.quantise(dy.t())), ref.value(*ref.quantise(x.detach().t()))
    want = dt @ xt.t()
    _within(dw, want, _product_bound(dt, xt, M, want, torch.float32), "dw")
    want = dy.double().sum(0)
    _within(db, want, (M + 2) * F32 * dy.double().abs().sum(0), "db")


def tiny(dtype):
    """Half of the least step of a type: what a subnormal result may be off by."""
    return 0.5 * {torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133, torch.float32: 2.0 ** -149}[dtype]


# ------------------------------------------------------------------ RMS norm

NSHAPES = [(1, 1), (3, 5), (1, 16), (70, 17), (33, 31), (65, 64), (40, 100), (9, 128), (50, 130), (21, 256),
           (7, 500), (6, 513), (5, 1024), (4, 1500), (3, 2048), (2, 3001), (3, 4096), (2, 5001), (2, 8192), (2, 16384)]


def _chain(width):
    """fp32 operations that a row's sum goes through: eight columns of up to four pieces a lane, at
    most ten lane or wave steps, then mean, root and division."""
    return 8 * 4 + 10 + 16 + 6


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", NSHAPES)
def test_rms_norm_forward(cuda, shape, dtype):
    R, C = shape
    x, r = _rows(21, R, C, dtype), _rows(22, R, C, dtype)
    w = (1.0 + 0.2 * torch.randn((C,), generator=_gen(23)))
    eps = 1e-6
    for weight, residual in ((w, r), (w.to(dtype), None), (None, r), (None, None)):
        y, h, _ = ref.rms_norm(x, weight, eps, residual)
        got = ops.rms_norm(x.to(cuda), None if weight is None else weight.to(cuda), eps,
                           None if residual is None else residual.to(cuda))
        if residual is not None:
            got, gh = got
            assert gh.dtype == dtype and torch.equal(gh.double().cpu(), h)
        assert got.dtype == dtype
        _within(got, y, (_chain(C) * F32 + half_step(dtype)) * 1.001 * y.abs() + tiny(dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", NSHAPES)
def test_rms_norm_to_8_bit_rows(cuda, shape, dtype):
    """Values within what the norm's own rounding may move across a rounding border: q differs from
    the definition's by one step at most, and only where the exact value lies on a border."""
    R, C = shape
    x, r = _rows(24, R, C, dtype), _rows(25, R, C, dtype)
    w = (1.0 + 0.2 * torch.randn((C,), generator=_gen(26)))
    for f8 in (E4M3, E5M2):
        y, h, _ = ref.rms_norm(x, w, 1e-6, r)
        got, gh = ops.rms_norm_f8(x.to(cuda), w.to(cuda), 1e-6, r.to(cuda), f8)
        assert torch.equal(gh.double().cpu(), h)
        s = got.scale.cpu().view(torch.uint8).int() - 127
        g = ref.value(got.data.cpu(), s)
        top = torch.nn.functional.pad(y.abs(), (0, -C % 128)).view(R, -1, 128).amax(2)
        near = 1.0 + _chain(C) * F32 * 1.001
        least = ref._scale_exponent(top / near, f8)
        most = ref._scale_exponent(top * near, f8)
        assert bool(((s >= least) & (s <= most)).all())
        # half a step of the format at y's size, and the norm's rounding
        bits, low = ref.LEAST8[f8][1], ref.LEAST8[f8][0]
        unit = ref.two(s).repeat_interleave(128, 1)[:, :C]
        step = torch.maximum(y.abs() * near * 2.0 ** -bits, unit * 2.0 ** (low - bits))
        _within(g, y, 0.5 * step + _chain(C) * F32 * 1.001 * y.abs())
        share = (got.data.cpu().double() != ref.quantise(y, f8)[0]).double().mean()
        assert share <= max(2.0 / y.numel(), 1e-3)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", NSHAPES + [(3000, 64), (2500, 20)])
def test_rms_norm_backward(cuda, shape, dtype):
    R, C = shape
    x, r = _rows(27, R, C, dtype), _rows(28, R, C, dtype)
    w = (1.0 + 0.2 * torch.randn((C,), generator=_gen(29)))
    dy, dh = _rows(30, R, C, dtype), _rows(31, R, C, dtype)
    xs, rs = x.to(cuda).requires_grad_(True), r.to(cuda).requires_grad_(True)
    ws = w.to(cuda).requires_grad_(True)
    y, h = ops.rms_norm(xs, ws, 1e-6, rs)
    dx, dr, dw = torch.autograd.grad((y, h), (xs, rs, ws), (dy.to(cuda), dh.to(cuda)))
    assert torch.equal(dx, dr)
    _, hh, inv = ref.rms_norm(x, w, 1e-6, r)
    want, want_w = ref.rms_norm_bwd(hh, w, inv, dy, dh)
    g = dy.double() * w.double()
    size = inv * (g.abs() + hh.abs() * inv ** 2 * (g * hh).abs().mean(1, keepdim=True)) + dh.double().abs()
    _within(dx, want, 3 * _chain(C) * F32 * size + half_step(dtype) * want.abs() * 1.001 + tiny(dtype), "dx")
    lines = (dy.double() * hh * inv).abs().sum(0)
    _within(dw, want_w, (_chain(C) + 128 + 8) * F32 * lines + 1e-30, "dw")
    # without the sum's gradient, without a weight, without a residual
    y = ops.rms_norm(xs, None, 1e-6)
    (dx,) = torch.autograd.grad(y, (xs,), dy.to(cuda))
    _, hh, inv = ref.rms_norm(x, None, 1e-6)
    want, _ = ref.rms_norm_bwd(hh, None, inv, dy)
    size = inv * (dy.double().abs() + hh.abs() * inv ** 2 * (dy.double() * hh).abs().mean(1, keepdim=True))
    _within(dx, want, 3 * _chain(C) * F32 * size + half_step(dtype) * want.abs() * 1.001 + tiny(dtype), "dx alone")


def test_rms_norm_gradient_against_differences(cuda):
    """The formula itself, by central differences of the 64-bit forward."""
    x, w, dy = _rows(32, 4, 12), 1.0 + 0.1 * torch.randn((12,), generator=_gen(33)), _rows(34, 4, 12)
    xs, ws = x.to(cuda).requires_grad_(True), w.to(cuda).requires_grad_(True)
    dx, dw = torch.autograd.grad(ops.rms_norm(xs, ws, 1e-3), (xs, ws), dy.to(cuda))

    def f(x, w):
        return (ref.rms_norm(x, w, 1e-3)[0] * dy.double()).sum()
    step = 1e-5
    for got, at in ((dx, 0), (dw, 1)):
        base = [x.double(), w.double()]
        want = torch.zeros_like(base[at]).reshape(-1)
        for i in range(want.numel()):
            d = torch.zeros_like(base[at]).reshape(-1)
            d[i] = step
            d = d.view_as(base[at])
            hi, lo = list(base), list(base)
            hi[at], lo[at] = base[at] + d, base[at] - d
            want[i] = (f(*hi) - f(*lo)) / (2 * step)
        _within(got, want.view_as(base[at]), 1e-5 * want.abs().max())


def test_rms_norm_rows_of_zeros_infinities_and_strides(cuda):
    x = _rows(35, 6, 40)
    x[1] = 0.0
    x[2, 3] = float("inf")
    x[3, 5] = float("nan")
    w = torch.ones((40,))
    y, _, _ = ref.rms_norm(x, w, 1e-6)
    got = ops.rms_norm(x.to(cuda), w.to(cuda), 1e-6)
    _within(got, y, _chain(40) * F32 * y.abs().nan_to_num(0.0) + 1e-30)
    assert bool((got[1] == 0).all())
    big = _rows(36, 30, 200).to(cuda)
    for v in (big[:, 3:133], big[::3, 1:65], big.t()[2:9, :], big.view(5, 6, 200)):
        assert torch.equal(ops.rms_norm(v, None, 1e-6), ops.rms_norm(v.contiguous(), None, 1e-6))
    assert ops.rms_norm(big[:0], None).shape == (0, 200)
    e = big[:0].clone().requires_grad_(True)
    ww = torch.ones((200,), device=cuda, requires_grad=True)
    gx, gw = torch.autograd.grad(ops.rms_norm(e, ww).sum(), (e, ww))
    assert gx.shape == (0, 200) and bool((gw == 0).all())


# ------------------------------------------------------------------ gradient norm, clip

def _grads(seed, dtypes, n=40, most=30000):
    g = _gen(seed)
    out = []
    for i in range(n):
        size = int(math.exp(torch.rand((), generator=g).item() * math.log(most)))
        out.append((torch.randn((size,), generator=g) * 3).to(dtypes[i % len(dtypes)]))
    return out


@pytest.mark.parametrize("p", [1.0, 2.0, float("inf")])
@pytest.mark.parametrize("dtypes", [[torch.float32], [torch.bfloat16], DTYPES])
def test_grad_norm_and_clip(cuda, dtypes, p):
    for n in (1, 2, 40, 300):
        grads = _grads(40 + n, dtypes, n)
        for max_norm in (1.0, 1e9):
            total, want = ref.clip(grads, max_norm, p)
            d = [g.to(cuda) for g in grads]
            keep = [g.clone() for g in d]
            _within(ops.grad_norm(d, p), total, 2 * F32 * total)
            flat = torch.empty((sum(g.numel() for g in d),), device=cuda)
            _within(ops.clip_norm_(d, max_norm, p, out=flat), total, 2 * F32 * total)
            assert all(torch.equal(a, b) for a, b in zip(d, keep))
            _within(flat, torch.cat([x.reshape(-1) for x in want]),
                    6 * F32 * torch.cat([x.abs().reshape(-1) for x in want]) + 2.0 ** -149)
            outs = [torch.empty(g.shape, dtype=torch.bfloat16, device=cuda) for g in d]
            ops.clip_norm_(d, max_norm, p, out=outs)
            assert ops.clip_norm_(d, max_norm, p).shape == ()
            for g, o, w in zip(d, outs, want):
                _within(o, w, (half_step(torch.bfloat16) + 6 * F32) * w.abs() * 1.001 + tiny(torch.bfloat16))
                _within(g, w, (half_step(g.dtype) + 6 * F32) * w.abs() * 1.001 + tiny(g.dtype))


def test_grad_norm_range_odd_starts_and_order(cuda):
    # squares of these leave fp32 at both ends
    for v in (1e-30, 1e30):
        g = torch.full((5000,), v, device=cuda)
        want = math.sqrt(5000.0) * float(g[0].double())
        assert abs(ops.grad_norm([g]).item() / want - 1) <= 2 * F32 * 1.001
    flat = torch.randn((50021,), generator=_gen(50)).to(cuda)
    half = flat.bfloat16()
    parts = [flat[1:8], flat[9:20010], half[3:3], half[5:40004], flat[20011:20012], flat[30001:]]
    total, want = ref.clip(parts, 2.5)
    _within(ops.grad_norm(parts), total, 2 * F32 * total)
    before = flat.clone()
    ops.clip_norm_(parts, 2.5)
    for g, w in zip(parts, want):
        _within(g, w, (half_step(g.dtype) + 6 * F32) * w.abs() * 1.001 + tiny(g.dtype))
    for i in (0, 8, 20010, 30000):  # what lies between stays
        assert flat[i] == before[i]
    # dense in another order: channels_last
    c = torch.randn((4, 6, 5, 3), generator=_gen(51)).to(cuda).to(memory_format=torch.channels_last)
    total, want = ref.clip([c], 1.0)
    ops.clip_norm_([c], 1.0)
    _within(c, want[0], 8 * F32 * want[0].abs())


def test_grad_norm_of_what_is_not_finite(cuda):
    inf, nan = float("inf"), float("nan")
    for bad, p in ((inf, 2.0), (nan, 2.0), (nan, inf), (-inf, 1.0), (nan, 1.0)):
        g = [torch.ones((10,), device=cuda), torch.tensor([1.0, bad, 2.0], device=cuda)]
        t = [torch.nn.Parameter(torch.zeros_like(x)) for x in g]
        for a, b in zip(t, g):
            a.grad = b.clone()
        want = torch.nn.utils.clip_grad_norm_(t, 1.0, p)
        got = ops.clip_norm_(g, 1.0, p)
        assert torch.equal(torch.isnan(got), torch.isnan(want)) and (torch.isnan(got) or got == want)
        for a, b in zip(t, g):
            assert torch.equal(torch.isnan(a.grad), torch.isnan(b))
            assert torch.equal(a.grad.nan_to_num(5.0), b.nan_to_num(5.0))
    assert ops.grad_norm([]).item() == 0.0
    assert ops.grad_norm([torch.zeros((0,), device=cuda)]).item() == 0.0


def test_clip_grad_norm_of_parameters_and_refused_overlaps(cuda):
    ps = [torch.nn.Parameter(torch.randn((5, 7), generator=_gen(60 + i)).to(cuda)) for i in range(4)]
    qs = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    for p, q in list(zip(ps, qs))[:3]:
        p.grad = torch.randn((5, 7), generator=_gen(70)).to(cuda)
        q.grad = p.grad.clone()
    a, b = ops.clip_grad_norm_(ps, 0.5), torch.nn.utils.clip_grad_norm_(qs, 0.5)
    assert torch.allclose(a, b, rtol=1e-6) and ps[3].grad is None
    for p, q in list(zip(ps, qs))[:3]:
        assert torch.allclose(p.grad, q.grad, rtol=1e-6, atol=0)
    flat = torch.ones((100,), device=cuda)
    with pytest.raises(RuntimeError):
        ops.clip_norm_([flat[:60], flat[50:]], 1.0)
    with pytest.raises(RuntimeError):
        ops.clip_norm_([flat, flat], 1.0)
    with pytest.raises(RuntimeError):
        ops.clip_norm_([flat[:50]], 1.0, out=flat[10:60])
    assert bool((flat == 1).all())
    assert ops.grad_norm([flat, flat[:50]]).item() == pytest.approx(math.sqrt(150.0))  # reading twice is fine


# ------------------------------------------------------------------ streams, graphs, together

def _tower(x, r, nw, w1, w2, dy):
    h0 = x
    y, h = ops.rms_norm(h0, nw, 1e-6, r)
    out = ops.f8_linear(torch.relu(ops.f8_linear(y, w1)), w2) + h
    grads = torch.autograd.grad(out, (x, nw, w1, w2), dy)
    total = ops.clip_norm_([g.detach() for g in grads], 0.5)
    return (out.detach(), total, *grads)


def test_a_training_step_of_a_pointwise_residual_block(cuda):
    """Norm -> 8-bit product -> ReLU -> 8-bit product -> residual, gradients, clip: one run of the
    operators together against the 64-bit forms with the same roundings passed through."""
    M, C, D = 300, 256, 64
    x, r, dy = _rows(80, M, C), _rows(81, M, C), _rows(82, M, C, size=1e-2)
    nw = 1.0 + 0.1 * torch.randn((C,), generator=_gen(83))
    w1, w2 = _rows(84, D, C, size=C ** -0.5), _rows(85, C, D, size=D ** -0.5)
    leaves = [t.to(cuda).requires_grad_(True) for t in (x, nw, w1, w2)]
    got = _tower(leaves[0], r.to(cuda), *leaves[1:], dy.to(cuda))

    def q(v, h=1):
        return ref.value(*ref.quantise(v.float(), h=h), h)
    y, h, inv = ref.rms_norm(x, nw, 1e-6, r)
    y = y.float()
    p1, p2 = q(w1, 128), q(w2, 128)
    a = (q(y) @ p1.t()).float()
    b = torch.relu(a)
    out = (q(b) @ p2.t()) + h
    d = dy.double()
    dw2 = q(d.t()) @ q(b.t()).t()
    da = (q(d) @ p2).float() * (a > 0)
    dw1 = q(da.t()) @ q(y.t()).t()
    dyy = (q(da) @ p1).float()
    dx, dnw = ref.rms_norm_bwd(h, nw, inv, dyy, dy)
    grads = [dx, dnw, dw1, dw2]
    total, grads = ref.clip(grads, 0.5)
    # fp32 rounding moves a few values across an 8-bit border (one step, 2^-3 of the value, each):
    # with at most one value in a hundred moved the 2-norm is off by 0.1 * 2^-3
    for g, w in zip(got, [out, total, *grads]):
        w = w.double()
        assert (g.double().cpu() - w).norm() <= 0.0125 * w.norm()


def test_on_another_stream_and_captured(cuda):
    M, C, D = 200, 128, 64
    x, r = _rows(90, M, C).to(cuda), _rows(91, M, C).to(cuda)
    w8 = ops.f8_weight_image(_rows(92, D, C, size=0.1).to(cuda))
    big = ops.f8_rows(_rows(93, 100, 40000).to(cuda))
    grads = [t.to(cuda) for t in _grads(94, [torch.float32], 20)]

    wide = ops.f8_rows(_rows(95, 3600, 256).to(cuda))

    def run():
        a8, h = ops.rms_norm_f8(x, None, 1e-6, r)
        y = ops.f8_matmul(a8, w8)
        z = ops.f8_matmul(big, big)  # a split sum: uses a workspace
        t = ops.f8_matmul(wide, wide, out_dtype=torch.bfloat16)  # 256 x 256 tiles
        u = ops.f8_matmul(wide, wide)
        flat = torch.empty((sum(g.numel() for g in grads),), device=cuda)
        total = ops.clip_norm_(grads, 1.0, out=flat)
        return h, y, z, t, u, flat, total
    want = [t.clone() for t in run()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert all(torch.equal(a, b) for a, b in zip(run(), want))
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = run()
        graphs.append((g, out))
    for k in range(3):
        x.mul_(0.5 if k else 2.0)
        for t in grads:
            t.mul_(1.5)
        want = [t.clone() for t in run()]
        for g, out in graphs:
            for t in out:
                t.zero_()
            g.replay()
        torch.cuda.synchronize()
        for g, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, want)), k


def test_empty_rows_broadcast_gradients_and_unused_outputs(cuda):
    """Gradients as autograd hands them over: expanded (a sum's), missing (an output nobody used), of
    rows that are a view; a weight that needs none."""
    x, r = _rows(100, 6, 40).to(cuda), _rows(101, 6, 40).to(cuda)
    w = (1.0 + 0.1 * torch.randn((40,), generator=_gen(102))).to(cuda)
    for use_y, use_h in ((True, False), (False, True), (True, True)):
        a, b, c = (t.clone().requires_grad_(True) for t in (x, r, w))
        y, h = ops.rms_norm(a, c, 1e-6, b)
        loss = (y.sum() if use_y else 0.0) + (3.0 * h.sum() if use_h else 0.0)
        loss.backward()
        _, hh, inv = ref.rms_norm(x, w, 1e-6, r)
        want = torch.zeros((6, 40), dtype=torch.float64)
        if use_y:
            dy = torch.ones((6, 40))
            want, want_w = ref.rms_norm_bwd(hh, w, inv, dy)
            _within(c.grad, want_w, 300 * F32 * (hh * inv).abs().sum(0))
            size = inv * (w.double().cpu().abs() + hh.abs() * inv ** 2
                          * (w.double().cpu() * hh).abs().mean(1, keepdim=True))
        else:
            assert c.grad is None or bool((c.grad == 0).all())
            size = torch.zeros_like(want)
        if use_h:
            want = want + 3.0
        _within(a.grad, want, 3 * _chain(40) * F32 * (size + 3.0))
        assert torch.equal(a.grad, b.grad)
    # one row of x shared by all rows, and a residual that is a view
    row = _rows(103, 1, 40).to(cuda).requires_grad_(True)
    y, h = ops.rms_norm(row.expand(6, 40), w, 1e-6, _rows(104, 6, 80).to(cuda)[:, 40:])
    (g,) = torch.autograd.grad(y.sum() + h.sum(), (row,))
    wide = row.detach().expand(6, 40).contiguous().requires_grad_(True)
    y, h = ops.rms_norm(wide, w, 1e-6, _rows(104, 6, 80).to(cuda)[:, 40:])
    (gw,) = torch.autograd.grad(y.sum() + h.sum(), (wide,))
    assert torch.equal(g, gw.sum(0, keepdim=True))
    # products of nothing
    e = torch.zeros((0, 16), device=cuda, requires_grad=True)
    m = _rows(105, 8, 16).to(cuda).requires_grad_(True)
    bias = torch.zeros((8,), device=cuda, requires_grad=True)
    ge, gm, gb = torch.autograd.grad(ops.f8_linear(e, m, bias).sum(), (e, m, bias))
    assert ge.shape == (0, 16) and bool((gm == 0).all()) and bool((gb == 0).all())
    # leading dimensions, a weight stored [K, N], rows in 8-bit form already, no gradient asked for
    t = _rows(106, 30, 16).to(cuda)
    want = ops.f8_linear(t, m.detach())
    assert torch.equal(ops.f8_linear(t.view(5, 6, 16), m.detach()).view(30, 8), want)
    assert torch.equal(ops.f8_linear(t, m.detach().t().contiguous(), turned=True), want)
    assert torch.equal(ops.f8_linear(t, m.detach(), x8=ops.f8_rows(t)), want)
    with torch.no_grad():
        assert torch.equal(ops.f8_linear(t, m), want)


def test_f8_matmul_into_outputs_that_start_anywhere(cuda):
    """Odd columns of a wider matrix, for few rows, tiles and thin layers over many rows."""
    for M, N, K in ((5, 40, 300), (300, 264, 200), (4100, 64, 96), (4100, 256, 512)):
        a, b = ops.f8_rows(_rows(110, M, K).to(cuda)), ops.f8_weight_image(_rows(111, N, K).to(cuda))
        for dtype in DTYPES:
            want = ops.f8_matmul(a, b, out_dtype=dtype)
            room = torch.full((M, N + 9), 5.0, dtype=dtype, device=cuda)
            ops.f8_matmul(a, b, out=room[:, 3:3 + N])
            assert torch.equal(room[:, 3:3 + N], want)
            assert bool((room[:, :3] == 5).all()) and bool((room[:, 3 + N:] == 5).all())


def test_operators_past_32_bit_offsets(cuda):
    """Rows whose bytes and elements lie beyond 2^32 and 2^31: the last ones are what they are alone."""
    R, C = 140000, 16384
    x = torch.zeros((R, C), dtype=torch.bfloat16, device=cuda)
    tail = _rows(120, 70, C, torch.bfloat16).to(cuda)
    x[-70:] = tail
    w = ops.f8_weight_image(_rows(121, 16, C, size=C ** -0.5).to(cuda))
    y = ops.rms_norm(x, None, 1e-6)
    assert torch.equal(y[-70:], ops.rms_norm(tail, None, 1e-6)) and float(y[:1000].abs().sum()) == 0
    del y
    q = ops.f8_rows(x)
    alone = ops.f8_rows(tail)
    assert torch.equal(q.data[-70:].view(torch.uint8), alone.data.view(torch.uint8))
    got = ops.f8_matmul(q, w)
    # the two calls may add the same exact products in another order: each is within the bound of one sum
    qa, qb = (ref.value(v.data.cpu(), v.scale.cpu().view(torch.uint8).int() - 127, h) for v, h in ((alone, 1), (w, 128)))
    want = qa @ qb.t()
    _within(got[-70:], want, _product_bound(qa, qb, C, want, torch.float32))
    _within(ops.f8_matmul(alone, w), want, _product_bound(qa, qb, C, want, torch.float32))
    assert float(got[:1000].abs().sum()) == 0
    del q, got
    xt = ops.f8_cols(x)
    assert torch.equal(xt.data[:, -70:].float(), ops.f8_cols(x[-(R % 128 or 128):]).data[:, -70:].float())
    del xt
    total = ops.clip_norm_([x], 1.0)
    want, (part,) = ref.clip([tail], 1.0)
    _within(total, want, 2 * F32 * want)
    _within(x[-70:], part, (half_step(torch.bfloat16) + 6 * F32) * part.abs() * 1.001 + tiny(torch.bfloat16))


def test_second_derivatives_and_too_many_rows_are_refused(cuda):
    x, w = _rows(120, 6, 16).to(cuda).requires_grad_(), _rows(121, 8, 16).to(cuda).requires_grad_()
    for y in (ops.rms_norm(x), ops.f8_linear(x, w)):
        with pytest.raises(RuntimeError, match="differentiable once"):
            torch.autograd.grad(y.sum(), x, create_graph=True)
    many = torch.zeros((1, 16), device=cuda).expand((1 << 22) + 1, 16)  # 2^22 + 1 rows in 64 bytes
    bias = torch.zeros((8,), device=cuda, requires_grad=True)
    for args in ((many, w), (many, w.detach(), bias)):
        with pytest.raises(ValueError, match="2\\^22 rows"):
            ops.f8_linear(*args)
    with pytest.raises(ValueError, match="2\\^22 columns"):
        ops.f8_linear(torch.zeros((1, 1), device=cuda).expand(1, (1 << 22) + 1),
                      torch.zeros((1, 1), device=cuda).expand(1, (1 << 22) + 1))


def test_what_the_operators_write_counts_as_modified(cuda):
    flat = torch.ones((32,), device=cuda)
    views = [flat[:16], flat[16:]]
    grads = [torch.ones((16,), device=cuda) for _ in range(2)]
    for write, touched in ((lambda: ops.clip_norm_(grads, 1.0), grads),
                           (lambda: ops.clip_norm_(grads, 1.0, out=views), [flat]),
                           (lambda: ops.clip_norm_(grads, 1.0, out=flat), [flat])):
        before = [t._version for t in touched]
        write()
        assert all(t._version > b for t, b in zip(touched, before))
    before = [t._version for t in grads]
    ops.grad_norm(grads)
    ops.clip_norm_(grads, 1.0, out=flat)
    assert [t._version for t in grads] == before
    a = ops.f8_rows(_rows(122, 4, 16).to(cuda))
    out = torch.ones((4, 4), device=cuda, requires_grad=True).clone()
    y = out.square()
    ops.f8_matmul(a, a, out=out.detach())
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 8, 8), (127, 64, 64), (129, 72, 24), (257, 128, 40), (500, 40, 136), (3000, 256, 64),
                                   (1300, 64, 256), (700, 200, 144), (33000, 256, 256), (66000, 32, 200)])
def test_f8_linear_weight_and_bias_gradient_in_one_reading(cuda, shape, dtype):
    R, K, N = shape
    assert ops._lib.lib().lcf_f8_weight_grad_workspace_bytes(R, K, N) > 0
    x, dy = _rows(130, R, K, dtype), _rows(131, R, N, dtype, 1e-2)
    dt, xt = ref.value(*ref.quantise(dy.t())), ref.value(*ref.quantise(x.t()))
    want, sums = dt @ xt.t(), dy.double().sum(0)
    for wtype, turned in ((torch.float32, False), (torch.float32, True), (torch.bfloat16, True), (torch.float16, False)):
        w = _rows(132, N, K, size=K ** -0.5).to(wtype)
        w = (w.t().contiguous() if turned else w).to(cuda).requires_grad_()
        bias = torch.zeros((N,), dtype=wtype, device=cuda, requires_grad=True)
        y = ops.f8_linear(x.to(cuda), w, bias, turned)
        dw, db = torch.autograd.grad(y, (w, bias), dy.to(cuda))
        again = torch.autograd.grad(ops.f8_linear(x.to(cuda), w, bias, turned), (w, bias), dy.to(cuda))
        assert dw.dtype == wtype and torch.equal(dw, again[0]) and torch.equal(db, again[1])
        _within(dw.t() if turned else dw, want, _product_bound(dt, xt, R, want, wtype) + tiny(wtype), "dw")
        # 128 rows of a block one behind the other, the blocks of a workgroup, then 64 bits
        _within(db, sums, (140 + R // 128) * F32 * dy.double().abs().sum(0) + half_step(wtype) * 1.01 * sums.abs()
                + tiny(wtype), "db")
        only, = torch.autograd.grad(ops.f8_linear(x.to(cuda), w, None, turned), w, dy.to(cuda))
        assert torch.equal(only, dw)


@pytest.mark.parametrize("dtype", DTYPES)
def test_f8_linear_weight_gradient_of_strided_and_unfinished_rows(cuda, dtype):
    R, K, N = 400, 64, 128
    room = torch.full((R, K + 24), float("nan"), dtype=dtype, device=cuda)
    room[:, 8:8 + K] = _rows(133, R, K, dtype).to(cuda)
    grads = torch.full((R, N + 3), float("nan"), dtype=dtype, device=cuda)
    grads[:, 1:1 + N] = _rows(134, R, N, dtype).to(cuda)
    w = torch.zeros((N, K), device=cuda, requires_grad=True)

    def grad(x, dy):
        return torch.autograd.grad(ops.f8_linear(x, w), w, dy)[0]
    want = grad(room[:, 8:8 + K].contiguous(), grads[:, 1:1 + N].contiguous())
    assert bool(want.isfinite().all())
    assert torch.equal(grad(room[:, 8:8 + K], grads[:, 1:1 + N].contiguous()), want)
    # rows that do not start on whole dwords take the columns forms: the same products in another order
    odd = grad(room[:, 8:8 + K], grads[:, 1:1 + N])
    assert (odd - want).abs().max() <= 1e-5 * want.abs().max()
    # an infinity or a NaN reaches its own row or column of the gradient and no other
    x, dy = room[:, 8:8 + K].contiguous(), grads[:, 1:1 + N].contiguous()
    x[5, 3], x[300, 17], dy[130, 9] = float("inf"), float("nan"), float("-inf")
    got = grad(x, dy)
    bad = torch.zeros((N, K), dtype=torch.bool, device=cuda)
    bad[:, 3] = bad[:, 17] = bad[9] = True
    assert bool(got[bad].isnan().all()) and bool(got[~bad].isfinite().all())


@pytest.mark.parametrize("K", [300, 384])
def test_f8_matmul_ignores_scales_behind_the_last_block(cuda, K):
    """Scales that are the first columns of a wider matrix whose others mean nothing (255 is no number):
    three blocks of 128, four bytes to a word."""
    M, N = 4100, 72
    a, b = _rows(80, M, K, torch.bfloat16), _rows(81, N, K, size=K ** -0.5)
    xa, xb, w = ops.f8_rows(a.to(cuda)), ops.f8_rows(b.to(cuda)), ops.f8_weight_image(b.to(cuda))

    def behind(x):
        room = torch.full((x.scale.shape[0], 8), 255, dtype=torch.uint8, device=cuda)
        room[:, :3] = x.scale.view(torch.uint8)
        return ops.F8Rows(x.data, room[:, :3])
    for out in DTYPES:
        for m in (M, 3000, 40):  # rows past b in registers, tiles, few rows
            part = ops.F8Rows(xa.data[:m], xa.scale[:m])
            for image in (xb, w):
                want = ops.f8_matmul(part, image, out_dtype=out)
                assert bool(torch.isfinite(want).all())
                for p, q in ((behind(part), image), (part, behind(image)), (behind(part), behind(image))):
                    assert torch.equal(ops.f8_matmul(p, q, out_dtype=out), want), (out, m)
    want = ops.f8_product(a.to(cuda), w)
    assert torch.equal(ops.f8_product(a.to(cuda), behind(w)), want)


def test_forward_mode_derivatives_are_refused(cuda):
    """A dual tensor need not require a gradient: without a refusal its tangent would be lost."""
    from torch.autograd import forward_ad
    x, w, r = (t.to(cuda) for t in (_rows(82, 20, 32), torch.ones(32), _rows(83, 20, 32)))
    m, b = _rows(84, 8, 32).to(cuda), torch.zeros(8, device=cuda)
    with forward_ad.dual_level():
        for grad in (False, True):
            def dual(t):
                return forward_ad.make_dual(t.clone().requires_grad_(grad), torch.ones_like(t))
            for call in (lambda: ops.rms_norm(dual(x), w), lambda: ops.rms_norm(x, dual(w)),
                         lambda: ops.rms_norm(x, w, residual=dual(r)), lambda: ops.f8_linear(dual(x), m),
                         lambda: ops.f8_linear(x, dual(m)), lambda: ops.f8_linear(x, m, dual(b))):
                with pytest.raises(RuntimeError):
                    call()
        assert torch.equal(ops.rms_norm(x, w), ops.rms_norm(x.clone(), w))  # what has no tangent goes through


def test_f8_linear_keeps_only_what_its_gradients_take(cuda):
    """The rows are kept for the weight's gradient alone and the weight not at all: a layer whose weight
    is frozen does not mind its rows being written to, nor a first layer its weight being stepped."""
    x0, w0, b0 = _rows(85, 50, 48).to(cuda), _rows(86, 24, 48).to(cuda), torch.zeros(24, device=cuda)
    dy = _rows(87, 50, 24).to(cuda)

    def grads(frozen, first, late):
        x, w, b = x0.clone(), w0.clone(), b0.clone().requires_grad_(True)
        leaf = x0.clone().requires_grad_(not first)
        w.requires_grad_(not frozen)
        rows = leaf * 1.0 if not first else x
        y = ops.f8_linear(rows, w, b)
        with torch.no_grad():
            if late and frozen:
                rows.zero_()
            if late:
                w.zero_()
        y.backward(dy)
        return [t.grad for t in (leaf, w, b) if t.requires_grad]
    for frozen, first in ((True, False), (False, True), (True, True), (False, False)):
        want, got = grads(frozen, first, False), grads(frozen, first, True)
        assert len(got) == 3 - frozen - first
        assert all(torch.equal(p, q) for p, q in zip(want, got))
    # rows that the weight's gradient does take may not change in between
    x, w = x0.clone(), w0.clone().requires_grad_(True)
    y = ops.f8_linear(x, w)
    x.zero_()
    with pytest.raises(RuntimeError):
        y.backward(dy)


@pytest.mark.parametrize("lead", [(2, 3), (0, 3), (), (4,)])
def test_f8_linear_of_no_columns_and_of_any_leading_sizes(cuda, lead):
    bias = torch.randn((8,), generator=_gen(88)).to(cuda)
    for K in (0, 32):
        x = torch.randn((*lead, K), generator=_gen(89)).to(cuda).requires_grad_(True)
        w = torch.randn((8, K), generator=_gen(90)).to(cuda).requires_grad_(True)
        y = ops.f8_linear(x, w, bias)
        assert y.shape == (*lead, 8)
        rows = ops.f8_linear(x.detach().reshape(math.prod(lead), K), w.detach(), bias)
        assert torch.equal(y.detach().reshape(math.prod(lead), 8), rows)
        y.sum().backward()
        assert x.grad.shape == x.shape and w.grad.shape == w.shape


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(50, 200, 20011), (64, 260, 9000), (17, 65, 8200), (1, 16, 30000), (16, 129, 8193),
                                   (33, 24, 4100), (48, 1000, 5000)])
def test_f8_matmul_long_sums_of_few_rows(cuda, shape, dtype):
    """Few rows over a long sum, split over workgroups, and the same call into the library without room for
    the split."""
    M, N, K = shape
    L, code = ops._lib.lib(), ops._TYPE_CODE[dtype]
    assert L.lcf_f8_gemm_split_bytes(M, N, K, code) > L.lcf_f8_gemm_workspace_bytes(M, N, K, code) == 0
    a, b = _rows(91, M, K), _rows(92, N, K, size=K ** -0.5)
    scale, shift = torch.rand((N,), generator=_gen(93)) + 0.5, torch.randn((N,), generator=_gen(94))
    qa, qb = ref.value(*ref.quantise(a)), ref.value(*ref.quantise(b))
    y = qa @ qb.t()
    xa, xb = ops.f8_rows(a.to(cuda)), ops.f8_rows(b.to(cuda))
    s, t = scale.to(cuda), shift.to(cuda)
    got = [ops.f8_matmul(xa, xb, s, t, True, dtype) for _ in range(3)]
    assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])
    one = torch.empty((M, N), dtype=dtype, device=cuda)
    assert L.lcf_f8_gemm(xa.data.data_ptr(), xa.data.stride(0), xa.scale.data_ptr(), xa.scale.stride(0), 0,
                         xb.data.data_ptr(), xb.data.stride(0), xb.scale.data_ptr(), xb.scale.stride(0), 0, 0, M, N, K,
                         s.data_ptr(), t.data_ptr(), 1, one.data_ptr(), N, code, None, 0,
                         torch.cuda.current_stream().cuda_stream) == 0
    want = (y * scale.double() + shift.double()).clamp(min=0)
    bound = (scale.double() * _product_bound(qa, qb, K, y, dtype)
             + 4 * F32 * (y.abs() * scale.double() + shift.double().abs()) + half_step(dtype) * want * 1.01 + tiny(dtype))
    _within(got[0], want, bound, "split")
    _within(one, want, bound, "whole")


@pytest.mark.parametrize("turned", [False, True])
@pytest.mark.parametrize("shape", [(20000, 50, 200), (9001, 260, 64), (30000, 18, 33)])
def test_f8_linear_weight_gradients_of_few_channels(cuda, shape, turned):
    """Channel counts that are no multiples of 8, or more than 256, over many rows."""
    M, N, K = shape
    x = _rows(95, M, K, torch.bfloat16).to(cuda)
    w = _rows(96, N, K, size=K ** -0.5).to(cuda)
    leaf = (w.t().contiguous() if turned else w).requires_grad_(True)
    dy = _rows(97, M, N, torch.bfloat16, 1e-2)
    dw, = torch.autograd.grad(ops.f8_linear(x, leaf, turned=turned), leaf, dy.to(cuda))
    dt, xt = ref.value(*ref.quantise(dy.t())), ref.value(*ref.quantise(x.t()))
    want = dt @ xt.t()
    _within(dw.t() if turned else dw, want, _product_bound(dt, xt, M, want, torch.float32), "dw")


@pytest.mark.parametrize("shape", [(8, 24, 130), (100, 64, 300), (4100, 16, 128)])
@pytest.mark.parametrize("f8", [E4M3, E5M2])
def test_f8_matmul_at_the_ends_of_the_scales(cuda, f8, shape):
    """Blocks of the smallest scale against blocks of large ones: fp32 outputs widen to bf16, whose least
    step is 2^-133 (half of it for each element, times what it meets); the 8-bit instruction has no such end."""
    M, N, K = shape
    size = torch.exp(-8 * torch.rand((M, 1), generator=_gen(98)))  # magnitudes from 1e-35 down to 1e-38 and less
    a = _rows(99, M, K) * size * 1e-35
    a[0] = a[0] * 1e-5
    b = _rows(100, N, K) * 1e35
    for left, right, swap in ((a, b, False), (b, a, True)):
        qa, qb = ref.value(*ref.quantise(left, f8)), ref.value(*ref.quantise(right, f8))
        want = qa @ qb.t()
        xa, xb = ops.f8_rows(left.to(cuda), f8), ops.f8_rows(right.to(cuda), f8)
        rounded = 2.0 ** -134 * (qb.abs().sum(1)[None, :] if not swap else qa.abs().sum(1)[:, None])
        for out in (torch.float32, torch.bfloat16):
            got = ops.f8_matmul(xa, xb, out_dtype=out)
            bound = _product_bound(qa, qb, K, want, out) + (1 + 2 * K * F32) * (rounded if out == torch.float32 else 0.0)
            _within(got, want, bound, (out, swap))
    # a block whose largest magnitude rounds up to 2^128
    top = torch.zeros((M, 128))
    top[:, 0] = 3.4e38
    one = torch.zeros((N, 128))
    one[:, 0] = 2.0 ** -40
    xa, xb = ops.f8_rows(top.to(cuda)), ops.f8_rows(one.to(cuda))
    assert bool((ops.f8_matmul(xa, xb) == float("inf")).all())
    assert bool((ops.f8_matmul(xa, xb, out_dtype=torch.bfloat16) == 2.0 ** 88).all())
