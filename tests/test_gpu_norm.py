"""GPU: root-mean-square norm and its gradient (a3b_rms_norm, a3b_rms_norm_backward) against the formulas in 64 bits.

Tolerances, with u = 2^-24 (half a step of fp32 at 1), n elements a row and N = n / 512 + 64 (at least the number of additions
one after the other, in every kernel): a sum of squares is off by at most (N + 1) u of itself, so r = 1 / sqrt(sum / n + eps)
by (N / 2 + 4) u with its own four roundings, y = h r w by (N / 2 + 6) u, and a stored value by half a step of its type more
(of its least subnormal near zero). An 8-bit value is y / s, both from fp32: half a step of 8 bits, and (N + 10) u of it.
Gradient: c = mean(d k) with k = h r is off by (N + 4) u mean|d k|, and r (d - k c) + gtotal carries it times |r k|, and the
roundings of each summand. dw is a sum of at most rows / 148 + 64 terms one after the other."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0**-24
INF = math.inf
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
LARGEST = {torch.float8_e4m3fn: 448.0, torch.float8_e5m2: 57344.0}
# of half a step: relative, and of the least subnormal
HALF8 = {torch.float8_e4m3fn: (2.0**-4, 2.0**-10), torch.float8_e5m2: (2.0**-3, 2.0**-17)}


def depth(n):
    return n / 512 + 64


def half(dtype):
    """(relative half step, half of the least subnormal)"""
    info = torch.finfo(dtype)
    return info.eps / 2, info.smallest_normal * info.eps / 2


def close(got, want, tol):
    got, want = got.double(), want.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    fine = torch.isfinite(want)
    rest = ~fine & ~torch.isnan(want)
    assert torch.equal(got[rest], want[rest])
    off = (got - want).abs()[fine] - tol.expand_as(want)[fine]
    assert off.numel() == 0 or off.max() <= 0, (off.max(), (got - want).abs()[fine].max())


def make(shape, dtype, seed, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def definition(x, weight, residual, eps):
    """h (as stored), r and y in 64 bits"""
    h = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    h = h.double()
    r = 1 / torch.sqrt(h.square().mean(-1, keepdim=True) + eps)
    y = h * r
    return h, r, y if weight is None else y * weight.double()


def check_forward(x, weight=None, residual=None, kind=None, group=None, eps=1e-6, out=None, total=None, given=True):
    from alpaka3_b200 import algo
    n = x.shape[-1]
    h, r, y = definition(x, weight, residual, eps)
    rstd = torch.full(x.shape[:-1], 77.0, device="cuda") if given else None
    if total is None and residual is not None and given:
        total = torch.full(x.shape, 7.0, dtype=x.dtype, device="cuda")
    if out is None:
        out = torch.zeros(x.shape, dtype=kind or x.dtype, device="cuda")
    scales = None
    if kind is not None:
        groups = -(-n // group) if group else 1
        scales = torch.full((*x.shape[:-1], groups), 77.0, device="cuda")
    got = algo.rms_norm(out, x, weight, residual=residual, total=total, rstd=rstd, scales=scales, group=group, eps=eps)
    assert got is out
    if total is not None:
        close(total, h, torch.zeros((), device="cuda", dtype=torch.float64))
    if rstd is not None:
        close(rstd[..., None], r, (depth(n) / 2 + 4) * U * r + 2.0**-150)
    loss = (depth(n) / 2 + 6) * U
    if kind is None:
        rel, least = half(x.dtype)
        close(out, y, (rel + loss) * y.abs() + least)
        return out
    size = group or n
    pad = -n % size
    parts = torch.nn.functional.pad(y, (0, pad)).unflatten(-1, (-1, size))
    s = parts.abs().amax(-1, keepdim=True) / LARGEST[kind]
    close(scales[..., None], s, (loss + U) * s + 2.0**-150)
    q = torch.where(s > 0, parts / s, torch.zeros_like(parts)).flatten(-2)[..., :n]
    rel, least = HALF8[kind]
    close(out.float(), q, torch.clamp(rel * q.abs(), min=least) + (depth(n) + 10) * U * q.abs())
    return out


# one element; below, at and above a pack, a part of a warp, a warp, a block of every kind; rows without packs
WIDTHS = [1, 2, 7, 8, 9, 16, 31, 32, 33, 64, 100, 128, 129, 255, 256, 257, 512, 1000, 1001, 1024, 1032, 2048, 2049, 4096, 5000,
          5003, 8192, 8200, 16384, 16385, 16392, 20000, 32768, 32769, 32776, 70000]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", WIDTHS)
def test_forward_against_64_bits(cuda, dtype, n):
    for rows in (1, 3, 37) if n > 4096 else (1, 5, 700):
        x = make((rows, n), dtype, n + rows, 1.5)
        w = make((n,), torch.float32, n).add_(1)
        check_forward(x, w.to(dtype), make((rows, n), dtype, n + 1, 2.0))
        check_forward(x, w, None)
    check_forward(x, None, make((rows, n), dtype, n + 2), given=False)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", list(LARGEST))
@pytest.mark.parametrize("n", [1, 5, 8, 16, 33, 64, 96, 128, 136, 200, 256, 1000, 1001, 1024, 2048, 4104, 8192, 16400, 32768, 40000])
def test_eight_bits(cuda, dtype, kind, n):
    for rows in (2, 640) if n <= 2048 else (1, 9):
        x = make((rows, n), dtype, n + rows, 1.5)
        # magnitudes of different groups differ
        x = (x.float() * torch.exp2(torch.arange(n, device="cuda") // 32 % 9 - 4.0)).to(dtype)
        w = make((n,), torch.float32, n).add_(1)
        for group in (None, 32, 64, 128):
            check_forward(x, w if group == 64 else w.to(dtype), make((rows, n), dtype, 3) if group == 32 else None, kind, group)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", list(LARGEST))
@pytest.mark.parametrize("n", [31, 95, 127, 129, 257, 1001, 4095, 4097, 8191, 8193, 16401, 32767, 32769])
def test_eight_bits_without_packs(cuda, dtype, kind, n):
    """Rows of every length at which another form takes over, and ones whose first element lies off 16 bytes; in place."""
    for rows in (3, 50):
        wide = make((rows, n + 1), dtype, n + rows, 1.5)
        x, res, w = wide[:, 1:], make((rows, n), dtype, 3), make((n,), torch.float32, n).add_(1)
        for group in (None, 32, 64, 128):
            check_forward(x, w, None, kind, group)
            check_forward(x, w.to(dtype), res, kind, group)
        x[0, n // 2:] = 0
        x[1].mul_(0)
        a = res.clone()
        check_forward(x, None, res, kind, 64)
        check_forward(x, None, a, kind, 64, total=a)
        check_forward(x, None, None, kind, 32)
        nan = x.clone()
        nan[2, n // 3] = math.nan
        check_forward(nan[:2], w, None, kind, 64)
        out, scales = torch.zeros(rows, n, dtype=kind, device="cuda"), torch.zeros(rows, -(-n // 64), device="cuda")
        from alpaka3_b200 import algo
        algo.rms_norm(out, nan, w, scales=scales, group=64)
        assert torch.isnan(scales[2]).all() and torch.isnan(out[2].float()).all() and not torch.isnan(scales[:2]).any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [64, 77, 1024, 4096, 40000])
def test_zeros_and_empty_groups(cuda, dtype, n):
    from alpaka3_b200 import algo
    x = make((4, n), dtype, 1)
    x[1] = 0
    x[2, : n // 2] = 0
    check_forward(x)
    for kind in LARGEST:
        for group in (None, 32, 64, 128):
            check_forward(x, None, None, kind, group)
    # a row of zeros without eps: 0 * infinity
    out, rstd = torch.zeros_like(x), torch.zeros(4, device="cuda")
    algo.rms_norm(out, x, rstd=rstd, eps=0.0)
    assert torch.isnan(out[1]).all() and rstd[1] == INF and torch.isfinite(out[[0, 2, 3]]).all()


@pytest.mark.parametrize("n", [8, 33, 256, 1024, 4096, 8192, 33000])
@pytest.mark.parametrize("size", [1e19, 3e25, 1e38, 1e-20, 3e-30])
def test_far_rows(cuda, n, size):
    """Squares that leave fp32's range: 1e19 .. 1e38 above it, 1e-20 .. 3e-30 (with a tiny eps) below it."""
    for dtype in (torch.float32, torch.bfloat16):
        x = make((3, n), dtype, 5).clamp(-3, 3).float()
        x[0] *= size
        x[2] *= size
        for eps in (1e-6, 0.0, 1e-45):
            check_forward(x.to(dtype), None, None, eps=eps)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [8, 33, 128, 1024, 4096, 33000])
def test_infinities_and_nan(cuda, dtype, n):
    from alpaka3_b200 import algo
    x = make((5, n), dtype, 6)
    x[1, n // 2] = INF
    x[3, n - 1] = math.nan
    out, rstd = torch.zeros_like(x), torch.zeros(5, device="cuda")
    algo.rms_norm(out, x, rstd=rstd)
    assert rstd[1] == 0 and torch.isnan(out[1, n // 2]) and (out[1, torch.arange(n, device="cuda") != n // 2] == 0).all()
    assert torch.isnan(rstd[3]) and torch.isnan(out[3]).all()
    assert torch.isfinite(out[[0, 2, 4]]).all() and torch.isfinite(rstd[[0, 2, 4]]).all()
    for kind in LARGEST:
        q, scales = torch.zeros(x.shape, dtype=kind, device="cuda"), torch.zeros(5, device="cuda")
        algo.rms_norm(q, x, scales=scales)
        assert torch.isnan(scales[[1, 3]]).all() and torch.isnan(q.float()[[1, 3]]).all()
        assert torch.isfinite(scales[[0, 2, 4]]).all() and torch.isfinite(q.float()[[0, 2, 4]]).all()


def test_tiny_scales(cuda):
    """Groups whose scale is below fp32's normal numbers have no reciprocal: their values are divided."""
    x = make((2, 256), torch.float32, 7)
    w = torch.full((256,), 1e-37, device="cuda")
    w[128:] = 1e-44
    from alpaka3_b200 import algo
    out, scales = torch.zeros(2, 256, dtype=torch.float8_e4m3fn, device="cuda"), torch.zeros(2, 4, device="cuda")
    algo.rms_norm(out, x, w, scales=scales, group=64)
    y = definition(x, w, None, 1e-6)[2]
    back = out.double().unflatten(-1, (4, 64)) * scales.double()[..., None]
    # y, s and their quotient each off by half of fp32's least subnormal 2^-149: s by 2^-150, so 448 s by 2^-141
    assert (back.flatten(-2) - y).abs().max() <= 2.0**-4 * y.abs().max() + 2.0**-140
    assert torch.isfinite(out.float()).all()
    assert (back.flatten(-2)[:, :128] - y[:, :128]).abs().max() <= (2.0**-4 + 2.0**-8) * y[:, :128].abs().max()


def test_layouts(cuda):
    """Strided rows of every tensor, one and two levels; what lies between rows stays as it was."""
    from alpaka3_b200 import algo
    for dtype in DTYPES:
        for n, gap in ((128, 64), (128, 3), (50, 14), (512, 8)):
            wide = make((6, 4, 2 * n + gap), dtype, n)
            x, res = wide[..., :n], make((6, 5, n + gap), dtype, 2)[:, 1:, gap:]
            room = torch.full((6, 4, 3 * n + gap), 5.0, dtype=dtype, device="cuda")
            before = room.clone()
            out, total = room[..., :n], room[..., n + gap:2 * n + gap]
            check_forward(x, make((n,), dtype, 4), res, out=out, total=total)
            room[..., :n] = before[..., :n]
            room[..., n + gap:2 * n + gap] = before[..., n + gap:2 * n + gap]
            assert torch.equal(room, before)
            # heads of the rows in another order
            check_forward(x.transpose(0, 1), None, res.transpose(0, 1))
            back = torch.zeros(4, 6, n, dtype=dtype, device="cuda").transpose(0, 1)
            check_forward(x, None, res, out=back)
    x = torch.zeros(3, 4, 5, 16, device="cuda")[:, :3, :4]
    with pytest.raises(ValueError, match="two strides"):
        algo.rms_norm(torch.zeros(3, 3, 4, 16, device="cuda"), x)


@pytest.mark.parametrize("n", [64, 77, 1024, 5000, 40001])
@pytest.mark.parametrize("dtype", DTYPES)
def test_in_place(cuda, dtype, n):
    from alpaka3_b200 import algo
    for rows in (3, 700) if n < 5000 else (3,):
        x, res, w = make((rows, n), dtype, 1), make((rows, n), dtype, 2), make((n,), dtype, 3)
        total, out = torch.empty_like(x), torch.empty_like(x)
        algo.rms_norm(out, x, w, residual=res, total=total)
        for o, t in (("x", "res"), ("res", "x"), ("x", None), ("res", None)):
            a = {"x": x.clone(), "res": res.clone()}
            algo.rms_norm(a[o], a["x"], w, residual=a["res"], total=a[t] if t else None)
            assert torch.equal(a[o], out) and (t is None or torch.equal(a[t], total)), (o, t)
        a = x.clone()
        algo.rms_norm(a, a, w)
        plain = algo.rms_norm(torch.empty_like(x), x, w)
        assert torch.equal(a, plain)
        # the same tensor twice
        twice = algo.rms_norm(torch.empty_like(x), x, w, residual=x)
        assert torch.equal(twice, algo.rms_norm(torch.empty_like(x), x, w, residual=x.clone()))


# ------------------------------------------------------------------------------------------------------ gradient
def check_backward(g, x, weight, gtotal=None, gx=None, eps=1e-6, want_weight=True, rstd=None):
    from alpaka3_b200 import algo
    n = x.shape[-1]
    if rstd is None:
        rstd = (1 / torch.sqrt(x.double().square().mean(-1) + eps)).float()
    r = rstd.double()[..., None]
    h, gd = x.double(), g.double()
    k = h * r
    d = gd if weight is None else gd * weight.double()
    c = (d * k).mean(-1, keepdim=True)
    want = r * (d - k * c)
    size = r * (4 * U * d.abs() + 5 * U * (k * c).abs() + k.abs() * (depth(n) + 6) * U * (d * k).abs().mean(-1, keepdim=True))
    if gtotal is not None:
        want = want + gtotal.double()
        size = size + 2 * U * gtotal.double().abs()
    rel, least = half(x.dtype)
    dtype = x.dtype if weight is None else weight.dtype
    gw = torch.full((n,), 7.0, dtype=dtype, device="cuda") if want_weight else None
    if gx is None:
        gx = torch.full(x.shape, 7.0, dtype=x.dtype, device="cuda")
    wantw = (gd * k).flatten(0, -2).sum(0)
    sizew = (gd * k).abs().flatten(0, -2).sum(0)
    assert algo.rms_norm_backward(gx, g, x, weight, rstd, grad_weight=gw, grad_total=gtotal) is gx
    close(gx, want, size * (1 + rel) + (rel + 2 * U) * want.abs() + least)
    if gw is not None:
        rows = x.numel() // n
        rel, least = half(dtype)
        close(gw, wantw, (rows / 148 + 68) * U * sizew + rel * wantw.abs() * (1 + 2.0**-10) + least)
    return gx, gw


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", WIDTHS)
def test_backward_against_64_bits(cuda, dtype, n):
    for rows in (1, 3, 37) if n > 4096 else (1, 5, 700, 1300):
        x, g = make((rows, n), dtype, n + rows, 2.0), make((rows, n), dtype, n, 0.1)
        w = make((n,), torch.float32, n).add_(1)
        check_backward(g, x, w.to(dtype), make((rows, n), dtype, 3, 0.1))
        check_backward(g, x, w)
    check_backward(g, x, None, want_weight=False)
    check_backward(g, x, None)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [24, 100, 128, 500, 1001, 1024, 4096, 8192])
def test_backward_of_few_rows(cuda, dtype, n):
    """As many rows as one block takes in one turn, which then leaves no partial sums, and one fewer and more."""
    for rows in {r + k for r in (1, 2, 4, 8, 16, 32, 64) for k in (-1, 0, 1)} - {0}:
        x, g = make((rows, n), dtype, n + rows, 2.0), make((rows, n), dtype, n, 0.1)
        w = make((n,), torch.float32, n).add_(1)
        check_backward(g, x, w.to(dtype), make((rows, n), dtype, 3, 0.1))
        check_backward(g, x, w)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [1, 7, 31, 100, 126, 128])
def test_backward_of_many_short_rows(cuda, dtype, n):
    """Rows without packs, of one warp each, sixteen in a block: in one turn and in several."""
    for rows in (16, 3001, 12000):
        wide = make((rows, n + 1), dtype, n)
        x, g = wide[:, 1:], make((rows, n), dtype, n + 1, 0.1)
        w = make((n,), torch.float32, n).add_(1)
        for _ in range(4):
            check_backward(g, x, w.to(dtype), make((rows, n), dtype, 3, 0.1))
            check_backward(g, x, w)


def test_many_rows(cuda):
    for n, rows, dtype in ((128, 40001, torch.bfloat16), (64, 70000, torch.float32), (1024, 5000, torch.float16),
                           (2048, 3001, torch.bfloat16), (1001, 2000, torch.float32), (35001, 600, torch.bfloat16)):
        x, g = make((rows, n), dtype, n, 2.0), make((rows, n), dtype, n + 1, 0.1)
        check_backward(g, x, make((n,), dtype, 2), make((rows, n), dtype, 3, 0.1))
        check_forward(x, make((n,), dtype, 2), g)


@pytest.mark.parametrize("n", [1, 24, 257, 2048])
def test_backward_against_differences(cuda, n):
    """Along random directions, of the 64-bit definition: with a step of 1e-4 the difference's own error is below 1e-6 of the
    sum of the terms' magnitudes."""
    from alpaka3_b200 import algo
    x, w, g, gt = (make(s, torch.float32, n + k) for k, s in enumerate(((6, n), (n,), (6, n), (6, n))))
    rstd = torch.empty(6, device="cuda")
    algo.rms_norm(torch.empty_like(x), x, w, rstd=rstd, eps=0.01)
    gx, gw = torch.empty_like(x), torch.empty_like(w)
    algo.rms_norm_backward(gx, g, x, w, rstd, grad_weight=gw, grad_total=gt)

    def loss(h, v):
        h, v = h.double(), v.double()
        return (h / torch.sqrt(h.square().mean(-1, keepdim=True) + 0.01) * v * g.double()).sum() + (h * gt.double()).sum()

    for seed in range(4):
        dx, dw = make((6, n), torch.float64, 50 + seed), make((n,), torch.float64, 60 + seed)
        diff = (loss(x.double() + 1e-4 * dx, w.double() + 1e-4 * dw)
                - loss(x.double() - 1e-4 * dx, w.double() - 1e-4 * dw)) / 2e-4
        terms = (gx.double() * dx).abs().sum() + (gw.double() * dw).abs().sum() + (g.double() * dw).abs().sum() + 1
        assert abs((gx.double() * dx).sum() + (gw.double() * dw).sum() - diff) <= 1e-5 * terms


def test_backward_layouts(cuda):
    for dtype in DTYPES:
        for n, gap in ((128, 64), (128, 3), (50, 14), (1024, 8)):
            wide = make((6, 4, 2 * n + gap), dtype, n)
            x, g = wide[..., :n], wide[..., n + gap:]
            gt = make((6, 5, n + gap), dtype, 2)[:, 1:, gap:]
            room = torch.full((6, 4, n + gap), 5.0, dtype=dtype, device="cuda")
            check_backward(g, x, make((n,), dtype, 4), gt, gx=room[..., :n])
            assert (room[..., n:] == 5).all()
            check_backward(g.transpose(0, 1), x.transpose(0, 1), None, gt.transpose(0, 1))


@pytest.mark.parametrize("n", [64, 77, 1024, 5000, 16400, 40001])
@pytest.mark.parametrize("dtype", DTYPES)
def test_backward_in_place(cuda, dtype, n):
    from alpaka3_b200 import algo
    for rows in (3, 1300) if n < 5000 else (3,):
        x, g, gt, w = (make(s, dtype, k) for k, s in enumerate(((rows, n), (rows, n), (rows, n), (n,))))
        rstd = (1 / torch.sqrt(x.double().square().mean(-1) + 1e-6)).float()
        gx, gw = torch.empty_like(x), torch.empty_like(w)
        algo.rms_norm_backward(gx, g, x, w, rstd, grad_weight=gw, grad_total=gt)
        for place in range(3):
            a = [x.clone(), g.clone(), gt.clone()]
            again = torch.empty_like(w)
            algo.rms_norm_backward(a[place], a[1], a[0], w, rstd, grad_weight=again, grad_total=a[2])
            assert torch.equal(a[place], gx) and torch.equal(again, gw)  # and the same bits in every call


def test_no_rows(cuda):
    from alpaka3_b200 import algo
    for dtype in DTYPES:
        x = torch.empty(0, 64, dtype=dtype, device="cuda")
        algo.rms_norm(torch.empty_like(x), x, residual=x, total=torch.empty_like(x), rstd=torch.empty(0, device="cuda"))
        gw = torch.full((64,), 3.0, dtype=dtype, device="cuda")
        algo.rms_norm_backward(torch.empty_like(x), x, x, None, torch.empty(0, device="cuda"), grad_weight=gw)
        assert (gw == 0).all()


def test_workspace_is_checked(cuda):
    from alpaka3_b200 import capi
    x, r, gw = torch.ones(40, 64, device="cuda"), torch.ones(40, device="cuda"), torch.zeros(64, device="cuda")
    size = capi.lib().a3b_rms_norm_backward_workspace(40, 64)
    ws = torch.empty(size + 16, dtype=torch.uint8, device="cuda")

    def call(at, bytes_):
        rows = (x.data_ptr(), 0, 64)
        return capi.lib().a3b_rms_norm_backward(None, capi.RMS_NORM_BACKWARD_ARGS.pack(
            1, 40, 64, *rows, *rows, 0, 0, 0, *rows, 0, r.data_ptr(), gw.data_ptr(), at, bytes_, capi.F32, capi.F32, capi.F32, 0))
    for at, bytes_ in ((0, size), (ws.data_ptr(), size - 1), (ws.data_ptr() + 8, size)):
        assert call(at, bytes_) == capi.ERR_INVALID and "workspace" in capi.last_error()
    assert call(ws.data_ptr(), size) == capi.OK
    torch.cuda.synchronize()


def test_streams_and_graphs(cuda):
    """Another stream than the current one; a captured call replayed on new inputs, two graphs that overlap."""
    from alpaka3_b200 import algo
    n, rows = 1024, 2000
    x, g, w = (make(s, torch.bfloat16, k) for k, s in enumerate(((rows, n), (rows, n), (n,))))
    rstd, out, gx, gw = torch.empty(rows, device="cuda"), torch.empty_like(x), torch.empty_like(x), torch.empty_like(w)

    def step(o, r, a, b, stream=None):
        algo.rms_norm(o, x, w, rstd=r, stream=stream)
        algo.rms_norm_backward(a, g, x, w, r, grad_weight=b, stream=stream)

    step(out, rstd, gx, gw)
    want = [t.clone() for t in (out, rstd, gx, gw)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = [torch.zeros_like(t) for t in want]
    side.wait_stream(torch.cuda.current_stream())
    step(*got, stream=side)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        o = [torch.zeros_like(t) for t in want]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step(*o)
        graphs.append(graph)
        outs.append(o)
    x.copy_(make((rows, n), torch.bfloat16, 9))
    step(out, rstd, gx, gw)
    want = [t.clone() for t in (out, rstd, gx, gw)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for o in outs:
        assert all(torch.equal(a, b) for a, b in zip(o, want))


@pytest.mark.parametrize("kind", list(LARGEST))
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,shift", [(64, 0), (512, 0), (2048, 0), (16384, 0), (65536, 0), (256, 1), (4096, 1), (8192, 1), (32768, 1)])
def test_eight_bits_next_to_a_middle(cuda, kind, dtype, n, shift):
    """Values that lie in the middle between two of 8 bits, but for the roundings of y / s, where every unit of the scale's
    reciprocal counts: the bits of y * (1 / s), each operation rounded to the nearest. Rows of +-1 have r = 1, so y is the
    weight; rows begin at 16 bytes (shift 0) or not."""
    from alpaka3_b200 import algo
    top, bits = LARGEST[kind], torch.arange(127, device="cuda", dtype=torch.uint8).view(kind).float()
    grid = bits[torch.isfinite(bits) & (bits > 0)]
    middle = (grid[1:] + grid[:-1]) / 2
    rows = 6
    x = torch.ones(rows, n + shift, dtype=dtype, device="cuda")[:, shift:]
    x[:, ::3] = -1
    for seed, group in enumerate((None, 32, 64, 128)):
        g = torch.Generator(device="cuda").manual_seed(n + seed)
        size = min(group or n, n)
        high = torch.rand(n // size, 1, generator=g, device="cuda") + 1
        s = high * torch.tensor(1 / top, device="cuda")  # the rounded 1 / top
        w = middle[torch.randint(len(middle), (n // size, size), generator=g, device="cuda")] * s
        w[:, size // 2:size // 2 + 1] = high
        out, scales = torch.zeros(rows, n, dtype=kind, device="cuda"), torch.zeros(rows, n // size, device="cuda")
        rstd = torch.zeros(rows, device="cuda")
        algo.rms_norm(out, x, w.flatten(), rstd=rstd, scales=scales, group=group, eps=0.0)
        assert (rstd == 1).all() and torch.equal(scales, s.flatten().expand(rows, -1))
        want = (w * (1 / s)).clamp(max=top).to(kind).float().flatten() * x.float()
        assert torch.equal(out.float(), want)


@pytest.mark.parametrize("kind", list(LARGEST))
@pytest.mark.parametrize("n", [256, 2048, 16384, 257, 5001, 40001])
def test_scales_below_normal_numbers(cuda, kind, n):
    """Weights from 1e-36 to 1e-45: every group by itself. What the kernel's fp32 steps give, subnormal numbers among them, is
    known to the bit; where max |y| / L rounds to 0, scale and values are 0. Against the definition the scale is off by the
    roundings of y and of itself, half of 2^-149 each, beside those of normal numbers."""
    from alpaka3_b200 import algo
    x, top = make((3, n), torch.float32, n), LARGEST[kind]
    for group in (None, 32, 128):
        for w in (1e-36, 1e-38, 1e-39, 1e-41, 1e-42, 3e-43, 3e-44, 1e-45):
            weight = torch.full((n,), w, device="cuda")
            if group:
                weight[n // 2:] = 1e-30  # neighbours of another size
            size = group or n
            out, rstd = torch.ones(3, n, device="cuda").to(kind), torch.zeros(3, device="cuda")
            scales = torch.ones(3, -(-n // size), device="cuda")
            algo.rms_norm(out, x, weight, rstd=rstd, scales=scales, group=group)
            y = x * rstd[:, None] * weight
            parts = torch.nn.functional.pad(y, (0, -n % size)).unflatten(-1, (-1, size))
            s = parts.abs().amax(-1) * torch.tensor(1 / top, device="cuda")
            assert torch.equal(scales, s)
            q = torch.where(s[..., None] < 2.0**-126, parts / s[..., None], parts * (1 / s)[..., None])
            q = torch.where(s[..., None] == 0, torch.zeros_like(q), q).clamp(-top, top).flatten(1)[:, :n]
            assert torch.equal(out.float(), q.to(kind).float())
            true = definition(x, weight, None, 1e-6)[2]
            true = torch.nn.functional.pad(true, (0, -n % size)).unflatten(-1, (-1, size)).abs().amax(-1) / top
            close(scales, true, ((depth(n) / 2 + 7) * U * true + 2.0**-149))
            if w < 1e-43:
                assert (s[:, 0] == 0).all() and (out[:, :min(size, n // 2)].float() == 0).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [8, 33, 256, 1024, 8192, 33000])
def test_rows_whose_root_is_beyond_fp32(cuda, dtype, n):
    """Magnitudes below 2^-128 without eps: r is infinite in fp32, and y = h r w with it; with the least eps it is not."""
    from alpaka3_b200 import algo
    x = make((3, n), dtype, n).clamp(-3, 3)
    x[1] = (x[1].float() * 1e-40).to(dtype)
    x[1, n // 2] = 0
    out, rstd = torch.zeros_like(x), torch.zeros(3, device="cuda")
    algo.rms_norm(out, x, rstd=rstd, eps=0.0)
    assert rstd[1] == INF and torch.equal(torch.isnan(out[1]), x[1] == 0)
    assert torch.isinf(out[1, x[1] != 0]).all() and torch.equal(out[1, x[1] != 0] > 0, x[1, x[1] != 0] > 0)
    check_forward(x[::2].contiguous(), eps=0.0)
    check_forward(x, eps=2.0**-149)


@pytest.mark.parametrize("kind", list(LARGEST))
@pytest.mark.parametrize("n", [64, 1000, 8192, 257, 5001, 40001])
def test_infinite_values_of_a_group(cuda, kind, n):
    """An infinite weight: the group's scale is infinite, its infinity NaN, what is finite 0; other groups are as without it."""
    from alpaka3_b200 import algo
    x, w = make((2, n), torch.float32, n), torch.ones(n, device="cuda")
    w[n - 2] = INF
    x[:, n - 2] = 1.0
    for group in (None, 32):
        size = group or n
        out, scales = torch.ones(2, n, device="cuda").to(kind), torch.ones(2, -(-n // size), device="cuda")
        algo.rms_norm(out, x, w, scales=scales, group=group)
        low = (n - 2) // size * size
        rest = torch.arange(low, min(low + size, n), device="cuda")
        assert (scales[:, low // size] == INF).all() and torch.isnan(out[:, n - 2].float()).all()
        assert (out.float()[:, rest[rest != n - 2]] == 0).all()
        assert torch.isfinite(scales[:, :low // size]).all() and torch.isfinite(out.float()[:, :low]).all()
