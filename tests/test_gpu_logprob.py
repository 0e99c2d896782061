"""GPU: token log probabilities and their gradient (a3b_token_logprobs, a3b_token_logprobs_backward) against the formulas
in 64 bits.

Tolerances, with u = 2^-24 (half a step of fp32 at 1) and V logits a row. The exponents d = (x - m) c carry three
roundings (the difference, c, the product), each e^.. the two units of ex2.approx (2^-22), and a sum of N positive terms
at most N u relative. Weighted with the terms themselves |d| averages to at most ln V. So
    ln s (and lse, logp beside their own roundings of u relative each) is off by at most
        T(V) = (N + 3 ln V + 4) u,   N = additions one after the other <= V / 256 + 64 + 20,
    the entropy ln s - u/s by at most T(V) plus the relative error of sum |d| e^d, the same terms with weights <= 1 + ln V:
        3 T(V) (1 + ln V).
Gradient element p (A + B t): p has relative error 2^-22 + 2^-22 |t|, the factors a few u, the stored value half a step of
its type."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0**-24
INF = math.inf


def tol_sum(v):
    return (v / 256 + 84 + 3 * math.log(v + 1) + 4) * U


def oracle(x, scale=1.0, where="cpu"):
    """q (log probabilities), lse and entropy of 2-D logits in 64 bits, by the documented rules."""
    z = x.double().to(where) * scale
    m = z.amax(-1, keepdim=True)
    safe = torch.where(torch.isinf(m), torch.zeros_like(m), m)
    ln_s = torch.log(torch.exp(z - safe).sum(-1, keepdim=True))
    lse = torch.where(m == INF, m, safe + ln_s)
    # not z - lse: next to the lowest value of fp32 that loses ln s even in 64 bits
    q = torch.where(lse == -INF, z, torch.where(m == INF, z - lse, (z - safe) - ln_s))
    p = torch.exp(q)
    h = -torch.where((p == 0) & (q == -INF), torch.zeros_like(p), p * q).sum(-1)
    h = torch.where(m[:, 0] == INF, torch.full_like(h, math.nan), h)
    return q, lse[:, 0], h


def ranks(x, k, where="cpu"):
    """indices of the k largest per row: NaN above all, -0 equal to 0, ties to the lower index"""
    return torch.sort(x.float().to(where) + 0.0, dim=-1, descending=True, stable=True)[1][:, :k]


def close(got, want, tol):
    got, want = got.double().cpu().flatten(), want.double().cpu().flatten()
    tol = torch.as_tensor(tol, dtype=torch.float64).expand_as(want) if not torch.is_tensor(tol) else tol.cpu().flatten()
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    rest = ~fine & ~torch.isnan(want)
    assert torch.equal(got[rest], want[rest])
    bad = (got[fine] - want[fine]).abs() > tol[fine]
    assert not bad.any(), ((got[fine] - want[fine]).abs().max(), tol[fine].max())


def forward(x, t, top=0, scale=1.0, want=("logp", "entropy", "lse")):
    from alpaka3_b200 import algo
    shape, dev = x.shape[:-1], x.device
    out = {k: torch.full(shape, 77.0, device=dev) for k in want}
    tops = {}
    if top:
        tops = {"top_logp": torch.full((*shape, top), 77.0, device=dev),
                "top_index": torch.full((*shape, top), -7, dtype=t.dtype if t is not None else torch.int64, device=dev)}
    algo.token_logprobs(out.get("logp"), x, t, entropy=out.get("entropy"), lse=out.get("lse"), scale=scale, **tops)
    return {**out, **tops}


def check_forward(x, t, top=0, scale=1.0, got=None):
    got = got or forward(x, t, top, scale)
    v = x.shape[-1]
    x2, t2 = x.reshape(-1, v), t.reshape(-1).cpu().long()
    q, lse, h = oracle(x2, scale)
    counts = (t2 >= 0) & (t2 < v)
    logp = torch.where(counts, q.gather(1, t2.clamp(0, v - 1)[:, None])[:, 0], torch.zeros(len(t2), dtype=torch.float64))
    tl = tol_sum(v)
    close(got["logp"], logp, tl + 4 * U * logp.abs().nan_to_num(posinf=0) + 4 * U)
    close(got["lse"], lse, tl + 4 * U * lse.abs().nan_to_num(posinf=0) + 4 * U)
    close(got["entropy"], h, 3 * tl * (1 + math.log(v + 1)))
    if top:
        order = ranks(x2, top)
        assert torch.equal(got["top_index"].reshape(-1, top).cpu().long(), order)
        close(got["top_logp"], q.gather(1, order), tl + 4 * U * q.gather(1, order).abs().nan_to_num(posinf=0) + 4 * U)
    return got


def make(rows, v, dtype, seed=0, spread=3.0):
    g = torch.Generator(device="cuda").manual_seed(seed + 7 * v + rows)
    x = (torch.randn(rows, v, generator=g, device="cuda") * spread).to(dtype)
    t = torch.randint(0, v, (rows,), generator=g, device="cuda")
    return x, t


DTYPES = [torch.float32, torch.float16, torch.bfloat16]
# one logit; below, at and above a pack, a warp's packs, a block's tile; odd sizes; several tiles
VOCABS = [1, 2, 7, 8, 9, 31, 33, 257, 1000, 2047, 2048, 2049, 4100, 8192, 16384, 16385, 32000, 50257, 131072, 140001]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("v", VOCABS)
def test_forward_against_64_bits(cuda, dtype, v):
    for rows, top, scale in ((1, min(v, 20), 1.0), (5, 0, 0.7), (3, min(v, 32), 1.3), (37, 1, 1.0)):
        x, t = make(rows, v, dtype, seed=top)
        if rows > 2:
            t[1] = -100
            t[2] = v  # outside: no token
        check_forward(x, t, top, scale)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("v", [5, 257, 2100, 20001, 70000, 150000])
def test_ties_and_masks(cuda, dtype, v):
    """Rows of equal values, of few finite ones, of nothing but -infinity, of the type's lowest value, of both; sorted
    rows (every tile brings new largest elements); zeros of either sign."""
    top = min(v, 32)
    g = torch.Generator(device="cuda").manual_seed(v)
    rows = []
    rows.append(torch.zeros(v))
    rows.append(torch.full((v,), -INF))
    few = torch.full((v,), -INF)
    few[torch.randperm(v, generator=torch.Generator().manual_seed(v))[:3]] = torch.tensor([1.0, 2.0, 2.0])[:v]
    rows.append(few)
    low = torch.full((v,), torch.finfo(dtype).min)
    rows.append(low.clone())
    low[::2] = -INF
    rows.append(low.clone())
    low[v // 2] = 3.0
    rows.append(low)
    rows.append(torch.linspace(-20, 20, v))
    rows.append(torch.linspace(20, -20, v))
    sign = torch.zeros(v)
    sign[1::2] = -0.0
    rows.append(sign)
    two = torch.zeros(v)
    two[v // 3:] = 1.0
    rows.append(two)
    last = torch.full((v,), -INF)
    last[v - 1] = -5.0
    rows.append(last)
    x = torch.stack(rows).to(dtype).cuda()
    t = torch.randint(0, v, (len(rows),), generator=g, device="cuda")
    check_forward(x, t, top)
    check_forward(x, t, 1)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("v", [6, 300, 9000, 40000])
def test_infinities_and_nan(cuda, dtype, v):
    x, t = make(6, v, dtype)
    x[0, v // 2] = math.nan
    x[1, v - 1] = INF
    x[2, 0] = INF
    x[2, v // 3] = INF
    x[3, v // 2] = INF
    x[3, 1] = math.nan
    x[4, 1:] = -INF
    t[1], t[2], t[4] = v - 1, 1, 0
    got = check_forward(x, t, 3)
    assert got["logp"][4].item() == 0.0 and got["entropy"][4].item() == 0.0


def test_large_and_small_values(cuda):
    """Far from zero the differences to the maximum count; scale only multiplies them."""
    x, t = make(4, 5000, torch.float32)
    x[0] += 1e4
    x[1] -= 1e4
    x[2] *= 1e3
    x[3] *= 1e-30
    check_forward(x, t, 5)
    check_forward(x, t, 5, scale=0.01)


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_and_alignment(cuda, dtype):
    v = 1003
    g = torch.Generator(device="cuda").manual_seed(1)
    buf = (torch.randn(4, 6, v + 5, generator=g, device="cuda") * 3).to(dtype)
    t = torch.randint(0, v, (4, 5), generator=g, device="cuda")
    for x in (buf[:, :-1, :v], buf[:, 1:, 5:], buf[:, :5, 1:v + 1], buf.flip(0)[:, :-1, 3:v + 3]):
        check_forward(x, t, 4)
    x = buf.transpose(0, 1)[:5, :, :v]
    check_forward(x, t.t().contiguous(), 4)
    one = buf[2, 3, 2:v + 2]  # a single row without leading dimensions
    check_forward(one, t[0, 0].reshape(()), 3)
    wide = buf[1, 1, :v].expand(7, v)  # the same row again and again
    check_forward(wide, torch.arange(7, device="cuda"), 2)


def test_int32_indices_and_missing_outputs(cuda):
    x, t = make(9, 5003, torch.bfloat16)
    full = check_forward(x, t, 6)
    got = forward(x, t.int(), 6)
    assert got["top_index"].dtype == torch.int32
    for k in full:
        assert torch.equal(got[k].long() if k == "top_index" else got[k], full[k])
    for want in (("logp",), ("entropy",), ("lse",), ("lse", "entropy")):
        some = forward(x, t if "logp" in want else None, 0, want=want)
        for k in want:
            # both are off by at most the bounds of check_forward; |logp|, |lse| < 40 here
            close(some[k], full[k], 2 * (3 * tol_sum(5003) * (1 + math.log(5004)) + 4 * U * 41))
    only = forward(x, None, 6, want=())
    assert torch.equal(only["top_index"], full["top_index"])
    from alpaka3_b200 import algo
    empty = torch.empty(0, 50, device="cuda")
    algo.token_logprobs(torch.empty(0, device="cuda"), empty, torch.empty(0, dtype=torch.int64, device="cuda"))


def test_rows_do_not_touch_neighbours(cuda):
    """What lies before, between and behind the outputs and the gradient's rows stays as it was."""
    from alpaka3_b200 import algo
    x, t = make(6, 1001, torch.bfloat16)
    lse = forward(x, t)["lse"]
    store = torch.full((8, 1010), 5.0, dtype=torch.bfloat16, device="cuda")
    g = torch.ones(6, device="cuda")
    algo.token_logprobs_backward(store[1:7, 3:1004], x, t, lse, grad_logp=g)
    assert (store[0] == 5).all() and (store[7] == 5).all() and (store[:, :3] == 5).all() and (store[:, 1004:] == 5).all()
    outs = torch.full((8, 3), 9.0, device="cuda")
    algo.token_logprobs(outs[1:7].reshape(-1)[:6], x, t)
    assert (outs.reshape(-1)[9:] == 9).all() and (outs.reshape(-1)[:3] == 9).all()


# many rows: a quarter, half or whole warp a row, a warp with several tiles, two and four warps, last tiles nearly empty
MANY = [(8192, 5003), (8200, 2060), (4100, 9001), (2048, 17011), (2051, 33000), (8192, 700), (8192, 1031),
        (20000, 65), (9001, 130), (8193, 262), (9000, 300), (8300, 517), (65537, 3)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,v", MANY)
def test_many_rows(cuda, dtype, rows, v):
    """Every kind of row among ordinary ones: constant, rising, falling, few left, none left, two values, low masks."""
    x, t = make(rows, v, dtype)
    x[0::97] = 0.0
    x[1::97] = torch.linspace(-30, 30, v, device="cuda").to(dtype)
    x[2::97] = torch.linspace(30, -30, v, device="cuda").to(dtype)
    x[3::97, 2:] = -INF
    x[4::97] = -INF
    x[5::97] = (torch.arange(v, device="cuda") % 7 == 0).to(dtype)
    x[6::97, 1:] = torch.finfo(dtype).min
    x[7::97, v // 2:] = 40.0
    x[8::97, -1] = 50.0
    x[9::97, v // 3] = math.nan
    top = min(v, 32)
    for k in (top, min(v, 8), min(v, 4)):
        got = forward(x, t, k)
        q, lse, h = oracle(x, where="cuda")
        tl = tol_sum(16 * v)  # a team of 8 threads, two sums each: V / 16 additions; a warp: V / 64
        picked = q.gather(1, t[:, None])[:, 0]
        size = 4 * U * (picked.abs().nan_to_num(0.0, posinf=0.0) + lse.abs().nan_to_num(0.0, posinf=0.0) + 1)
        close(got["logp"], picked, tl + size)
        close(got["lse"], lse, tl + size)
        close(got["entropy"], h, 3 * tl * (1 + math.log(v + 1)))
        order = ranks(x, k, where="cuda")
        assert torch.equal(got["top_index"], order)
        best = q.gather(1, order)
        close(got["top_logp"], best, tl + 4 * U * (best.abs().nan_to_num(0.0, posinf=0.0) + 1))
        # without the entropy another kernel runs; without alternatives a third
        plain = forward(x, t, k, want=("logp", "lse"))
        assert torch.equal(plain["top_index"], order)
        bare = forward(x, t, want=("logp", "lse"))
        for some in (plain, bare, forward(x, t)):
            close(some["logp"], picked, tl + size)
            close(some["lse"], lse, tl + size)


@pytest.mark.parametrize("dtype", DTYPES)
def test_very_long_rows(cuda, dtype):
    """Millions of logits a row: many tiles a slice; one row with its best at the very end."""
    v = 5_000_003
    x, t = make(2, v, dtype)
    x[1, -40:] = torch.linspace(20, 30, 40, device="cuda").to(dtype)
    t[1] = v - 1
    check_forward(x, t, 32)
    check_backward(x, t)


def test_many_rows_gradient(cuda):
    """Rows of many chunks and rows of a part of one, in one launch of more than 2^16 warps."""
    from alpaka3_b200 import algo
    for rows, v, dtype in ((20011, 65, torch.bfloat16), (3000, 4099, torch.float32)):
        x, t = make(rows, v, dtype)
        f = forward(x, t)
        g = torch.randn(rows, device="cuda")
        res = torch.empty_like(x)
        algo.token_logprobs_backward(res, x, t, f["lse"], grad_logp=g)
        q = x.double() - f["lse"].double()[:, None]
        p = torch.exp(q)
        want = -g.double()[:, None] * p
        want.scatter_add_(1, t[:, None], g.double()[:, None])
        tol = g.abs().double()[:, None] * (p * 2.0**-21 * (1 + q.abs()) + 2 * U)
        tol += want.abs() * torch.finfo(dtype).eps / 2
        assert ((res.double() - want).abs() <= tol).all()


def test_repeated_calls_give_the_same_bits(cuda):
    x, t = make(64, 30011, torch.bfloat16)
    runs = [forward(x, t, 20) for _ in range(4)]
    for r in runs[1:]:
        assert all(torch.equal(r[k], runs[0][k]) for k in r)


# ---------------------------------------------------------------------------------------------------- gradient
def check_backward(x, t, scale=1.0, use=("logp", "entropy", "lse"), out=None, seed=3):
    from alpaka3_b200 import algo
    v, dev = x.shape[-1], x.device
    shape = x.shape[:-1]
    f = forward(x, t, scale=scale)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    g = {k: torch.randn(shape, generator=gen, device=dev) if k in use else None for k in ("logp", "entropy", "lse")}
    x2 = x.reshape(-1, v).double().cpu()  # before an in-place call
    res = torch.full_like(x, 55.0) if out is None else out
    algo.token_logprobs_backward(res, x, t if "logp" in use else None, f["lse"],
                                 entropy=f["entropy"] if "entropy" in use else None, grad_logp=g["logp"],
                                 grad_entropy=g["entropy"], grad_lse=g["lse"], scale=scale)
    lse, ent = f["lse"].reshape(-1).double().cpu(), f["entropy"].reshape(-1).double().cpu()
    zero = torch.zeros_like(lse)
    gp, gh, gl = ((g[k].reshape(-1).double().cpu() if g[k] is not None else zero) for k in ("logp", "entropy", "lse"))
    t2 = t.reshape(-1).cpu().long()
    counts, some = ((t2 >= 0) & (t2 < v)), lse != -INF
    gp = torch.where(counts & some, gp, zero)
    gh, gl = torch.where(some, gh, zero), torch.where(some, gl, zero)
    lse = torch.where(some, lse, zero)
    # Next to 2^100 a step of lse's fp32 is 2^76: the difference from a product in 64 bits would be that rounding alone. The
    # product is rounded as lse was (the scale to fp32, then the product), so that a row of one value is at 0, not -ln V.
    rounded = (x2 * torch.tensor(scale, dtype=torch.float32).double().item()).float().double()
    product = torch.where((lse.abs() > 2.0**80)[:, None], rounded, x2 * scale)
    q = product - lse[:, None]
    p = q.exp()
    pq = torch.where(p == 0, torch.zeros_like(p), p * (q + ent[:, None]))
    want = p * (gl - gp)[:, None] - gh[:, None] * pq
    want.scatter_add_(1, t2.clamp(0, v - 1)[:, None], gp[:, None])
    want *= scale
    mag = (gl.abs() + gp.abs() + (gh * ent).abs())[:, None] + (gh[:, None] * q).abs()
    mag = torch.where(p == 0, torch.zeros_like(mag), mag)
    type_step = torch.finfo(x.dtype).eps / 2
    # p's error grows with |t| = |q| / ln 2; under the smallest normal number a type loses a fixed amount
    tol = scale * p * mag * (2.0**-21 + 2.0**-21 * q.abs().nan_to_num(posinf=0)) + want.abs() * (type_step + 2 * U)
    # The kernel forms ln p / ln 2 as a fused c x - lse / ln 2, both factors rounded to fp32, plus a rest that carries
    # what the two roundings left: |rest| <= 2 * 2^-24 |lse| / ln 2 < 2^-22 |lse|. The rest is rounded too, and the sum of
    # two terms that cancel: 2^-24 |rest| each, 2^-44 |lse| with room for both. It counts where q itself is 0.
    tol = tol + scale * p * gh.abs()[:, None] * torch.where(some, lse.abs(), zero)[:, None] * 2.0**-44
    tol = tol.nan_to_num(0.0) + gp.abs()[:, None] * scale * 2 * U + torch.finfo(x.dtype).tiny * max(type_step * 2, 2.0**-8)
    close(res.reshape(-1, v), want, tol)
    return res


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("v", [1, 7, 8, 33, 257, 2049, 8193, 16400, 50257])
def test_gradient_against_64_bits(cuda, dtype, v):
    for rows, use, scale in ((1, ("logp",), 1.0), (6, ("logp", "entropy", "lse"), 0.7), (3, ("entropy",), 1.0),
                             (2, ("lse",), 1.4)):
        x, t = make(rows, v, dtype, seed=rows)
        if rows > 2:
            t[1] = -100
            t[2] = v
        check_backward(x, t, scale, use)


@pytest.mark.parametrize("dtype", DTYPES)
def test_gradient_masked_rows(cuda, dtype):
    v = 3001
    x, t = make(6, v, dtype)
    x[0] = -INF
    x[1, ::2] = -INF
    x[2] = torch.finfo(dtype).min
    x[3, 1:] = -INF
    x[4, ::3] = torch.finfo(dtype).min
    t[1], t[3] = 0, 0  # a masked token; the only one left
    res = check_backward(x, t)
    assert (res[0] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_gradient_strides_alignment_in_place(cuda, dtype):
    g = torch.Generator(device="cuda").manual_seed(5)
    buf = (torch.randn(3, 5, 1010, generator=g, device="cuda") * 3).to(dtype)
    t = torch.randint(0, 1003, (3, 4), generator=g, device="cuda")
    for a in (0, 1, 3):
        for b in (0, 2, 3):
            store = torch.zeros(3, 5, 1010, dtype=dtype, device="cuda")
            check_backward(buf[:, :-1, a:a + 1003], t, out=store[:, 1:, b:b + 1003])
    check_backward(buf[:, :-1, :1003], t, out=torch.empty(3, 4, 1003, dtype=dtype, device="cuda"))
    check_backward(buf[:, :-1, :1003].contiguous(), t, out=torch.empty_like(buf)[:, 1:, 2:1005])
    want = check_backward(buf[:, :-1, 1:1004], t)
    x = buf[:, :-1, 1:1004]
    assert torch.equal(check_backward(x, t, out=x), want)  # in place


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("v", [1, 3, 15, 64, 130, 135, 255, 257, 263, 519])
def test_gradient_many_short_rows(cuda, dtype, v):
    """Rows enough for teams of a quarter warp, and the vocabularies at which they stop: odd starts, masks, in place."""
    x, t = make(2053, v, dtype)
    x[0::97] = -INF
    x[1::97, 1:] = -INF
    x[2::97] = torch.finfo(dtype).min
    x[3::97, ::2] = -INF
    t[4::97], t[5::97], t[1::97] = -100, v, 0
    t[6::97], t[7::97] = 0, v - 1
    want = check_backward(x, t, 0.7)
    assert (want[0::97] == 0).all()
    store = torch.zeros(2053, v + 5, dtype=dtype, device="cuda")
    check_backward(x, t, 0.7, out=store[:, 1:v + 1])
    assert (store[:, 0] == 0).all() and (store[:, v + 1:] == 0).all()
    assert torch.equal(check_backward(x, t, 0.7, out=x), want)


def test_gradient_against_differences(cuda):
    """Central differences of the forward kernel's own outputs, in fp32 with a step of 2^-6: the third derivative of
    these functions is below 4 in the tested rows, so the quotient is off by at most 4 h^2 / 6 < 2e-4, and the outputs'
    error T(V) + 4 u |value| over the step by less than 2 * 6e-6 / 2^-6 = 8e-4."""
    from alpaka3_b200 import algo
    v, h = 50, 2.0**-6
    x, t = make(1, v, torch.float32, spread=1.5)
    f = forward(x, t)
    for name in ("logp", "entropy", "lse"):
        grad = torch.empty_like(x)
        algo.token_logprobs_backward(grad, x, t, f["lse"], entropy=f["entropy"],
                                     **{"grad_" + name: torch.ones(1, device="cuda")})
        up = forward(x + h * torch.eye(v, device="cuda"), t.expand(v).contiguous())[name]
        down = forward(x - h * torch.eye(v, device="cuda"), t.expand(v).contiguous())[name]
        assert ((up - down) / (2 * h) - grad[0]).abs().max().item() < 1e-3


# ----------------------------------------------------------------------------- streams, graphs, sizes, refusals
def test_other_stream_and_captured_graphs(cuda):
    from alpaka3_b200 import algo
    x, t = make(33, 20011, torch.bfloat16)
    want = forward(x, t, 8)
    ones = torch.ones(33, device="cuda")
    side = torch.cuda.Stream()
    got = {k: torch.zeros_like(w) for k, w in want.items()}
    side.wait_stream(torch.cuda.current_stream())  # what the outputs were filled with is in place by then
    algo.token_logprobs(got["logp"], x, t, entropy=got["entropy"], lse=got["lse"], top_logp=got["top_logp"],
                        top_index=got["top_index"], stream=side)
    side.synchronize()
    assert all(torch.equal(got[k], want[k]) for k in want)

    # two graphs captured one after the other, replayed at the same time on two streams
    graphs, results = [], []
    for k in range(2):
        graph = torch.cuda.CUDAGraph()
        xs = x.clone()
        out = {n: torch.zeros_like(w) for n, w in want.items()}
        grad = torch.zeros_like(xs)
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            algo.token_logprobs(out["logp"], xs, t, entropy=out["entropy"], lse=out["lse"], top_logp=out["top_logp"],
                                top_index=out["top_index"])
            algo.token_logprobs_backward(grad, xs, t, out["lse"], grad_logp=ones)
        graphs.append(graph)
        results.append((xs, out, grad))
    y, _ = make(33, 20011, torch.bfloat16, seed=9)
    results[1][0].copy_(y)
    other = forward(y, t, 8)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for (xs, out, grad), expect in zip(results, (want, other)):
        assert all(torch.equal(out[k], expect[k]) for k in expect)
        direct = torch.zeros_like(grad)
        algo.token_logprobs_backward(direct, xs, t, expect["lse"], grad_logp=ones)
        assert torch.equal(grad, direct) and direct.float().abs().sum() > 0


@pytest.mark.slow
def test_offsets_past_32_bits(cuda):
    """2.7e9 bf16 logits: the last rows lie past element 2^31 and byte 2^32."""
    from alpaka3_b200 import algo
    rows, v = 41000, 65537
    x = torch.zeros(rows, v, dtype=torch.bfloat16, device="cuda")
    tail, _ = make(3, v, torch.bfloat16)
    x[-3:] = tail
    t = torch.full((rows,), 5, device="cuda")
    got = forward(x, t, 4)
    check_forward(tail, t[-3:], 4, got={k: w[-3:] for k, w in got.items()})
    assert (got["top_index"][:-3] == torch.arange(4, device="cuda")).all()
    algo.token_logprobs_backward(x, x, t, got["lse"], grad_logp=torch.ones(rows, device="cuda"))
    g = torch.empty_like(tail)
    algo.token_logprobs_backward(g, tail, t[-3:].contiguous(), got["lse"][-3:].contiguous(),
                                 grad_logp=torch.ones(3, device="cuda"))
    assert torch.equal(x[-3:], g)


def test_refusals(cuda):
    from alpaka3_b200 import algo, capi
    x, t = make(4, 100, torch.float32)
    lp = torch.empty(4, device="cuda")
    tl, ti = torch.empty(4, 3, device="cuda"), torch.empty(4, 3, dtype=torch.int64, device="cuda")
    for bad in (dict(logits=x.double()), dict(logits=x.long()), dict(targets=t.float()), dict(logp=lp.double()),
                dict(top_logp=tl, top_index=ti.int())):
        with pytest.raises(TypeError):
            algo.token_logprobs(**{"logp": lp, "logits": x, "targets": t, **bad})
    for bad in (dict(logits=x.cpu()), dict(logits=x.t()), dict(logits=x[:, ::2]), dict(targets=t[:3]),
                dict(targets=t.cpu()), dict(logp=lp[:2]), dict(top_logp=tl), dict(top_logp=tl, top_index=ti[:, :2]),
                dict(targets=None), dict(entropy=torch.empty(8, device="cuda")[::2])):
        with pytest.raises(ValueError):
            algo.token_logprobs(**{"logp": lp, "logits": x, "targets": t, **bad})
    for bad in (dict(scale=0.0), dict(scale=-1.0), dict(scale=INF), dict(scale=math.nan),
                dict(top_logp=torch.empty(4, 33, device="cuda"),
                     top_index=torch.empty(4, 33, dtype=torch.int64, device="cuda")), dict(logp=None)):
        with pytest.raises(capi.A3BError):
            algo.token_logprobs(**{"logp": lp, "logits": x, "targets": t, **bad})
    with pytest.raises(capi.A3BError):  # more alternatives than logits
        algo.token_logprobs(None, x[:, :2], None, top_logp=tl, top_index=ti)
    g = torch.empty_like(x)
    for bad in (dict(grad_logits=g.half()), dict(grad_logits=g[:3]), dict(lse=None), dict(lse=lp[:2]),
                dict(grad_logits=g.t().contiguous().t())):
        with pytest.raises(ValueError):
            algo.token_logprobs_backward(**{"grad_logits": g, "logits": x, "targets": t, "lse": lp, "grad_logp": lp, **bad})
    store = torch.empty(500, device="cuda")
    xs = store[:400].view(4, 100)
    for bad in (dict(grad_logits=store[100:].view(4, 100), logits=xs), dict(grad_entropy=lp), dict(targets=None),
                dict(grad_logits=store[:100].expand(4, 100)), dict(scale=0.0)):
        with pytest.raises(capi.A3BError):
            algo.token_logprobs_backward(**{"grad_logits": g, "logits": x, "targets": t, "lse": lp, "grad_logp": lp, **bad})


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("v", [512, 513, 516, 517, 518, 1024, 1030, 1031, 1032, 1033, 1034, 1035, 1036, 1037, 1038, 1039, 2056])
def test_gradient_of_lowest_values_in_place(cuda, dtype, v):
    """Rows of the type's lowest value (for fp32 and bf16 element by element), at every start, where the last chunk has no
    pack of its own: in place the same bits as apart. Three ordinary rows lie between."""
    from alpaka3_b200 import algo
    pitch = v + 16
    g = torch.Generator(device="cuda").manual_seed(v)
    buf = (torch.randn(6, pitch, generator=g, device="cuda") * 3).to(dtype)
    t = torch.randint(0, v, (6,), generator=g, device="cuda")
    t[2] = v - 1
    one = torch.ones(6, device="cuda")
    for start in range(8):
        store = buf.clone()
        x = store[:, start:start + v]
        x[::2] = torch.finfo(dtype).min
        f = forward(x, t)
        apart = torch.full((6, pitch), 4.0, dtype=dtype, device="cuda")[:, start:start + v]
        for out in (apart, x):
            algo.token_logprobs_backward(out, x, t, f["lse"], entropy=f["entropy"], grad_logp=one, grad_entropy=-one,
                                         grad_lse=0.5 * one)
        assert torch.isfinite(apart).all() and torch.equal(x, apart), start
        assert torch.equal(store[:, :start], buf[:, :start]) and torch.equal(store[:, start + v:], buf[:, start + v:])


# ------------------------------------------------------------------------------------ logits far from zero
# ln p stays as the formula has it while |z| grows: only the steps of z itself (and of lse) do.
def far_values(dtype, scale):
    """+-10^3 .. +-10^38, as far as the type and scale * value hold them."""
    top = 6e4 if dtype == torch.float16 else 2e38
    return [s * 10.0**k for k in range(3, 39) for s in (1.0, -1.0) if 10.0**k <= top and 10.0**k * max(scale, 1.0) < 2e38]


def far_rows(v, dtype, scale, seed=0):
    """For each of these values: a row of it alone, all but three logits at it, the first or the second half at it, and a
    row spread around it; as many targets, some of them on such logits."""
    g = torch.Generator(device="cuda").manual_seed(seed + v)
    values = far_values(dtype, scale)
    base = (torch.randn(5 * len(values), v, generator=g, device="cuda") * 3)
    for i, w in enumerate(values):
        rows = base[5 * i:5 * i + 5]
        keep = torch.randint(0, v, (3,), generator=g, device="cuda")
        rows[0] = w
        kept = rows[1, keep].clone()
        rows[1] = w
        rows[1, keep] = kept
        rows[2, :v // 2 + 1] = w
        rows[3, v // 2:] = w
        rows[4] += w
    t = torch.randint(0, v, (len(base),), generator=g, device="cuda")
    return base.to(dtype), t


def check_far(x, t, top, scale, additions):
    """Exponents are t = c x + offset with offset = -(c high) as rounded to fp32: half a step of it, R <= 2^-24 |c high|, is
    in every t, and at most 32 (beyond |c high| = 2^30 the offset is exact). So a t of size R + |d| is rounded by u (R + |d|)
    at most, its power is off by R u more than T(V) counts, s / 2^R by as much; u / s - R takes two sums of terms R times
    as large, each off by T(V) at most: 2 R T(V) more in the entropy."""
    v = x.shape[-1]
    got = forward(x, t, top, scale)
    q, lse, h = oracle(x, scale, where="cuda")
    r = (x.double().amax(-1).abs() * scale * 1.4427 * U).clamp(max=32.0)
    tl = (additions + 20 + 3 * math.log(v + 1) + 4) * U + r * U
    logp = q.gather(1, t[:, None])[:, 0]
    close(got["logp"], logp, tl + 4 * U * (logp.abs() + 1))
    close(got["lse"], lse, tl + 4 * U * (lse.abs() + 1))
    close(got["entropy"], h, 3 * tl * (1 + math.log(v + 1)) + 2 * r * tl)
    if top:
        order = ranks(x, top, where="cuda")
        assert torch.equal(got["top_index"], order)
        best = q.gather(1, order)
        close(got["top_logp"], best, tl[:, None] + 4 * U * (best.abs() + 1))


@pytest.mark.parametrize("scale", [1.0, 0.7, 1 / 0.3, 10.0, 1e6])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("v", [5, 300, 2100, 9000, 50257, 140001])
def test_far_logits(cuda, dtype, v, scale):
    """All rows in one call, then a few rows a call (slices of a row over a cluster where it is long)."""
    x, t = far_rows(v, dtype, scale)
    top = min(v, 5)
    check_far(x, t, top, scale, v / 64 + 64)
    step = 9 if v > 20000 else len(x)
    for lo in range(0, len(x), step):
        check_far(x[lo:lo + step], t[lo:lo + step], top if lo % 2 else 0, scale, v / 64 + 64)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,v", [(8200, 65), (8200, 260), (8200, 700), (8192, 5003), (4100, 9001), (2048, 17011)])
def test_far_logits_in_many_rows(cuda, dtype, rows, v):
    """The same rows over and over, for the teams that many rows get: a part of a warp, a warp, two and four."""
    x, t = far_rows(v, dtype, 0.7)
    again = torch.arange(rows, device="cuda") % len(x)
    for top in (0, 3):
        check_far(x[again], t[again], top, 0.7, v / 16 + 64)  # 8 threads a row, two sums each


def test_entropy_and_lse_alone_of_far_logits(cuda):
    """The kernels without entropy, and without a token."""
    x, t = far_rows(20011, torch.float32, 1.0)
    full = forward(x, t)
    for want in (("logp",), ("entropy",), ("lse",), ("logp", "lse")):
        some = forward(x, t if "logp" in want else None, want=want)
        for k in want:
            assert torch.isfinite(some[k]).all()
            # both within check_far's bounds; a masked token's logp or a row's lse may be of any size
            size = full[k].abs().double()
            close(some[k], full[k], 2 * (3 * (20011 / 64 + 120 + 32) * U * (1 + math.log(20012) + 32) + 4 * U * size))


def check_far_backward(x, t, scale, seed=3):
    """As check_backward, with two things more. Above |lse| = 2^24 the documented product is rounded to fp32 as lse was. Below
    it the rest that goes into the factors (|rest| <= 2^-22 |lse|, three roundings of 2^-24 each and their ln 2) puts an
    error of less than 2^-44 |lse| on every p. And a power below 2^-126 is flushed to zero (2^-122 with the rest's 2^4 at
    most apart from it): what has so small a p is off by its own term at most. Returns p; in place gives the same bits."""
    from alpaka3_b200 import algo
    f = forward(x, t, scale=scale)
    gen = torch.Generator(device="cuda").manual_seed(seed)
    g = [torch.randn(len(x), generator=gen, device="cuda") for _ in range(3)]
    args = dict(entropy=f["entropy"], grad_logp=g[0], grad_entropy=g[1], grad_lse=g[2], scale=scale)
    res = torch.full_like(x, 55.0)
    algo.token_logprobs_backward(res, x, t, f["lse"], **args)
    lse, ent = f["lse"].double()[:, None], f["entropy"].double()[:, None]
    counts = ((t >= 0) & (t < x.shape[-1]))[:, None]
    gp, gh, gl = (k.double()[:, None] for k in g)
    gp = torch.where(counts, gp, torch.zeros_like(gp))
    z = x.double() * scale
    rounded = (x.double() * torch.tensor(scale, dtype=torch.float32).double().item()).float().double()
    q = torch.where(lse.abs() > 2.0**24, rounded, z) - lse
    p = q.exp()
    want = p * ((gl - gp) - gh * (q + ent))
    want.scatter_add_(1, t.clamp(min=0)[:, None], gp)
    want *= scale
    mag = (gl.abs() + gp.abs() + (gh * ent).abs()) + (gh * q).abs()
    rest = lse.abs() * 2.0**-44 * (lse.abs() <= 2.0**24)
    step = torch.finfo(x.dtype).eps / 2
    tol = scale * p * (mag * (2.0**-21 * (1 + q.abs()) + rest) + gh.abs() * rest) + want.abs() * (step + 2 * U)
    tol = tol + gp.abs() * scale * 2 * U + torch.finfo(x.dtype).tiny * max(step * 2, 2.0**-8)
    close(res, want, tol + scale * (p * mag).where(p < 2.0**-122, torch.zeros_like(p)))
    y = x.clone()
    algo.token_logprobs_backward(y, y, t, f["lse"], **args)
    assert torch.equal(y, res)
    return p


@pytest.mark.parametrize("scale", [1.0, 0.7, 1 / 0.3, 10.0, 1e6])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("v", [5, 300, 2100, 9001, 50257])
def test_gradient_of_far_logits(cuda, dtype, v, scale):
    if dtype == torch.float16 and scale > 100:
        pytest.skip("the gradients leave fp16's range")
    x, t = far_rows(v, dtype, scale)
    t[::7] = -100
    p = check_far_backward(x, t, scale)
    # z <= lse stays true of the rounded numbers, so no probability is far above 1 however large lse's own step is
    assert p.max().item() <= math.exp(2.0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("v", [64, 130, 257])
def test_gradient_of_far_logits_in_many_short_rows(cuda, dtype, v):
    x, t = far_rows(v, dtype, 0.7)
    again = torch.arange(2053, device="cuda") % len(x)
    check_far_backward(x[again], t[again], 0.7)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("v", [5, 130, 1032, 4099])
def test_gradient_of_far_logits_to_other_alignments(cuda, dtype, v):
    """The gradient's rows may start and step differently from the logits': the same bits, the neighbours untouched."""
    from alpaka3_b200 import algo
    x, t = far_rows(v, dtype, 1.0)
    f = forward(x, t)
    one = torch.ones(len(x), device="cuda")
    args = dict(entropy=f["entropy"], grad_logp=one, grad_entropy=0.5 * one, grad_lse=-one)
    want = torch.full_like(x, 55.0)
    algo.token_logprobs_backward(want, x, t, f["lse"], **args)
    for a, b, pitch in ((0, 1, v + 3), (3, 0, v + 5), (1, 2, v + 8), (2, 2, v + 4)):
        src = torch.zeros(len(x), pitch, dtype=dtype, device="cuda")
        src[:, a:a + v] = x
        out = torch.full((len(x), v + 11), 9.0, dtype=dtype, device="cuda")
        algo.token_logprobs_backward(out[:, b:b + v], src[:, a:a + v], t, f["lse"], **args)
        assert torch.equal(out[:, b:b + v], want), (a, b)
        assert (out[:, :b] == 9).all() and (out[:, b + v:] == 9).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,v", [(6, 6), (6, 1033), (6, 9000), (2052, 130)])
def test_gradient_of_infinities_and_nan(cuda, dtype, rows, v):
    """A NaN makes its row's gradient NaN. Beside +infinity nothing else has a probability: a gradient of 0 but for the
    token's own term; what is infinite has none that is a number. Without and with the entropy, which is NaN there."""
    from alpaka3_b200 import algo
    x, t = make(rows, v, dtype)
    x[0::6, v // 2] = math.nan
    x[1::6, v - 1] = INF
    x[2::6, 0], x[2::6, v // 3] = INF, INF
    x[3::6, v // 2], x[3::6, 1] = INF, math.nan
    x[4::6] = -INF
    t[1::6], t[2::6] = 1, 0
    f = forward(x, t)
    one = torch.ones(rows, device="cuda")
    for more in ({}, dict(entropy=f["entropy"], grad_entropy=one), dict(grad_lse=one)):
        g = torch.full_like(x, 55.0)
        algo.token_logprobs_backward(g, x, t, f["lse"], grad_logp=3 * one, scale=1.0, **more)
        assert torch.isnan(g[0::6]).all() and torch.isnan(g[3::6]).all() and (g[4::6] == 0).all()
        assert torch.isfinite(g[5::6]).all()
        for k, holes in ((1, [v - 1]), (2, [0, v // 3])):
            want = torch.zeros(v, device="cuda")
            if k == 1:
                want[1] = 3.0  # the token's own term
            want[holes] = math.nan
            for row in g[k::6].float():
                assert torch.equal(row.nan_to_num(77.0), want.nan_to_num(77.0))
        same = x.clone()
        algo.token_logprobs_backward(same, same, t, f["lse"], grad_logp=3 * one, scale=1.0, **more)
        assert torch.equal(same.nan_to_num(77.0), g.nan_to_num(77.0))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("v", [130, 9001])
def test_lowest_values_at_a_temperature(cuda, dtype, v):
    """scale * the lowest value is below fp32's range. A row of nothing else: lse -infinity, a gradient of zeros, logp and
    entropy as for any row of one value. Beside other logits such a mask has no probability, like -infinity."""
    scale = 1 / 0.3
    x, t = make(4, v, dtype)
    x[0] = torch.finfo(dtype).min
    x[1, ::2], x[2, 3:] = torch.finfo(dtype).min, torch.finfo(dtype).min
    t[1], t[2] = 1, 4  # a token that is left, and a masked one
    got = forward(x, t, 3, scale)
    masked = x.masked_fill(x == torch.finfo(dtype).min, -INF)
    q, lse, h = oracle(masked, scale)
    logp = q.gather(1, t[:, None].cpu())[:, 0]
    logp[0], h[0] = -math.log(v), math.log(v)
    close(got["logp"], logp, tol_sum(v) + 4 * U * (logp.abs().nan_to_num(posinf=0) + 1))
    close(got["lse"], lse, tol_sum(v) + 4 * U * (lse.abs().nan_to_num(posinf=0) + 1))
    close(got["entropy"], h, 3 * tol_sum(v) * (1 + math.log(v + 1)))
    assert torch.equal(got["top_index"].cpu(), ranks(x, 3))
    from alpaka3_b200 import algo
    one = torch.ones(4, device="cuda")
    grads = []
    for logits in (x, masked):
        g = torch.full_like(x, 55.0)
        algo.token_logprobs_backward(g, logits, t, got["lse"], entropy=got["entropy"], grad_logp=one, grad_entropy=one,
                                     grad_lse=-one, scale=scale)
        grads.append(g)
    assert (grads[0][0] == 0).all() and torch.isfinite(grads[0]).all() and torch.equal(grads[0], grads[1])
