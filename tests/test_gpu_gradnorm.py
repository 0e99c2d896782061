"""GPU: norm and clipping of lists of gradients (a3b_grad_norm, a3b_clip_grads, a3b_clip_grad_norm) against 64 bits, and a
training step's tail as it is used: loss, its gradient, the weights' gradients, clipping.

Tolerances, u = 2^-24: a pack of at most 8 squares is summed in fp32 (each product and sum off by u relative of a positive
total: at most 6 u), packs in fp64: the sum is off by 6 u, its root by 3 u, stored in fp32 by u more: 4 u for l2, 7 u for
l1, u for max (no sums). fp64 inputs: n 2^-53 for n terms. A clipped element is off by the norm's error, two roundings of
the factor and the product (3 u) and half a step of its type."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0**-24
REL = {"l2": 4 * U, "l1": 7 * U, "max": U}
BF, HF, SF, DF = torch.bfloat16, torch.float16, torch.float32, torch.float64


def exact(tensors, kind):
    v = [t.double().cpu().abs().flatten() for t in tensors if t.numel()]
    if not v:
        return 0.0
    if kind == "max":
        return max(x.max().item() for x in v)
    total = math.fsum((x if kind == "l1" else x * x).sum().item() for x in v)
    return math.sqrt(total) if kind == "l2" else total


def tensors_of(spec, seed=0, spread=0.02):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [(torch.randn(n, generator=g, device="cuda") * spread).to(dt) for n, dt in spec]


def check(ins, max_norm, kind="l2", outs=None, norm_dtype=torch.float32):
    from alpaka3_b200 import algo
    norm = torch.full((1,), -3.0, dtype=norm_dtype, device="cuda")
    before = [t.clone() for t in ins]
    want = exact(ins, kind)
    lst = algo.TensorList(ins, outs)
    algo.clip_grad_norm(norm, lst, max_norm, kind)
    got = norm.item()
    wide = all(t.dtype == DF for t in ins)
    rel = 1e-13 + (2.0**-52 if norm_dtype == DF else U) if wide else REL[kind]
    assert got == want or abs(got - want) <= rel * want, (got, want)
    factor = min(1.0, max_norm / (want + 1e-6))
    for t, b, o in zip(ins, before, outs or ins):
        step = torch.finfo(t.dtype).eps / 2
        y = b.double() * factor
        small = torch.finfo(t.dtype).tiny * torch.finfo(t.dtype).eps  # smallest step below the normal numbers
        err = (o.double() - y).abs()
        own = 1e-13 if t.dtype == DF and wide else REL[kind] + 3 * U
        assert (err <= y.abs() * (own + step) + small).all(), err.max()
        if outs is not None:
            assert torch.equal(t, b)
    return got


SPECS = [
    [(1, SF)],
    [(5, BF), (0, SF), (1, HF), (3, DF)],
    [(4096, BF)],
    [(4095, SF), (4097, SF), (8193, BF), (16385, HF), (2049, DF)],
    [(n, dt) for n in (1, 2, 3, 7, 8, 9, 15, 16, 17, 100, 1000, 8191, 8192, 8193) for dt in (BF, HF, SF, DF)],
    [(1000003, BF), (77, SF), (300001, HF)],
    [(17 + 13 * (i % 7), (BF, SF)[i % 2]) for i in range(2500)],  # more tensors than one launch takes
    [(5000001, SF)],
]


@pytest.mark.parametrize("kind", ["l2", "l1", "max"])
@pytest.mark.parametrize("spec", range(len(SPECS)))
def test_norm_and_clip_against_64_bits(cuda, spec, kind):
    for max_frac in (0.3, 7.0):
        ins = tensors_of(SPECS[spec], seed=spec)
        outs = [torch.full_like(t, 9.0) for t in ins]
        limit = max(exact(ins, kind), 1e-3) * max_frac
        check(ins, limit, kind, outs)
        check([t.clone() for t in ins], limit, kind)


def test_norm_alone_and_partial(cuda):
    from alpaka3_b200 import algo
    ins = tensors_of(SPECS[5], 3)
    for kind in ("l2", "l1", "max"):
        norm = torch.empty(1, dtype=DF, device="cuda")
        part = torch.empty(1, dtype=DF, device="cuda")
        algo.grad_norm(norm, ins, kind, partial=part)
        want = exact(ins, kind)
        assert abs(norm.item() - want) <= REL[kind] * want
        assert norm.item() == (math.sqrt(part.item()) if kind == "l2" else part.item())
        only = torch.empty(1, dtype=DF, device="cuda")
        algo.grad_norm(None, ins, kind, partial=only)
        assert torch.equal(only, part)
        # two halves combined, as two ranks would
        parts = [torch.empty(1, dtype=DF, device="cuda") for _ in range(2)]
        algo.grad_norm(None, ins[:1], kind, partial=parts[0])
        algo.grad_norm(None, ins[1:], kind, partial=parts[1])
        both = torch.maximum(*parts) if kind == "max" else parts[0] + parts[1]
        a, b = [t.clone() for t in ins], [t.clone() for t in ins]
        seen = torch.empty(1, device="cuda")
        algo.clip_grads(seen, a, both, want / 3, kind)
        algo.clip_grad_norm(norm, b, want / 3, kind)
        assert abs(seen.item() - want) <= 2 * REL[kind] * want
        for s, t in zip(a, b):
            assert ((s.double() - t.double()).abs() <= t.double().abs() * (torch.finfo(s.dtype).eps + 8 * U)).all()


def test_one_rank_of_a_sharded_step(cuda):
    from alpaka3_b200 import algo, dist
    ins = tensors_of(SPECS[4], 8)
    a, b = [t.clone() for t in ins], [t.clone() for t in ins]
    n1, n2 = torch.empty(1, device="cuda"), torch.empty(1, device="cuda")
    dist.clip_grad_norm(n1, a, 0.5)
    algo.clip_grad_norm(n2, b, 0.5)
    assert torch.equal(n1, n2) and all(torch.equal(x, y) for x, y in zip(a, b))


def test_range_of_squares(cuda):
    """Squares that leave fp32's range in either direction, beside zeros and alone."""
    for v in (1e-30, 3e-23, 1e-19, 1e19, 3e30):
        for dt in (SF, BF):
            x = torch.zeros(4099, device="cuda")
            x[::7] = v
            check([x.to(dt)], 1e30, "l2", norm_dtype=DF)
            check([x.to(dt), torch.ones(33, dtype=dt, device="cuda")], 1e30, "l2", norm_dtype=DF)
    zero = [torch.zeros(100, dtype=BF, device="cuda"), torch.zeros(3, device="cuda")]
    assert check(zero, 1.0) == 0.0
    assert check([torch.full((9,), -0.0, device="cuda")], 1.0) == 0.0


@pytest.mark.parametrize("kind", ["l2", "l1", "max"])
@pytest.mark.parametrize("dtype", [BF, HF, SF, DF])
def test_infinities_and_nan(cuda, kind, dtype):
    from alpaka3_b200 import algo
    norm = torch.empty(1, device="cuda")
    x = torch.ones(5003, dtype=dtype, device="cuda")
    x[4321] = math.nan
    y = torch.ones(77, dtype=dtype, device="cuda")
    algo.clip_grad_norm(norm, [y, x], 1.0, kind)
    assert math.isnan(norm.item()) and torch.isnan(x).all() and torch.isnan(y).all()
    x = torch.ones(5003, dtype=dtype, device="cuda")
    x[11] = -math.inf
    y = torch.ones(77, dtype=dtype, device="cuda")
    algo.clip_grad_norm(norm, [x, y], 1.0, kind)
    assert norm.item() == math.inf and torch.isnan(x[11]) and x.nan_to_num(0).abs().sum() == 0 and (y == 0).all()


def test_limits_zero_and_infinite(cuda):
    from alpaka3_b200 import algo
    norm = torch.empty(1, device="cuda")
    x = torch.ones(1001, dtype=BF, device="cuda")
    algo.clip_grad_norm(norm, [x], math.inf)
    assert (x == 1).all()
    algo.clip_grad_norm(norm, [x], 0.0)
    assert (x == 0).all()
    algo.clip_grad_norm(norm, [], 1.0)
    assert norm.item() == 0.0
    algo.clip_grad_norm(norm, [torch.empty(0, device="cuda")], 1.0)
    assert norm.item() == 0.0
    algo.clip_grad_norm(None or norm, [torch.empty(0, 5, dtype=BF, device="cuda"), x], 1.0)


@pytest.mark.parametrize("dtype", [BF, HF, SF, DF])
def test_alignment_and_layouts(cuda, dtype):
    """Every alignment of input and output against one another; permuted dimensions; neighbours stay as they were."""
    for a in range(0, 9):
        for b in (0, 1, a):
            store = torch.full((9000,), 3.0, dtype=dtype, device="cuda")
            src = tensors_of([(9000, dtype)], a)[0]
            check([src[a:a + 8200]], 0.1, outs=[store[b:b + 8200]])
            assert (store[:b] == 3).all() and (store[b + 8200:] == 3).all()
    t = tensors_of([(24 * 10, dtype)], 1)[0].view(2, 3, 4, 10)
    check([t.permute(3, 1, 0, 2), t.new_ones(5, 7).t()], 0.1)


def test_a_list_used_again_and_destroyed(cuda):
    """New values in the same tensors; a list may go as soon as the call has returned."""
    from alpaka3_b200 import algo
    ins = tensors_of(SPECS[4], 2)
    lst = algo.TensorList(ins)
    norm = torch.empty(1, device="cuda")
    for k in range(3):
        for t, n in zip(ins, tensors_of(SPECS[4], 10 + k)):
            t.copy_(n)
        want = exact(ins, "l2")
        algo.clip_grad_norm(norm, lst, want / 2)
        assert abs(norm.item() - want) <= REL["l2"] * want
        assert abs(exact(ins, "l2") - want / 2) <= 0.01 * want
    del lst


def test_streams_graphs_and_repeatability(cuda):
    from alpaka3_b200 import algo
    spec = [(100003, BF), (7, SF), (50001, SF)]
    base = tensors_of(spec, 4)
    wants = []
    for _ in range(3):
        ins, norm = [t.clone() for t in base], torch.empty(1, device="cuda")
        algo.clip_grad_norm(norm, ins, 0.5)
        wants.append([norm] + ins)
    assert all(torch.equal(a, b) for w in wants[1:] for a, b in zip(w, wants[0]))
    side = torch.cuda.Stream()
    ins, norm = [t.clone() for t in base], torch.empty(1, device="cuda")
    side.wait_stream(torch.cuda.current_stream())
    algo.clip_grad_norm(norm, ins, 0.5, stream=side)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip([norm] + ins, wants[0]))
    # two graphs over one list, replayed at the same time: each has its own workspace
    src = [t.clone() for t in base]
    graphs, results = [], []
    for _ in range(2):
        outs, norm = [torch.zeros_like(t) for t in base], torch.empty(1, device="cuda")
        lst = algo.TensorList(src, outs)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            algo.clip_grad_norm(norm, lst, 0.5)
        graphs.append(graph)
        results.append([norm] + outs)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for r in results:
        assert all(torch.equal(a, b) for a, b in zip(r, wants[0]))


@pytest.mark.slow
def test_offsets_past_32_bits(cuda):
    n = (1 << 32) + 12345  # elements and bytes past 2^32
    x = torch.zeros(n, dtype=BF, device="cuda")
    x[-3:] = 2.0
    x[5] = 1.0
    from alpaka3_b200 import algo
    norm = torch.empty(1, device="cuda")
    algo.clip_grad_norm(norm, [x], math.sqrt(13.0) / 2)
    assert abs(norm.item() - math.sqrt(13.0)) <= 4 * U * 4
    assert (x[-3:].float() - 1.0).abs().max() <= 2.0**-8 and abs(x[5].item() - 0.5) <= 2.0**-9 and x[6:-3].max() == 0


def test_after_early_started_reductions(cuda):
    """The stream's reductions may overlap; the list's kernels see and leave everything in order."""
    from alpaka3_b200 import algo
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        x = torch.ones(1 << 20, device="cuda")
        sq = torch.empty(1, device="cuda")
        norm = torch.empty(1, device="cuda")
        algo.set_early_start(True, s)
        try:
            for _ in range(5):
                x.fill_(1.0)
                algo.transform_reduce(0.0, sq, "plus", "square", x)
                algo.clip_grad_norm(norm, [x], 512.0)
                algo.transform_reduce(0.0, sq, "plus", "square", x)
                s.synchronize()
                assert abs(norm.item() - 1024.0) <= 1024 * REL["l2"]
                assert abs(sq.item() - 512.0**2) <= 512.0**2 * 20 * U
        finally:
            algo.set_early_start(False, s)


def test_refusals(cuda):
    from alpaka3_b200 import algo, capi
    x, norm = torch.ones(100, device="cuda"), torch.empty(1, device="cuda")
    for bad in (x.long(), x.bool()):
        with pytest.raises(TypeError):
            algo.TensorList([bad])
    for bad in ([x.cpu()], [x[::2]], [x.expand(2, 100)]):
        with pytest.raises(ValueError):
            algo.TensorList(bad)
    for outs in ([x[:50]], [x.half()], [], [x, x], [torch.ones(10, 10, device="cuda")]):
        with pytest.raises(ValueError):
            algo.TensorList([x], outs)
    for args in ((norm, [x], 1.0, "l3"), (torch.empty(2, device="cuda"), [x], 1.0), (norm.cpu(), [x], 1.0),
                 (None, [], 1.0)):
        with pytest.raises(ValueError):
            algo.clip_grad_norm(*args)
    with pytest.raises(TypeError):
        algo.clip_grad_norm(norm.half(), [x], 1.0)
    with pytest.raises(TypeError):
        algo.grad_norm(norm, [x], partial=norm)
    with pytest.raises(ValueError):
        algo.grad_norm(None, [x])
    for limit in (-1.0, math.nan):
        with pytest.raises(capi.A3BError):
            algo.clip_grad_norm(norm, [x], limit)
    store = torch.ones(300, device="cuda")
    part = torch.ones(1, dtype=DF, device="cuda")
    # the same tensor twice, overlapping outputs, an output over another tensor's input, over a part of its own
    for ins, outs in (([x, x], None), ([store[:200], store[100:]], None), ([store[:100], store[100:200]],
                      [store[100:200], store[200:]]), ([store[:200]], [store[1:201]])):
        lst = algo.TensorList(ins, outs)
        with pytest.raises(capi.A3BError, match="overlap"):
            algo.clip_grad_norm(norm, lst, 1.0)
        with pytest.raises(capi.A3BError, match="overlap"):
            algo.clip_grads(norm, lst, part, 1.0)
    algo.grad_norm(norm, [x, x])  # the norm alone may count a tensor twice
    assert abs(norm.item() - math.sqrt(200.0)) <= 15 * 4 * U


def test_tail_of_a_training_step(cuda):
    """Hidden states and an output layer: logits -> log probabilities, entropy, lse -> a loss with an entropy bonus and a
    penalty on lse -> gradient of the logits (in place) -> gradients of the layer and the states -> clipping; against
    autograd in 64 bits on the same bf16 logits. The logits' gradient is off by half a bf16 step (2^-9 relative to 2^-8)
    of each element; the products average it, so 2^-7 of the largest element bounds the rest."""
    from alpaka3_b200 import algo
    n, d, v = 48, 64, 1003
    g = torch.Generator(device="cuda").manual_seed(0)
    h = torch.randn(n, d, generator=g, device="cuda").to(BF)
    w = (torch.randn(v, d, generator=g, device="cuda") * 0.3).to(BF)
    t = torch.randint(0, v, (n,), generator=g, device="cuda")
    t[::5] = -100
    weight, beta, z = torch.randn(n, generator=g, device="cuda"), 0.02, 0.003
    logits = h @ w.t()
    x64 = logits.double().requires_grad_()
    q = torch.log_softmax(x64, -1)
    lse64 = torch.logsumexp(x64, -1)
    picked = torch.where(t >= 0, q.gather(1, t.clamp(min=0)[:, None])[:, 0], torch.zeros(n, dtype=DF, device="cuda"))
    loss = -(weight.double() * picked).sum() - beta * -(q.exp() * q).sum() + z * (lse64**2).sum()
    loss.backward()
    logp, ent, lse = (torch.empty(n, device="cuda") for _ in range(3))
    algo.token_logprobs(logp, logits, t, entropy=ent, lse=lse)
    got = -(weight * logp).sum() - beta * ent.sum() + z * lse.square().sum()
    assert abs(got.item() - loss.item()) <= 1e-5 * (weight.abs().double() * picked.abs()).sum().item()
    algo.token_logprobs_backward(logits, logits, t, lse, entropy=ent, grad_logp=-weight,
                                 grad_entropy=torch.full((n,), -beta, device="cuda"), grad_lse=2 * z * lse)
    big = x64.grad.abs().max().item()
    assert (logits.double() - x64.grad).abs().max().item() <= 2.0**-8 * big
    grads = [logits.t() @ h, logits @ w]
    wants = [x64.grad.t() @ h.double(), x64.grad @ w.double()]
    for a, b in zip(grads, wants):
        assert (a.double() - b).abs().max().item() <= 2.0**-6 * b.abs().max().item()
    total = exact(grads, "l2")
    norm = torch.empty(1, device="cuda")
    algo.clip_grad_norm(norm, grads, total / 10)
    assert abs(norm.item() - total) <= REL["l2"] * total
    assert abs(exact(grads, "l2") - total / 10) <= 2.0**-8 * total / 10


@pytest.mark.parametrize("kind", ["l2", "l1", "max"])
@pytest.mark.parametrize("dtype", [BF, SF])
@pytest.mark.parametrize("n", [4099, 300001])
def test_factors_below_the_normal_numbers(cuda, kind, dtype, n):
    """Elements near fp32's largest number: max_norm / norm is below 2^-126, and has all its bits. In one cluster and in a
    block for every chunk."""
    g = torch.Generator(device="cuda").manual_seed(n)
    for limit in (1.0, 37.0, 1e-3):
        x = (torch.rand(n, generator=g, device="cuda") * 3e38).to(dtype)
        small = torch.randn(77, generator=g, device="cuda").to(dtype)
        outs = [torch.full_like(x, 9.0), torch.full_like(small, 9.0)]
        check([x, small], limit, kind, outs, norm_dtype=DF)
        check([x, small], limit, kind, norm_dtype=DF)


def test_workspace_apart_from_the_results(cuda):
    from alpaka3_b200 import algo, capi
    L, x = capi.lib(), torch.ones(1 << 20, device="cuda")
    lst = algo.TensorList([x])
    need = L.a3b_grad_norm_workspace(lst._handle)
    ws = torch.zeros(need + 64, dtype=torch.uint8, device="cuda")
    out = torch.zeros(1, dtype=DF, device="cuda")
    s, p, stream = ws.data_ptr(), out.data_ptr(), algo.stream_handle()
    for call in (lambda at: L.a3b_grad_norm(stream, lst._handle, 0, s, ws.numel(), p, capi.F32, at),
                 lambda at: L.a3b_grad_norm(stream, lst._handle, 0, s, ws.numel(), at, capi.F64, p),
                 lambda at: L.a3b_clip_grad_norm(stream, lst._handle, 0, 1e9, s, ws.numel(), capi.F64, at)):
        for at in (s, s + need - 8):
            assert call(at) == capi.ERR_INVALID and "workspace" in capi.last_error()
        assert call(s + need) == capi.OK  # behind what is used
    torch.cuda.synchronize()
    assert ws.view(DF)[need // 8].item() == 1024.0 and (x == 1).all()


def test_gradients_of_a_model_of_which_some_are_missing(cuda):
    """A plain sequence of gradients with None among them, in place and to outputs of their own."""
    from alpaka3_b200 import algo
    params = [torch.nn.Parameter(torch.randn(k, device="cuda")) for k in (100, 7, 1, 50000)]
    for p in (params[0], params[3]):
        p.grad = torch.randn_like(p)
    grads = [p.grad for p in params]
    given = [grads[0].clone(), grads[3].clone()]
    want, norm = exact(given, "l2"), torch.empty(1, device="cuda")
    outs = [torch.full((k,), 9.0, device="cuda") for k in (100, 7, 1, 50000)]
    algo.clip_grad_norm(norm, algo.TensorList(grads, outs), want / 2)
    assert abs(norm.item() - want) <= REL["l2"] * want and (outs[1] == 9).all() and (outs[2] == 9).all()
    algo.clip_grad_norm(norm, grads, want / 2)
    assert abs(norm.item() - want) <= REL["l2"] * want and params[1].grad is None
    for o, g, b in ((outs[0], grads[0], given[0]), (outs[3], grads[3], given[1])):
        assert torch.equal(o, g) and ((g - b / 2).abs() <= b.abs() * 8 * U).all()
