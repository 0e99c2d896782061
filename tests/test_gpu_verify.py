"""GPU: verification of drafted tokens (a3b_verify_drafts) against the formula in 64 bits. What comes out are whole numbers, so
everything is tested for equality: the comparisons and the largest quotients are those of 64 bits, and inputs are such that
no two of them lie within 64 bits' own error (random fp32 numbers) or are equal on purpose (ties)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

INF = math.inf
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def log_sums(x, scale):
    return torch.logsumexp(x.double() * scale, -1).float()


def oracle(c, scale=1.0, draft_scale=None):
    """(tokens, accepted), one sequence after the other"""
    logits, drafts = c["logits"], c["drafts"].tolist()
    draft_scale = scale if draft_scale is None else draft_scale
    b, k1, v = logits.shape
    tokens, accepted = torch.full((b, k1), -1, dtype=torch.int64), torch.zeros(b, dtype=torch.int64)
    for i in range(b):
        n, rate, top = 0, None, c.get("top")
        if top is not None and 0 <= top[i, 0] < v:
            while n < k1 - 1 and 0 <= drafts[i][n] < v and drafts[i][n] == top[i, n]:
                tokens[i, n] = drafts[i][n]
                n += 1
            tokens[i, n] = top[i, n] if 0 <= top[i, n] < v else -1
            accepted[i] = n
            continue
        while True:
            p = torch.exp(logits[i, n].double() * scale - c["lse"][i, n].double())
            if n == k1 - 1 or not 0 <= drafts[i][n] < v:
                rate = p
                break
            if c.get("draft_logits") is not None:
                q = torch.exp(c["draft_logits"][i, n].double() * draft_scale - c["draft_lse"][i, n].double())
            else:
                q = torch.zeros_like(p)
                q[drafts[i][n]] = 1
            if c["uniform"][i, n].double() * q[drafts[i][n]] < p[drafts[i][n]]:
                tokens[i, n] = drafts[i][n]
                n += 1
                continue
            rate = p - q
            if not (rate > 0).any():
                rate = p
            break
        accepted[i] = n
        score = torch.where(rate > 0, rate / c["noise"][i].double(), torch.full_like(rate, -1.0))
        if score.max() >= 0 and (rate > 0).any():
            tokens[i, n] = int((score == score.max()).nonzero()[0])
    return tokens, accepted


def make(b, k, v, dtype, seed=0, model=True, scale=1.0, draft_scale=None, spread=2.5, index=torch.int64):
    g = torch.Generator(device="cuda").manual_seed(seed + 31 * v + 7 * b + k)
    x = torch.randn(b, k + 1, v, generator=g, device="cuda") * spread
    y = x[:, :k] + torch.randn(b, k, v, generator=g, device="cuda")
    c = {"logits": x.to(dtype), "noise": torch.empty(b, v, device="cuda").exponential_(generator=g).clamp_(min=1e-30),
         "uniform": torch.rand(b, k, generator=g, device="cuda")}
    y = y.to(dtype)
    race = torch.empty(b, k, v, device="cuda").exponential_(generator=g)
    ds = scale if draft_scale is None else draft_scale
    c["drafts"] = (torch.softmax(y.float() * ds, -1) / race).argmax(-1).to(index)
    c["lse"] = log_sums(c["logits"], scale)
    if model:
        c |= {"draft_logits": y, "draft_lse": log_sums(y, ds)}
    return c


def verify(c, scale=1.0, draft_scale=None, stream=None, out=None):
    from alpaka3_b200 import algo
    b, k = c["drafts"].shape
    tokens, accepted = out or (torch.full((b, k + 1), 55, dtype=c["drafts"].dtype, device="cuda"),
                               torch.full((b,), 55, dtype=c["drafts"].dtype, device="cuda"))
    top = c.get("top")
    got = algo.verify_drafts(tokens, accepted, c["drafts"], c.get("logits"), c.get("lse"), c.get("uniform"), c.get("noise"),
                             draft_logits=c.get("draft_logits"), draft_lse=c.get("draft_lse"), scale=scale,
                             draft_scale=draft_scale, top_index=top, stream=stream)
    assert got is tokens
    return tokens, accepted


def check(c, scale=1.0, draft_scale=None):
    tokens, accepted = verify(c, scale, draft_scale)
    want, count = oracle(c, scale, draft_scale)
    assert torch.equal(accepted.cpu().long(), count)
    assert torch.equal(tokens.cpu().long(), want)
    return tokens, accepted


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("v", [1, 2, 7, 8, 33, 64, 257, 1000, 2048, 4099, 16384, 50257, 131072])
def test_against_64_bits(cuda, dtype, v):
    for b, k, model in ((1, 4, True), (3, 0, False), (5, 3, False), (9, 5, True)):
        check(make(b, k, v, dtype, 1, model))
        check(make(b, k, v, dtype, 2, model, 0.8, 1.3 if model else None), 0.8, 1.3 if model else None)


def test_many_sequences(cuda):
    for b, k, v, dtype in ((700, 2, 500, torch.bfloat16), (1500, 1, 33, torch.float32), (300, 4, 4096, torch.float16),
                           (2000, 0, 257, torch.float32)):
        _, accepted = check(make(b, k, v, dtype, 3))
        assert k == 0 or (0 < accepted.double().mean() < k)


@pytest.mark.parametrize("index", [torch.int64, torch.int32])
@pytest.mark.parametrize("k", [1, 31, 32, 33, 64, 70])
def test_long_drafts(cuda, k, index):
    """Drafts that all stand, up to more than a warp looks at; and ones that end at any place."""
    c = make(6, k, 50, torch.float32, 4, index=index)
    c["uniform"].zero_()
    _, accepted = check(c)
    assert (accepted == k).all()
    for i in range(6):
        c["drafts"][i, min(k - 1, i * 13):] = (-1, 50, -100, 2**31 - 1, -2**31, 51)[i]
    _, accepted = check(c)
    assert accepted.tolist() == [min(k - 1, i * 13) for i in range(6)]
    c["uniform"].fill_(1.0)  # only what the draft held less likely than the target stands
    check(c)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("v", [5, 1000, 40000])
def test_masks(cuda, dtype, v):
    g = torch.Generator(device="cuda").manual_seed(v)
    for low in (-INF, torch.finfo(dtype).min, -1e4):
        c = make(8, 3, v, dtype, 5)
        out = torch.rand(8, 1, v, generator=g, device="cuda") < 0.4
        out[..., v // 2] = False
        for name, rows in (("logits", 4), ("draft_logits", 3)):
            c[name].masked_fill_(out.expand(8, rows, v), low)
        c["logits"][1, :] = low  # a sequence with nothing left, or with equal tokens
        c["logits"][2, 1] = low
        c["draft_logits"][3, 0] = low
        c["lse"], c["draft_lse"] = log_sums(c["logits"], 1.0), log_sums(c["draft_logits"], 1.0)
        if low != -INF and dtype != torch.float16 and low < -1e30:
            c["lse"][1], c["lse"][2, 1], c["draft_lse"][3, 0] = low, low, low  # as fp32 holds low + ln v
        tokens, accepted = check(c)
        if low == -INF:
            assert accepted[1] == 0 and (tokens[1] == -1).all()
        check({**c, "draft_logits": None, "draft_lse": None})


def test_same_distributions(cuda):
    """The draft's distribution is the target's: everything stands for uniform below 1; refused at 1, no rate is left and the
    token is drawn from the target."""
    for v in (3, 300, 50257):
        c = make(20, 4, v, torch.bfloat16, 6)
        c["draft_logits"], c["draft_lse"] = c["logits"][:, :4], c["lse"][:, :4].contiguous()
        c["uniform"].clamp_(max=1 - 2.0**-24)
        _, accepted = check(c)
        assert (accepted == 4).all()
        c["uniform"][:, 2] = 1.0
        tokens, accepted = check(c)
        assert (accepted == 2).all() and (tokens[:, 2] >= 0).all()


def test_nearly_the_same(cuda):
    """Differences of nearly equal probabilities, where 32 bits alone would not tell the largest quotient."""
    for v in (300, 50257):
        c = make(30, 2, v, torch.float32, 7)
        g = torch.Generator(device="cuda").manual_seed(v)
        c["draft_logits"] = c["logits"][:, :2] + 1e-6 * torch.randn(30, 2, v, generator=g, device="cuda")
        c["draft_lse"] = log_sums(c["draft_logits"], 1.0)
        c["uniform"].fill_(1.0)
        check(c)


def test_ties(cuda):
    """Equal rates and equal noise: the lowest token, wherever the equal ones lie."""
    for v in (2, 9, 1000, 20000, 100003):
        c = make(6, 1, v, torch.float32, 8, model=False)
        c["logits"].zero_()
        c["noise"].fill_(2.0)
        c["drafts"].fill_(0)
        c["lse"] = log_sums(c["logits"], 1.0)
        c["uniform"].fill_(1.0)
        tokens, _ = check(c)
        assert (tokens[:, 0] == 1).all()
        c["drafts"].fill_(-1)
        for i, at in enumerate((0, v // 3, v // 2, v - 2, v - 1, 0)):
            c["noise"][i, at] = c["noise"][i, v - 1] = 0.5
        check(c)


@pytest.mark.parametrize("size", [50.0, 3e3, 1e6, 3e7, 1e15, 3e37])
def test_far_logits(cuda, size):
    """Logits around +-size, whose rounded lse is off by more than a probability: the formula for these very inputs holds."""
    for v in (40, 3000):
        for sign in (1, -1):
            c = make(6, 2, v, torch.float32, 9)
            for name in ("logits", "draft_logits"):
                c[name].add_(sign * size)
            c["lse"], c["draft_lse"] = log_sums(c["logits"], 1.0), log_sums(c["draft_logits"], 1.0)
            check(c)
            check({**c, "draft_logits": None, "draft_lse": None})


def test_infinities_and_nan(cuda):
    for v in (20, 5000):
        c = make(7, 2, v, torch.float32, 10)
        c["uniform"].zero_()
        c["logits"][0, 0, 3] = math.nan
        c["logits"][1, 1, 4] = INF
        c["logits"][2, 2, v - 1] = math.nan
        c["draft_logits"][3, 0, 5] = math.nan
        c["draft_logits"][4, 1, v - 1] = INF
        c["lse"], c["draft_lse"] = log_sums(c["logits"], 1.0), log_sums(c["draft_logits"], 1.0)
        c["lse"][1, 1], c["draft_lse"][4, 1] = INF, INF  # as token_logprobs gives
        tokens, accepted = verify(c)
        tokens, accepted = tokens.cpu(), accepted.cpu()
        assert accepted[0] == 0 and tokens[0].tolist() == [-1, -1, -1]
        assert accepted[1] == 1 and tokens[1, 1:].tolist() == [-1, -1]
        assert accepted[2] == 2 and tokens[2, 2] == -1
        want, count = oracle({**c, "draft_logits": c["draft_logits"].nan_to_num(nan=0.0)})
        assert accepted[3] == 0  # refused, and drawn from the target alone
        p = torch.exp(c["logits"][3, 0].double() - c["lse"][3, 0].double())
        assert tokens[3, 0] == (p / c["noise"][3].double()).argmax()
        assert torch.equal(tokens[5:], want[5:]) and torch.equal(accepted[5:], count[5:])
        # noise at zero wins where there is a rate, and only there
        c = make(3, 0, v, torch.float32, 11, model=False)
        c["logits"][:, :, 7] = -INF
        c["noise"][:, 7] = 0
        c["noise"][1, 11] = c["noise"][1, 9] = 0
        c["noise"][2, 13] = 1e-42
        c["lse"] = log_sums(c["logits"], 1.0)
        tokens, _ = check(c)
        assert tokens[1, 0] == 9


def test_layouts(cuda):
    """Logits, draft logits and noise as parts of larger arrays, at every alignment."""
    for dtype in DTYPES:
        for v, gap in ((64, 8), (64, 3), (1001, 6), (2048, 2048)):
            c = make(5, 3, v, dtype, 12)
            want = verify(c)
            room = torch.full((5, 6, v + gap), math.nan, dtype=dtype, device="cuda")
            far = torch.full((7, 5, v + gap), math.nan, dtype=dtype, device="cuda")
            clock = torch.full((5, v + gap), math.nan, device="cuda")
            room[:, 1:5, gap:], far[1:6, :3, :v], clock[:, gap:] = c["logits"], c["draft_logits"], c["noise"]
            got = verify({**c, "logits": room[:, 1:5, gap:], "draft_logits": far[1:6, :3, :v], "noise": clock[:, gap:]})
            assert all(torch.equal(a, b) for a, b in zip(got, want))
            turned = c["logits"].transpose(0, 1).contiguous().transpose(0, 1)
            got = verify({**c, "logits": turned})
            assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("index", [torch.int64, torch.int32])
def test_greedy(cuda, index):
    from alpaka3_b200 import algo
    b, k, v = 9, 40, 700
    c = make(b, k, v, torch.float32, 13, index=index)
    logp, top = torch.empty(b, k + 1, 1, device="cuda"), torch.empty(b, k + 1, 1, dtype=index, device="cuda")
    algo.token_logprobs(None, c["logits"], None, top_logp=logp, top_index=top)
    top = top[..., 0].contiguous()
    drafts = top[:, :k].clone()
    for i in range(b):
        if i * 5 < k:
            drafts[i, i * 5] = (int(drafts[i, i * 5]) + 1) % v if i % 2 else -1
    greedy = {"drafts": drafts, "top": top}
    tokens, accepted = verify(greedy)
    want, count = oracle({**c, **greedy})
    assert torch.equal(tokens.cpu().long(), want) and torch.equal(accepted.cpu().long(), count)
    assert accepted.tolist() == [min(i * 5, k) for i in range(b)]
    # some sequences greedy, the others drawn
    mixed = top.clone()
    mixed[::2, 0] = -1
    check({**c, "top": mixed})
    one = {"drafts": torch.empty(3, 0, dtype=index, device="cuda"), "top": torch.tensor([[4], [-1], [2]], dtype=index, device="cuda")}
    tokens, accepted = verify(one)
    assert tokens.flatten().tolist() == [4, -1, 2] and accepted.tolist() == [0, 0, 0]


def test_distribution(cuda):
    """Whatever the draft proposes, the first token is distributed as the target's: counts of 60000 draws within six standard
    deviations, for a draft model and for looked up drafts; and so is the second after a given first."""
    b, v = 60000, 6
    g = torch.Generator(device="cuda").manual_seed(14)
    x = torch.tensor([1.0, 0.3, -0.5, 2.0, -3.0, 0.0], device="cuda")
    y = torch.tensor([0.2, 1.5, -2.0, 1.0, 0.0, -INF], device="cuda")
    p = torch.softmax(x.double(), -1)
    for model in (True, False):
        race = torch.empty(b, 1, v, device="cuda").exponential_(generator=g)
        drafts = (torch.softmax(y, -1) / race).argmax(-1) if model else torch.full((b, 1), 3, device="cuda")
        c = {"logits": x.expand(b, 2, v), "lse": log_sums(x, 1.0).expand(b, 2).contiguous(), "drafts": drafts,
             "uniform": torch.rand(b, 1, generator=g, device="cuda"),
             "noise": torch.empty(b, v, device="cuda").exponential_(generator=g).clamp_(min=1e-30)}
        if model:
            c |= {"draft_logits": y.expand(b, 1, v), "draft_lse": log_sums(y, 1.0).expand(b, 1).contiguous()}
        tokens, accepted = verify(c)
        for column, size in ((tokens[:, 0], b), (tokens[accepted == 1, 1], int(accepted.sum()))):
            counts = torch.bincount(column, minlength=v).double()
            assert counts.sum() == size
            assert ((counts - size * p).abs() <= 6 * (size * p * (1 - p)).sqrt()).all()


def test_empty_batch(cuda):
    c = {k: (t[:0] if t is not None else None) for k, t in make(2, 3, 10, torch.float32).items()}
    tokens, accepted = verify(c)
    assert tokens.numel() == 0 and accepted.numel() == 0


def test_streams_and_graphs(cuda):
    c = make(40, 4, 20000, torch.bfloat16, 15)
    want = verify(c)
    side = torch.cuda.Stream()
    out = tuple(torch.zeros_like(t) for t in want)
    side.wait_stream(torch.cuda.current_stream())
    verify(c, stream=side, out=out)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, want))
    graphs, outs = [], []
    for _ in range(2):
        o = tuple(torch.zeros_like(t) for t in want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            verify(c, out=o)
        graphs.append(graph)
        outs.append(o)
    c["uniform"].copy_(c["uniform"].flip(0))
    c["noise"].copy_(c["noise"].flip(0))
    want = verify(c)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for o in outs for a, b in zip(o, want))


@pytest.mark.parametrize("v", [3, 20, 5000, 40000, 131072])
def test_noise_that_takes_no_part(cuda, v):
    """Tokens whose noise is negative or NaN are never drawn and hide no other, whatever their rate: behind a refused draft,
    behind drafts that all stand, and without a draft; in one block and in a cluster of blocks."""
    for b in (1, 5):
        for model in (True, False):
            g = torch.Generator(device="cuda").manual_seed(v + b)
            c = make(b, 2, v, torch.float32, 16, model=model)
            flip = torch.rand(b, v, generator=g, device="cuda") < 0.3
            flip[0, c["drafts"][0, 0]] = True  # what the draft took is not drawn for its sign
            c["noise"] = torch.where(flip, -c["noise"], c["noise"])
            nan = flip & (torch.rand(b, v, generator=g, device="cuda") < 0.2)
            for uniform in (1.0, 0.0, None):
                if uniform is not None:
                    c["uniform"].fill_(uniform)
                check(c)
                got, want = verify({**c, "noise": c["noise"].masked_fill(nan, math.nan)}), oracle(c)
                assert all(torch.equal(a.cpu().long(), w) for a, w in zip(got, want))
            none = {**c, "drafts": torch.full_like(c["drafts"], -1)}
            check(none)
            tokens, _ = check({**none, "noise": -c["noise"].abs()})
            assert (tokens == -1).all()


def test_rates_without_a_clock(cuda):
    """p = (0.2, 0.3, 0.5), and token 2 was looked up and refused."""
    p = torch.tensor([0.2, 0.3, 0.5], device="cuda")
    c = {"logits": p.log().expand(1, 2, 3).contiguous(), "lse": torch.zeros(1, 2, device="cuda"),
         "drafts": torch.tensor([[2]], device="cuda"), "uniform": torch.ones(1, 1, device="cuda")}
    for noise, token in (((1, 1, -0.1), 1), ((1, -1, -0.1), 0), ((-1, -1, 1), -1), ((-1, 1, 1), 1), ((math.nan, 1, -2), 1)):
        tokens, accepted = verify({**c, "noise": torch.tensor([noise], device="cuda", dtype=torch.float32)})
        assert tokens.tolist() == [[token, -1]] and accepted.item() == 0, noise


@pytest.mark.parametrize("v", [1000, 5000, 50257, 131072])
@pytest.mark.parametrize("noise", [3e38, 1e35, 1e-30])
def test_quotients_far_from_one(cuda, v, noise):
    """Noise of any positive size: quotients below fp32's normal numbers, which hold few digits, and large ones."""
    c = make(20, 1, v, torch.float32, 17, model=False, spread=0.02)
    c["noise"] = (torch.rand(20, v, device="cuda", generator=torch.Generator(device="cuda").manual_seed(v)) * 1e-3 + 1) * noise
    c["uniform"].fill_(1.0)
    check(c)
    c["drafts"].fill_(-1)
    check(c)


@pytest.mark.parametrize("dtype", DTYPES)
def test_products_are_rounded(cuda, dtype):
    """scale * z is a 64-bit number before lse is taken from it. Token 0: its product rounds to lse itself, so p = 1 and the draft
    leaves nothing of it; the exact product is up to 4e-12 more. So token 2 is drawn, with a rate of e^-486, e^-179 or e^-85."""
    for scale, z in ((1.9, -40960.0), (0.7, -40960.0), (1.0 / 3, -24576.0)):
        assert scale * z == round(scale * z)
        c = {"logits": torch.tensor([z, -INF, z - 256], device="cuda").expand(1, 2, 3).to(dtype).contiguous(),
             "lse": torch.full((1, 2), scale * z, device="cuda"), "drafts": torch.tensor([[1]], device="cuda"),
             "uniform": torch.full((1, 1), 0.5, device="cuda"), "noise": torch.ones(1, 3, device="cuda"),
             "draft_logits": torch.tensor([[[0.0, -1.0, -INF]]], device="cuda").to(dtype),
             "draft_lse": torch.zeros(1, 1, device="cuda")}
        tokens, _ = check(c, scale, 1.0)
        assert tokens.tolist() == [[2, -1]]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scale", [1.9, 0.7, 2.0**-6, 2.0**8])
def test_masks_and_scales(cuda, dtype, scale):
    """Rows masked by finite values, some wholly, at a scale: probabilities are those of the rounded product."""
    g = torch.Generator(device="cuda").manual_seed(18)
    for v in (2, 7, 27, 3000):
        for low in (torch.finfo(dtype).min, -1e4):
            for share in (0.5, 0.95):
                c = make(40, 2, v, dtype, 18, True, scale, 0.9, 20.0)
                for name, s, lse in (("logits", scale, "lse"), ("draft_logits", 0.9, "draft_lse")):
                    c[name].masked_fill_(torch.rand(c[name].shape, generator=g, device="cuda") < share, low)
                    c[lse] = log_sums(c[name], s)
                check(c, scale, 0.9)
                check({**c, "draft_logits": None, "draft_lse": None}, scale, 0.9)
