"""GPU: the operators around a model's layers as a step uses them, one after the other: a training step with tied embedding and
head up to the clipped gradients, against 64-bit automatic differentiation, and a speculative decoding step."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

VOCAB, WIDTH, SCALE, EPS = 501, 96, math.sqrt(96), 1e-5


def norm64(h, w):
    return h / torch.sqrt(h.square().mean(-1, keepdim=True) + EPS) * w


def loss64(p, tokens, targets):
    table, w1, w2, a = p
    h = table[tokens] * SCALE
    h = h + norm64(h, w1) @ a
    q = torch.log_softmax(norm64(h, w2) @ table.T, -1)
    return -q.gather(-1, targets[..., None]).sum()


def test_training_step(cuda):
    """In 32 bits every gradient is within 2e-4 of its norm: products of at most 501 terms (their error 501 x 2^-24 = 3e-5 of
    the terms' magnitudes) three after one another, and the operators' own errors far below that."""
    from alpaka3_b200 import algo
    g = torch.Generator(device="cuda").manual_seed(1)
    rand = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    table, w1, w2, a = rand(VOCAB, WIDTH) * 0.3, 1 + 0.1 * rand(WIDTH), 1 + 0.1 * rand(WIDTH), rand(WIDTH, WIDTH) * 0.1
    tokens = torch.randint(0, VOCAB, (4, 33), generator=g, device="cuda")
    tokens[:, ::3] = 7  # a frequent one
    targets = torch.randint(0, VOCAB, (4, 33), generator=g, device="cuda")
    p = [t.double().requires_grad_() for t in (table, w1, w2, a)]
    loss64(p, tokens, targets).backward()
    want = [t.grad for t in p]

    shape = (4, 33, WIDTH)
    new = lambda *s: torch.empty(s, device="cuda")  # noqa: E731
    h0, y, z, total, f = (new(*shape) for _ in range(5))
    r1, r2, logp, lse = (new(4, 33) for _ in range(4))
    algo.embedding(h0, table, tokens, scale=SCALE)
    algo.rms_norm(y, h0, w1, rstd=r1, eps=EPS)
    torch.matmul(y, a, out=z)
    algo.rms_norm(f, z, w2, residual=h0, total=total, rstd=r2, eps=EPS)
    logits = f @ table.T
    algo.token_logprobs(logp, logits, targets, lse=lse)
    assert abs(-logp.double().sum() - loss64([t.detach() for t in p], tokens, targets)) <= 1e-4 * 4 * 33
    algo.token_logprobs_backward(logits, logits, targets, lse, grad_logp=torch.full((4, 33), -1.0, device="cuda"))
    flat = lambda t: t.reshape(-1, t.shape[-1])  # noqa: E731
    gtable = flat(logits).T @ flat(f)
    gf, gt, gh0, gw1, gw2 = logits @ table, new(*shape), new(*shape), new(WIDTH), new(WIDTH)
    algo.rms_norm_backward(gt, gf, total, w2, r2, grad_weight=gw2)
    ga = flat(y).T @ flat(gt)
    algo.rms_norm_backward(gh0, gt @ a.T, h0, w1, r1, grad_weight=gw1, grad_total=gt)
    algo.embedding_backward(gtable, gh0, tokens, scale=SCALE, add=gtable)
    got = [gtable, gw1, gw2, ga]
    for x, y in zip(got, want):
        assert (x.double() - y).norm() <= 2e-4 * y.norm()
    norm = new(1)
    algo.clip_grad_norm(norm, got, 1.0)
    size = math.sqrt(sum(t.square().sum().item() for t in want))
    assert abs(norm.item() - size) <= 2e-4 * size and size > 1
    for x, y in zip(got, want):
        assert (x.double() - y / size).norm() <= 5e-4 * y.norm() / size


def test_captured_training_step(cuda):
    """The operators of a step captured into one graph give the same bits as one after the other, on new tokens too."""
    from alpaka3_b200 import algo
    g = torch.Generator(device="cuda").manual_seed(2)
    table, w = torch.randn(VOCAB, WIDTH, generator=g, device="cuda"), torch.randn(WIDTH, generator=g, device="cuda")
    tokens = torch.randint(0, VOCAB, (300,), generator=g, device="cuda")

    def step(o):
        algo.embedding(o["h"], table, tokens, scale=SCALE)
        algo.rms_norm(o["y"], o["h"], w, rstd=o["r"])
        algo.rms_norm_backward(o["gh"], o["y"], o["h"], w, o["r"], grad_weight=o["gw"])
        algo.embedding_backward(o["gt"], o["gh"], tokens, scale=SCALE)

    def outputs():
        return {"h": torch.empty(300, WIDTH, device="cuda"), "y": torch.empty(300, WIDTH, device="cuda"),
                "r": torch.empty(300, device="cuda"), "gh": torch.empty(300, WIDTH, device="cuda"),
                "gw": torch.empty(WIDTH, device="cuda"), "gt": torch.empty(VOCAB, WIDTH, device="cuda")}

    eager, captured = outputs(), outputs()
    step(eager)  # loads and sets up what the first call sets up
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(captured)
    for seed in range(3):
        tokens.copy_(torch.randint(0, VOCAB, (300,), generator=g, device="cuda"))
        step(eager)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(eager[k], captured[k]) for k in eager)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_speculative_step(cuda, dtype):
    """Drafts to rows, rows to 8 bits, those to logits, log-sum-exp and then tokens; the draft model is a smaller head."""
    from alpaka3_b200 import algo
    b, k = 9, 4
    g = torch.Generator(device="cuda").manual_seed(3)
    rand = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    table, w = (rand(VOCAB, WIDTH) * 0.5).to(dtype), (1 + 0.1 * rand(WIDTH)).to(dtype)
    head, small = rand(WIDTH, VOCAB).to(dtype), None
    small = (head.float() + 0.3 * rand(WIDTH, VOCAB)).to(dtype)
    last = torch.randint(0, VOCAB, (b, 1), generator=g, device="cuda")

    def rows(tokens):
        h = torch.empty(*tokens.shape, WIDTH, dtype=dtype, device="cuda")
        algo.embedding(h, table, tokens)
        q = torch.empty(h.shape, dtype=torch.float8_e4m3fn, device="cuda")
        s = torch.empty(*tokens.shape, WIDTH // 32, device="cuda")
        algo.rms_norm(q, h, w, scales=s, group=32)
        back = (q.float().unflatten(-1, (-1, 32)) * s[..., None]).flatten(-2)
        exact = norm64(h.double(), w.double())
        assert (back.double() - exact).abs().max() <= 2.0**-4 * exact.abs().max()
        return back.to(dtype)

    # the drafts, one after the other; a bigram model: a position's row is that of the token before
    drafts, draft_logits = [], []
    t = last
    for _ in range(k):
        z = rows(t) @ small
        t = (torch.softmax(z.float(), -1) / torch.empty(z.shape, device="cuda").exponential_(generator=g)).argmax(-1)
        drafts.append(t)
        draft_logits.append(z)
    drafts, draft_logits = torch.cat(drafts, 1), torch.cat(draft_logits, 1)
    logits = rows(torch.cat([last, drafts], 1)) @ head
    lse, draft_lse, logp = torch.empty(b, k + 1, device="cuda"), torch.empty(b, k, device="cuda"), torch.empty(b, k, device="cuda")
    algo.token_logprobs(None, logits, None, lse=lse)
    algo.token_logprobs(logp, draft_logits, drafts, lse=draft_lse)
    uniform, noise = torch.rand(b, k, generator=g, device="cuda"), torch.empty(b, VOCAB, device="cuda").exponential_(generator=g)
    tokens, accepted = torch.empty(b, k + 1, dtype=torch.int64, device="cuda"), torch.empty(b, dtype=torch.int64, device="cuda")
    algo.verify_drafts(tokens, accepted, drafts, logits, lse, uniform, noise, draft_logits=draft_logits, draft_lse=draft_lse)
    p = torch.exp(logits.double() - lse.double()[..., None])
    q = torch.exp(draft_logits.double() - draft_lse.double()[..., None])
    seen = 0
    for i in range(b):
        n = int(accepted[i])
        for j in range(min(n + 1, k)):
            d = drafts[i, j]
            assert (uniform[i, j].double() * q[i, j, d] < p[i, j, d]) == (j < n)
        assert torch.equal(tokens[i, :n], drafts[i, :n]) and (tokens[i, n + 1:] == -1).all()
        rate = p[i, n] if n == k else (p[i, n] - q[i, n]).clamp(min=0)
        assert tokens[i, n] == (rate / noise[i].double()).argmax()
        seen += n
    assert 0 < seen < b * k
