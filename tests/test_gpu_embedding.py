"""GPU: rows of a table by tokens and the table's gradient (a3b_embedding, a3b_embedding_backward).

The lookup is one fp32 product rounded once: the same bits as in elementary operations. Gradients are tested on whole numbers,
whose sums below 2^24 are the same in any order, for equality; and on random ones against 64 bits: with u = 2^-24, a token at m
places is summed in chunks of at most 256, whose sums are added in eight parts, so at most D = 256 + m / 32 + 16 additions
one after the other: (D + 3) u of the sum of magnitudes, and half a step of the type."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0**-24
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
PAIRS = [(F32, F32), (F16, F16), (BF16, BF16), (F32, F16), (F32, BF16), (F16, F32), (BF16, F32)]


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def table(vocab, n, dtype, seed=0):
    return torch.randn(vocab, n, generator=gen(seed + n), device="cuda").to(dtype)


def pick(shape, vocab, seed=0, dtype=torch.int64, skew=False, outside=True):
    t = torch.randint(0, vocab, shape, generator=gen(seed), device="cuda")
    if skew:  # half of the places one token, and small ones more often
        t = torch.minimum(t, torch.randint(0, vocab, shape, generator=gen(seed + 1), device="cuda"))
        t[torch.rand(shape, generator=gen(seed + 2), device="cuda") < 0.5] = vocab // 2
    if outside:
        t[torch.rand(shape, generator=gen(seed + 3), device="cuda") < 0.1] = -100
        t[torch.rand(shape, generator=gen(seed + 4), device="cuda") < 0.03] = vocab
    return t.to(dtype)


def lookup(w, t, scale, dtype, first=0):
    t = t.long() - first
    known = (t >= 0) & (t < w.shape[0])
    rows = w.float()[torch.where(known, t, torch.zeros_like(t))] * torch.tensor(scale, dtype=F32, device="cuda")
    return torch.where(known[..., None], rows, torch.zeros_like(rows)).to(dtype)


@pytest.mark.parametrize("pair", PAIRS)
@pytest.mark.parametrize("n", [1, 3, 8, 16, 33, 100, 128, 1000, 1001, 1024, 2048, 5000])
def test_lookup(cuda, pair, n):
    from alpaka3_b200 import algo
    source, target = pair
    w = table(301, n, source)
    for shape, index, scale in (((1,), torch.int64, 1.0), ((7, 9), torch.int32, math.sqrt(n)), ((3000,), torch.int64, -0.3)):
        t = pick(shape, 301, n, index)
        out = torch.full((*shape, n), 7.0, dtype=target, device="cuda")
        assert algo.embedding(out, w, t, scale=scale) is out
        assert torch.equal(out, lookup(w, t, scale, target))


def test_lookup_layouts(cuda):
    from alpaka3_b200 import algo
    for source, target in PAIRS:
        for n, gap in ((64, 16), (64, 3), (37, 5)):
            w = table(50, n + gap, source)[:, gap:]
            t = pick((6, 5), 50, 1)
            room = torch.full((6, 7, n + 2 * gap), 5.0, dtype=target, device="cuda")
            out = room[:, 1:6, gap:gap + n]
            algo.embedding(out, w, t, scale=2.0)
            assert torch.equal(out, lookup(w, t, 2.0, target))
            out.fill_(5.0)
            assert (room == 5.0).all()
    w, t = table(50, 64, F32), pick((6, 5), 50, 1)
    back = torch.empty(5, 6, 64, device="cuda").transpose(0, 1)
    algo.embedding(back, w, t)
    assert torch.equal(back, lookup(w, t, 1.0, F32))


def test_parts_of_a_table(cuda):
    """A table cut in two: each part gives zeros for the other's tokens, so the parts' outputs add up; likewise the gradients
    are the parts of the whole one. Tokens at both ends of 64 bits are outside."""
    from alpaka3_b200 import algo
    w, t = table(101, 48, F32), pick((40, 6), 101, 3)
    t.view(-1)[0], t.view(-1)[1] = 2**63 - 1, -2**63
    whole = algo.embedding(torch.empty(40, 6, 48, device="cuda"), w, t)
    assert (whole.view(-1, 48)[:2] == 0).all()
    g = torch.randint(-4, 5, (40, 6, 48), generator=gen(4), device="cuda").float()
    gw = algo.embedding_backward(torch.empty_like(w), g, t)
    total = torch.zeros_like(whole)
    for lo, hi in ((0, 37), (37, 101)):
        total += algo.embedding(torch.empty_like(whole), w[lo:hi], t, first=lo)
        part = algo.embedding_backward(torch.empty(hi - lo, 48, device="cuda"), g, t, first=lo)
        assert torch.equal(part, gw[lo:hi])
    assert torch.equal(total, whole)
    # far offsets: tokens near the ends of 64 bits
    for base in (-2**63, 2**63 - 1 - 100, 2**40):
        far = torch.tensor([base, base + 1, base + 50, 0, -1], device="cuda")
        out = algo.embedding(torch.empty(5, 48, device="cuda"), w, far, first=base)
        assert torch.equal(out, torch.cat([w[[0, 1, 50]], torch.zeros(2, 48, device="cuda")]))


def test_long_table(cuda):
    """Rows behind 2^32 elements."""
    from alpaka3_b200 import algo
    n, vocab = 4096, (1 << 20) + 40
    w = torch.empty(vocab, n, dtype=BF16, device="cuda")
    ids = torch.tensor([0, 1, (1 << 19) + 3, 1 << 20, vocab - 1], device="cuda")
    w[ids] = table(5, n, BF16)
    out = algo.embedding(torch.empty(5, n, dtype=BF16, device="cuda"), w, ids)
    assert torch.equal(out, table(5, n, BF16))
    w.fill_(3.0)
    algo.embedding_backward(w, out, ids, add=w)
    assert torch.equal(w[ids], (out.float() + 3).to(BF16))
    assert (w[ids[3] - 1] == 3).all() and (w[2] == 3).all()
    algo.embedding_backward(w, out, ids)
    assert torch.equal(w[ids], out) and (w[ids[3] - 1] == 0).all() and w[vocab - 20:vocab - 1].abs().max() == 0


# ------------------------------------------------------------------------------------------------------ gradient
def summed(g, t, vocab, scale, add, first=0):
    """in 64 bits, with the sum of magnitudes and the number of places"""
    t = t.long().flatten() - first
    known = (t >= 0) & (t < vocab)
    t, rows = t[known], g.double().reshape(-1, g.shape[-1])[known]
    out, size = (torch.zeros(vocab, g.shape[-1], dtype=torch.float64, device="cuda") for _ in range(2))
    out.index_add_(0, t, rows)
    size.index_add_(0, t, rows.abs())
    scale = torch.tensor(scale, dtype=F32).double().item()
    out, size = out * scale, size * abs(scale)
    if add is not None:
        out, size = out + add.double(), size + add.double().abs()
    return out, size, torch.bincount(t, minlength=vocab)


def whole_numbers(shape, dtype, seed):
    return torch.randint(-3, 4, shape, generator=gen(seed), device="cuda").to(dtype)


@pytest.mark.parametrize("pair", PAIRS)
@pytest.mark.parametrize("n", [1, 8, 33, 64, 128, 200, 1024, 1001])
def test_gradient_exactly(cuda, pair, n):
    """pair: (type of grad_out, type of the table)"""
    from alpaka3_b200 import algo
    source, target = pair
    for count, vocab, skew in ((1, 5, False), (2, 1, False), (31, 40, False), (500, 37, True), (1000, 3001, True),
                               (8192, 700, True), (8193, 700, True), (20000, 1031, True)):
        if n >= 1000 and count > 8193:
            continue
        t = pick((count,), vocab, count, skew=skew, outside=count > 2)
        g = whole_numbers((count, n), source, n)
        want = summed(g, t, vocab, 2.0, None)[0]
        gw = torch.full((vocab, n), 7.0, dtype=target, device="cuda")
        assert algo.embedding_backward(gw, g, t, scale=2.0) is gw
        assert torch.equal(gw, want.to(target))
        add = whole_numbers((vocab, n), target, 3)
        want = want + add.double()
        algo.embedding_backward(gw, g, t, scale=2.0, add=add)
        assert torch.equal(gw, want.to(target))
        algo.embedding_backward(add, g, t, scale=2.0, add=add)  # in place
        assert torch.equal(add, want.to(target))


@pytest.mark.parametrize("count,vocab,n", [(300, 1000, 256), (5000, 50, 64), (40000, 3, 96), (100000, 131072, 32),
                                           (131072, 70000, 40), (60000, 600000, 16)])
def test_gradient_against_64_bits(cuda, count, vocab, n):
    from alpaka3_b200 import algo
    for source, target in ((F32, F32), (BF16, BF16), (F16, F32)):
        t = pick((count // 4, 4), vocab, vocab, skew=True, dtype=torch.int32)
        g = torch.randn(count // 4, 4, n, generator=gen(n), device="cuda").to(source)
        want, size, places = summed(g, t, vocab, 0.7, None)
        gw = algo.embedding_backward(torch.empty(vocab, n, dtype=target, device="cuda"), g, t, scale=0.7)
        info = torch.finfo(target)
        tol = (256 + places.double()[:, None] / 32 + 19) * U * size + info.eps / 2 * want.abs() * (1 + 2.0**-10) \
            + info.smallest_normal * info.eps
        assert ((gw.double() - want).abs() <= tol).all()
        again = algo.embedding_backward(torch.empty(vocab, n, dtype=target, device="cuda"), g, t, scale=0.7)
        assert torch.equal(gw, again)


@pytest.mark.parametrize("count", [1, 40, 2000, 9000, 70000])
def test_one_token_everywhere(cuda, count):
    from alpaka3_b200 import algo
    g = whole_numbers((count, 72), F32, 1)
    for token, vocab in ((0, 1), (4, 9), (8, 9)):
        t = torch.full((count,), token, device="cuda")
        gw = algo.embedding_backward(torch.full((vocab, 72), 7.0, device="cuda"), g, t)
        want = torch.zeros(vocab, 72, device="cuda")
        want[token] = g.double().sum(0).float()
        assert torch.equal(gw, want)
    gw = algo.embedding_backward(torch.full((9, 72), 7.0, device="cuda"), g, torch.full((count,), -1, device="cuda"))
    assert (gw == 0).all()


@pytest.mark.parametrize("count", [3000, 12000])
def test_sorted_and_reversed_tokens(cuda, count):
    from alpaka3_b200 import algo
    g = whole_numbers((count, 16), F32, 1)
    for t in (torch.arange(count, device="cuda"), torch.arange(count, device="cuda").flip(0),
              torch.arange(count, device="cuda") // 7, torch.arange(count, device="cuda") % 511,
              (torch.arange(count, device="cuda") % 512) * 1025):
        vocab = int(t.max()) + 2
        gw = algo.embedding_backward(torch.full((vocab, 16), 7.0, device="cuda"), g, t)
        assert torch.equal(gw.double(), summed(g, t, vocab, 1.0, None)[0])


@pytest.mark.parametrize("pair", PAIRS)
def test_few_tokens_of_many(cuda, pair):
    """Few tokens beside the table's rows: the table is filled while they are sorted. One stretch or strided rows, with and
    without packs, with and without something added; and at the counts where the way of sorting changes."""
    from alpaka3_b200 import algo
    source, target = pair
    for count, vocab, n in ((1, 16, 8), (1, 17, 5), (20, 1000, 64), (20, 1001, 33), (300, 5000, 7), (62, 1000, 24), (63, 1000, 24),
                            (4096, 70000, 8), (4097, 70000, 8), (16384, 3000, 8), (16385, 3000, 8)):
        t = pick((count,), vocab, count, skew=count > 20, outside=count > 2)
        g = whole_numbers((count, n), source, n)
        want = summed(g, t, vocab, 1.0, None)[0]
        gw = torch.full((vocab, n), 7.0, dtype=target, device="cuda")
        algo.embedding_backward(gw, g, t)
        assert torch.equal(gw, want.to(target)), (count, vocab, n)
        room = torch.full((vocab + 1, n + 8), 5.0, dtype=target, device="cuda")
        part = room[:vocab, 8 - n % 2:8 - n % 2 + n]
        algo.embedding_backward(part, g, t)
        assert torch.equal(part, want.to(target))
        add = whole_numbers((vocab, n), target, 3)
        algo.embedding_backward(part, g, t, add=add)
        assert torch.equal(part, (want + add.double()).to(target))
        part.fill_(5.0)
        assert (room == 5.0).all()
        # one stretch that begins off 16 bytes
        flat = torch.full((vocab * n + 2,), 5.0, dtype=target, device="cuda")
        algo.embedding_backward(flat[1:-1].view(vocab, n), g, t)
        assert torch.equal(flat[1:-1].view(vocab, n), want.to(target)) and flat[0] == 5 and flat[-1] == 5


def test_workspace_is_checked(cuda):
    from alpaka3_b200 import capi
    g, t, gw = torch.zeros(40, 64, device="cuda"), torch.zeros(40, dtype=torch.int64, device="cuda"), torch.zeros(9, 64, device="cuda")
    size = capi.lib().a3b_embedding_backward_workspace(40, 64, 9)
    ws = torch.empty(size + 16, dtype=torch.uint8, device="cuda")

    def call(at, bytes_):
        return capi.lib().a3b_embedding_backward(None, capi.EMBEDDING_BACKWARD_ARGS.pack(
            1, 40, 64, 9, 0, g.data_ptr(), 0, 64, t.data_ptr(), 0, 0, gw.data_ptr(), 64, at, bytes_, 1.0, capi.F32, capi.I64,
            capi.F32, 0))
    for at, bytes_ in ((0, size), (ws.data_ptr(), size - 1), (ws.data_ptr() + 8, size)):
        assert call(at, bytes_) == capi.ERR_INVALID and "workspace" in capi.last_error()
    assert call(ws.data_ptr(), size) == capi.OK
    torch.cuda.synchronize()


def test_no_tokens_and_infinities(cuda):
    from alpaka3_b200 import algo
    for n in (8, 5):
        none = torch.empty(0, dtype=torch.int64, device="cuda")
        w = table(6, n, F32)
        assert algo.embedding(torch.empty(0, n, device="cuda"), w, none).numel() == 0
        gw = algo.embedding_backward(torch.full((6, n), 7.0, device="cuda"), torch.empty(0, n, device="cuda"), none)
        assert (gw == 0).all()
        gw = algo.embedding_backward(torch.full((6, n), 7.0, device="cuda"), torch.empty(0, n, device="cuda"), none, add=w)
        assert torch.equal(gw, w)
        # what belongs to no token does not reach the gradient, whatever it is
        g = torch.ones(4, n, device="cuda")
        g[1], g[3] = math.nan, math.inf
        gw = algo.embedding_backward(torch.empty(6, n, device="cuda"), g, torch.tensor([2, -100, 2, 6], device="cuda"))
        assert (gw[2] == 2).all() and gw.sum() == 2 * n
        out = algo.embedding(torch.empty(2, n, device="cuda"), w.fill_(math.inf), torch.tensor([9, 1], device="cuda"))
        assert (out[0] == 0).all() and (out[1] == math.inf).all()


def test_gradient_layouts(cuda):
    from alpaka3_b200 import algo
    for source, target in PAIRS:
        for n, gap in ((64, 16), (64, 3), (37, 5)):
            g = whole_numbers((6, 7, n + gap), source, 2)[:, 1:6, gap:]
            t = pick((6, 5), 50, 1)
            room = torch.full((50, n + 2 * gap), 5.0, dtype=target, device="cuda")
            add = whole_numbers((50, n + gap), target, 4)[:, :n]
            gw = room[:, gap:gap + n]
            algo.embedding_backward(gw, g, t, add=add)
            assert torch.equal(gw, summed(g, t, 50, 1.0, add)[0].to(target))
            gw.fill_(5.0)
            assert (room == 5.0).all()


@pytest.mark.parametrize("count", [2000, 20000])
def test_streams_and_graphs(cuda, count):
    from alpaka3_b200 import algo
    vocab, n = 5000, 128
    t, g = pick((count,), vocab, 3, skew=True), torch.randn(count, n, generator=gen(1), device="cuda")
    want = algo.embedding_backward(torch.empty(vocab, n, device="cuda"), g, t)
    side = torch.cuda.Stream()
    got = torch.zeros(vocab, n, device="cuda")
    side.wait_stream(torch.cuda.current_stream())
    algo.embedding_backward(got, g, t, stream=side)
    side.synchronize()
    assert torch.equal(got, want)
    graphs, outs = [], []
    for _ in range(2):
        o = torch.zeros(vocab, n, device="cuda")
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            algo.embedding_backward(o, g, t)
        graphs.append(graph)
        outs.append(o)
    t.copy_(pick((count,), vocab, 9, skew=True))
    algo.embedding_backward(want, g, t)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_refusal_leaves_the_workspace(cuda):
    """A gradient of more blocks than one launch holds is refused before anything is launched. The table (2^31 - 65 rows of
    34816 elements) is an address that no kernel is given."""
    from alpaka3_b200 import capi
    n, vocab = 34816, 2**31 - 65
    for count in (40, 9000, 40000):  # sorted with the sums, by one cluster, in several launches
        g, t = torch.ones(1, n, device="cuda"), torch.arange(count, device="cuda")
        size = capi.lib().a3b_embedding_backward_workspace(count, n, vocab)
        ws = torch.full((size,), 7, dtype=torch.uint8, device="cuda")
        rc = capi.lib().a3b_embedding_backward(None, capi.EMBEDDING_BACKWARD_ARGS.pack(
            1, count, n, vocab, 0, g.data_ptr(), 0, 0, t.data_ptr(), 0, 0, 1 << 60, n, ws.data_ptr(), size, 1.0, capi.F32,
            capi.I64, capi.F32, 0))
        assert rc == capi.ERR_TOO_LARGE and "one launch" in capi.last_error()
        torch.cuda.synchronize()
        assert (ws == 7).all()


def test_longest_rows(cuda):
    """65535 * 512 accesses a row, by single elements and by packs of four; one more is refused before anything is launched."""
    from alpaka3_b200 import algo, capi
    most = 65535 * 512
    for n in (most - 1, 4 * most):
        room = torch.arange(n, device="cuda", dtype=torch.int32).bitwise_and_(0xffff).float()
        out = torch.zeros(2, n, device="cuda")
        algo.embedding(out, room[None], torch.tensor([0, 1], device="cuda"), scale=2.0)
        assert torch.equal(out[0], 2 * room) and (out[1] == 0).all()
    for n in (most + 1, 4 * most + 4):
        table, out = torch.ones(1, n, device="cuda"), torch.full((1, n), 7.0, device="cuda")
        with pytest.raises(capi.A3BError, match="one launch") as e:
            algo.embedding(out, table, torch.tensor([0], device="cuda"))
        assert e.value.status == capi.ERR_TOO_LARGE
        torch.cuda.synchronize()
        assert (out == 7).all()
