"""CPU: the checks of arguments of the row reductions and the gradient lists (they run before any CUDA call), and the
combination of norm partials over two gloo ranks."""
import ctypes
import math

import pytest
import torch


@pytest.fixture(scope="module")
def L():
    if torch.cuda.is_available():
        pytest.skip("the addresses in these calls are made up: only where no GPU could use one")
    from alpaka3_b200 import capi
    return capi.lib()


P = ctypes.c_void_p(0x10000000)  # stands for a device address: nothing below may use it
ODD = ctypes.c_void_p(0x10000001)


def forward(L, **kw):
    from alpaka3_b200 import capi
    a = dict(dtype=capi.F32, logits=P, outer=1, inner=4, vocab=100, so=0, si=100, scale=1.0, index=capi.I64, targets=P,
             logp=P, entropy=None, lse=None, top=0, top_logp=None, top_index=None)
    a.update(kw)
    return L.a3b_token_logprobs(None, *a.values())


def backward(L, **kw):
    from alpaka3_b200 import capi
    a = dict(dtype=capi.F32, logits=P, outer=1, inner=4, vocab=100, so=0, si=100, scale=1.0, index=capi.I64, targets=P,
             lse=P, entropy=None, grad_logp=P, grad_entropy=None, grad_lse=None, grad=ctypes.c_void_p(0x20000000), gso=0,
             gsi=100)
    a.update(kw)
    return L.a3b_token_logprobs_backward(None, *a.values())


def test_forward_refusals(L):
    from alpaka3_b200 import capi
    for kw in (dict(dtype=capi.F64), dict(dtype=capi.I32), dict(dtype=99), dict(index=capi.U32), dict(vocab=0),
               dict(scale=0.0), dict(scale=-1.0), dict(scale=math.inf), dict(scale=math.nan), dict(scale=1e-60),
               dict(logits=None), dict(logits=ctypes.c_void_p(0x10000002)), dict(logp=None), dict(targets=None),
               dict(top=33, top_logp=P, top_index=P), dict(top=5), dict(top=5, top_logp=P),
               dict(vocab=3, top=4, top_logp=P, top_index=P), dict(outer=1 << 63, inner=4), dict(targets=ODD),
               dict(logp=ODD), dict(entropy=ODD), dict(lse=ODD), dict(top=5, top_logp=ODD, top_index=P),
               dict(top=5, top_logp=P, top_index=ODD), dict(index=capi.I32, targets=ctypes.c_void_p(0x10000002))):
        assert forward(L, **kw) == capi.ERR_INVALID, kw
        assert capi.last_error()
    for kw in (dict(vocab=(1 << 31) - 64), dict(inner=1 << 31), dict(outer=1 << 16, inner=1 << 16)):
        assert forward(L, **kw) == capi.ERR_TOO_LARGE, kw
    assert forward(L, inner=0, logits=None) == capi.OK  # no rows


def test_backward_refusals(L):
    from alpaka3_b200 import capi
    for kw in (dict(lse=None), dict(grad=None), dict(targets=None), dict(grad_entropy=P), dict(scale=0.0),
               dict(grad=ctypes.c_void_p(0x20000001)), dict(gsi=99), dict(gsi=0), dict(gsi=-50),
               dict(outer=3, gso=399, gsi=100), dict(outer=3, gso=0), dict(grad=ctypes.c_void_p(0x10000004)),
               dict(grad=P, gsi=101), dict(grad=ctypes.c_void_p(0x10000000 + 1596)),
               dict(grad=ctypes.c_void_p(0x10000000 - 1596)), dict(si=1 << 62), dict(lse=ODD), dict(entropy=ODD),
               dict(grad_logp=ODD), dict(grad_entropy=ODD, entropy=P), dict(grad_lse=ODD), dict(targets=ODD)):
        rc = backward(L, **kw)
        assert rc == capi.ERR_INVALID, (kw, rc)
    assert backward(L, inner=0) == capi.OK


def make(L, ins, outs, sizes, dtypes):
    n = len(ins)
    h = ctypes.c_void_p()
    rc = L.a3b_tensor_list_create((ctypes.c_void_p * n)(*ins), None if outs is None else (ctypes.c_void_p * n)(*outs),
                                  (ctypes.c_uint64 * n)(*sizes), (ctypes.c_int * n)(*dtypes), n, ctypes.byref(h))
    return rc, h


def test_list_refusals(L):
    from alpaka3_b200 import capi
    F, B, D = capi.F32, capi.BF16, capi.F64
    for ins, outs, sizes, dtypes in (([0x1000], None, [4], [capi.I32]), ([None], None, [4], [F]),
                                     ([0x1002], None, [4], [F]), ([0x1000], [0x2001], [4], [B]),
                                     ([0x1004], None, [4], [D]), ([0x1000], None, [1 << 60], [F])):
        rc, h = make(L, ins, outs, sizes, dtypes)
        assert rc == capi.ERR_INVALID and not h.value, (ins, rc)
    assert L.a3b_tensor_list_create(None, None, None, None, 2, ctypes.byref(ctypes.c_void_p())) == capi.ERR_INVALID
    assert L.a3b_tensor_list_create(None, None, None, None, 0, None) == capi.ERR_INVALID
    assert L.a3b_tensor_list_destroy(None) == capi.OK
    rc, h = make(L, [], None, [], [])
    assert rc == capi.OK
    for kind, limit, dt, p in ((9, 1.0, F, P), (0, -1.0, F, P), (0, math.nan, F, P), (0, 1.0, B, P), (0, 1.0, F, None)):
        assert L.a3b_clip_grads(None, h, kind, p, limit, dt, P) == capi.ERR_INVALID
    assert L.a3b_clip_grads(None, None, 0, P, 1.0, F, P) == capi.ERR_INVALID
    assert L.a3b_grad_norm(None, h, 0, P, 8, None, F, None) == capi.ERR_INVALID  # no output
    assert L.a3b_grad_norm(None, h, 0, None, 8, P, F, None) == capi.ERR_INVALID
    assert L.a3b_grad_norm(None, h, 0, ctypes.c_void_p(0x10004), 8, P, F, None) == capi.ERR_INVALID
    assert L.a3b_clip_grad_norm(None, h, 0, 1.0, None, 0, F, P) == capi.ERR_INVALID
    assert L.a3b_clip_grad_norm(None, h, 0, 1.0, P, 64, F, ODD) == capi.ERR_INVALID
    assert L.a3b_clip_grad_norm(None, h, 0, 1.0, P, 64, D, ctypes.c_void_p(0x10004)) == capi.ERR_INVALID
    assert L.a3b_grad_norm(None, h, 0, P, 64, ctypes.c_void_p(0x10004), F, P) == capi.ERR_INVALID
    assert L.a3b_clip_grads(None, h, 0, ctypes.c_void_p(0x10004), 1.0, F, P) == capi.ERR_INVALID
    assert L.a3b_tensor_list_destroy(h) == capi.OK


def overlapping(ins, outs, sizes):
    """by comparing all pairs"""
    n = len(ins)
    hit = lambda a, b, na, nb: na and nb and a < b + 4 * nb and b < a + 4 * na  # noqa: E731
    for i in range(n):
        for j in range(n):
            if i != j and hit(outs[i], outs[j], sizes[i], sizes[j]):
                return True
            if hit(outs[i], ins[j], sizes[i], sizes[j]) and not (i == j and outs[i] == ins[i]):
                return True
    return False


def test_overlaps_against_all_pairs(L):
    """Random small lists: scaling is refused exactly where an output touches another tensor."""
    import random

    from alpaka3_b200 import capi
    r = random.Random(4)
    seen = {True: 0, False: 0}
    for _ in range(3000):
        n = r.randint(1, 5)
        sizes = [r.randint(0, 6) for _ in range(n)]
        if r.random() < 0.5:  # mostly apart
            at = [4096 + 4 * 10 * k for k in r.sample(range(2 * n), 2 * n)]
            ins = at[:n]
            outs = [i if r.random() < 0.5 else o for i, o in zip(ins, at[n:])]
            if r.random() < 0.4:
                outs[r.randrange(n)] += 4 * r.randint(0, 12)
        else:
            ins = [4096 + 4 * r.randint(0, 40) for _ in range(n)]
            outs = [i if r.random() < 0.6 else 4096 + 4 * r.randint(0, 40) for i in ins]
        rc, h = make(L, ins, outs, sizes, [capi.F32] * n)
        assert rc == capi.OK
        # refused for its limit, if not before that for an overlap
        rc = L.a3b_clip_grads(None, h, 0, P, math.nan, capi.F32, None)
        refused = rc == capi.ERR_INVALID and "overlap" in capi.last_error()
        L.a3b_tensor_list_destroy(h)
        want = overlapping(ins, outs, sizes)
        assert refused == want, (ins, outs, sizes)
        seen[want] += 1
    assert min(seen.values()) > 300


def test_row_layouts():
    from alpaka3_b200 import algo
    x = torch.empty(4, 6, 10)
    assert algo._rows(x, "x") == (1, 24, 0, 10)
    assert algo._rows(x[:, :-1], "x") == (4, 5, 60, 10)
    assert algo._rows(x.transpose(0, 1), "x") == (6, 4, 10, 60)
    assert algo._rows(x[0, 0], "x")[:2] == (1, 1)
    assert algo._rows(x[:1, :, :7], "x") == (1, 6, 0, 10)
    assert algo._rows(x[:0], "x")[1] == 0
    assert algo._rows(torch.empty(2, 3, 4, 5), "x") == (1, 24, 0, 5)
    assert algo._rows(torch.empty(5).expand(3, 5), "x") == (1, 3, 0, 0)
    for bad in (x.transpose(1, 2), x[..., ::2], torch.empty(2, 3, 4, 5)[:, :-1, :-1], torch.empty(())):
        with pytest.raises(ValueError):
            algo._rows(bad, "x")


def test_dense_layouts():
    from alpaka3_b200 import algo
    x = torch.empty(4, 6, 10)
    for t in (x, x.permute(2, 0, 1), x[1], x[:1], torch.empty(()), torch.empty(0, 3), torch.empty(3, 1, 5).transpose(0, 1)):
        assert algo._is_dense(t)
    for t in (x[:, :-1], x[..., ::2], torch.empty(5).expand(3, 5), x[:, 0]):
        assert not algo._is_dense(t)


def test_cpu_tensors_are_refused():
    from alpaka3_b200 import algo
    x = torch.zeros(2, 5)
    with pytest.raises(ValueError):
        algo.token_logprobs(torch.empty(2), x, torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError):
        algo.TensorList([x])
    with pytest.raises(TypeError):
        algo.token_logprobs(torch.empty(2), x.double(), torch.zeros(2, dtype=torch.int64))
    assert len(algo.TensorList([])) == 0


def _norm_worker(rank, port, q):
    import torch.distributed as td

    from alpaka3_b200 import dist as ad
    td.init_process_group("gloo", init_method=f"tcp://127.0.0.1:{port}", rank=rank, world_size=2)
    try:
        one = lambda v: torch.tensor([v], dtype=torch.float64)  # noqa: E731
        q.put((rank, ad.combine_norm(one((1.5 + rank) ** 2)).item(), ad.combine_norm(one(1.5 + rank), "max").item(),
               ad.combine_norm(one(math.nan if rank else 3.0), "max").item()))
        q.close()
        q.join_thread()
    finally:
        td.destroy_process_group()


def test_combined_norm_two_ranks():
    import socket

    import torch.multiprocessing as mp
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    procs = [ctx.Process(target=_norm_worker, args=(r, port, q)) for r in range(2)]
    for p in procs:
        p.start()
    got = [q.get(timeout=120) for _ in procs]
    for p in procs:
        p.join(timeout=60)
        assert p.exitcode == 0
    for _, l2, largest, nan in got:
        assert l2 == 1.5**2 + 2.5**2 and largest == 2.5 and math.isnan(nan)


def test_combined_norm_one_rank():
    from alpaka3_b200 import dist as ad
    assert ad.combine_norm(torch.tensor([4.0], dtype=torch.float64)).item() == 4.0


class _CpuList:
    """Stands for algo.TensorList where there is no GPU."""

    def __init__(self, inputs):
        self.inputs = list(inputs)
        self.device = self.inputs[0].device if self.inputs else None


def _cpu_grad_norm(norm, tensors, kind="l2", partial=None):
    x = torch.cat([t.double().flatten() for t in tensors.inputs] + [torch.zeros(1, dtype=torch.float64)])
    partial.copy_((x.square().sum() if kind == "l2" else x.abs().max()).reshape(1))


def _cpu_clip_grads(norm, tensors, partial, max_norm, kind="l2"):
    value = partial.sqrt() if kind == "l2" else partial
    for t in tensors.inputs:
        t.mul_(min(1.0, max_norm / (value.item() + 1e-6)))
    return None if norm is None else norm.copy_(value)


def _clip_worker(rank, port, q):
    """dist.clip_grad_norm on gloo with the kernels' calls replaced: rank 1 has no shard."""
    import torch.distributed as td

    from alpaka3_b200 import algo
    from alpaka3_b200 import dist as ad
    algo.TensorList, algo.grad_norm, algo.clip_grads = _CpuList, _cpu_grad_norm, _cpu_clip_grads
    td.init_process_group("gloo", init_method=f"tcp://127.0.0.1:{port}", rank=rank, world_size=2)
    try:
        got = []
        for given in (False, True):
            for kind in ("l2", "max"):
                shard = [] if rank else [torch.full((8,), 3.0), torch.full((2,), 4.0)]
                norm = torch.zeros(1) if given else None
                res = ad.clip_grad_norm(norm, shard, 1.0, kind)
                got.append((None if res is None else res.item(), [t[0].item() for t in shard]))
        q.put((rank, got))
        q.close()
        q.join_thread()
    finally:
        td.destroy_process_group()


def test_sharded_clipping_two_ranks():
    """Every rank takes the same steps: with and without a norm to write, with and without a shard."""
    import socket

    import torch.multiprocessing as mp
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    procs = [ctx.Process(target=_clip_worker, args=(r, port, q)) for r in range(2)]
    for p in procs:
        p.start()
    got = dict(q.get(timeout=120) for _ in procs)
    for p in procs:
        p.join(timeout=60)
        assert p.exitcode == 0
    total = math.sqrt(8 * 9 + 2 * 16)
    for rank in range(2):
        for (norm, values), given, size in zip(got[rank], (False, False, True, True), (total, 4.0, total, 4.0)):
            assert (abs(norm - size) <= 2.0**-23 * size) if given else norm is None
            want = [] if rank else [3.0 / size, 4.0 / size]
            assert len(values) == len(want) and all(abs(a - b) <= 1e-5 for a, b in zip(values, want))


def test_norm_and_partial_apart(L):
    """The norm is written while other blocks still read the partial: one stretch of memory for both is refused."""
    from alpaka3_b200 import capi
    F, D = capi.F32, capi.F64
    rc, h = make(L, [0x40000000], None, [100], [F])
    assert rc == capi.OK
    at = lambda d: ctypes.c_void_p(0x10000000 + d)  # noqa: E731
    for dtype, d, hit in ((D, 0, True), (F, 0, True), (F, 4, True), (D, 8, False), (F, 8, False), (F, -4, False),
                          (D, -8, False)):
        for call in (lambda: L.a3b_clip_grads(None, h, 0, P, math.nan, dtype, at(d)),  # refused for its limit if not before
                     lambda: L.a3b_grad_norm(None, h, 0, None, 0, P, dtype, at(d))):  # ... for the lack of a workspace
            assert call() == capi.ERR_INVALID
            assert ("overlap" in capi.last_error()) == hit, (dtype, d, capi.last_error())
    L.a3b_tensor_list_destroy(h)


def test_parameters_without_a_gradient():
    """[p.grad for p in parameters] may hold None: such a parameter is left out, with its output."""
    from alpaka3_b200 import algo
    assert len(algo.TensorList([None, None])) == 0 and algo.TensorList([None]).device is None
    assert len(algo.TensorList([None], [torch.zeros(3)])) == 0
    with pytest.raises(ValueError, match="equally many"):
        algo.TensorList([None], [])
    with pytest.raises(ValueError, match="CUDA"):  # what is left is checked as ever
        algo.TensorList([None, torch.zeros(3)])
