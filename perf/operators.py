"""What the language-model reductions are measured on: token log probabilities, their gradient, and the clipping of a
list of gradients by its global norm.

* ``logprobs``  ``algo.token_logprobs``: for every row of logits the log probability of its token, the entropy of the
                row's distribution, its log-sum-exp, and its most likely alternatives.
* ``backward``  ``algo.token_logprobs_backward``: the gradient of those three with respect to the logits.
* ``clip``      ``algo.clip_grad_norm``: the norm over all tensors of a list, and the tensors scaled down to it.

``run`` computes them in plain torch operations, or, where ``own`` is true, with the framework's kernels.
"""
import functools
import math
import random

import torch

own = False

_DTYPE = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
_SIZE = {"bf16": 2, "f16": 2, "f32": 4}


# ------------------------------------------------------------------------------------------------------- cases
def _rows_case(op, name, batch, rows, vocab, dtype, top=0, scale=1.0, masked=False, ignored=False):
    """`batch` sequences of `rows` rows each. With batch > 1 the logits are the first `rows` of rows + 1 positions of
    every sequence, as where position i predicts token i + 1."""
    return {"op": op, "name": name, "batch": batch, "rows": rows, "vocab": vocab, "dtype": dtype, "top": top,
            "scale": scale, "masked": masked, "ignored": ignored}


def _layers_case(name, width, layers, vocab, dtype):
    return {"op": "clip", "name": name, "form": "layers", "width": width, "layers": layers, "vocab": vocab,
            "dtype": dtype, "kind": "l2", "clips": True}


def _ragged_case(name, count, smallest, largest, dtype, pick, kind="l2", clips=True):
    return {"op": "clip", "name": name, "form": "ragged", "count": count, "smallest": smallest, "largest": largest,
            "pick": pick, "dtype": dtype, "kind": kind, "clips": clips}


def listed():
    return [
        # one sequence being decoded: a token was sampled at temperature 0.8, its 20 alternatives are reported
        _rows_case("logprobs", "decode 1x32000 bf16 top20", 1, 1, 32000, "bf16", top=20, scale=1.25),
        # a batch being decoded with 32-bit logits, some of the vocabulary ruled out by a grammar
        _rows_case("logprobs", "decode 64x131072 f32 top5", 1, 64, 131072, "f32", top=5, masked=True),
        # scoring a prompt: every position's token with its alternatives, vocabulary of an odd size
        _rows_case("logprobs", "prompt 2048x50257 bf16 top4", 1, 2048, 50257, "bf16", top=4),
        # a vocabulary of bytes: many short rows
        _rows_case("logprobs", "bytes 32768x257 f16 top2", 1, 32768, 257, "f16", top=2),
        # the forward pass of a training step: 8 sequences, prompt tokens left out of the loss
        _rows_case("logprobs", "train 8x1024x131072 bf16", 8, 1024, 131072, "bf16", ignored=True),
        # the gradient for a few rows: the answer tokens of a short episode
        _rows_case("backward", "episode 16x32000 bf16", 1, 16, 32000, "bf16", scale=1.25),
        # the gradient of a policy loss with an entropy bonus, vocabulary of an odd size
        _rows_case("backward", "policy 4x512x50257 bf16", 4, 512, 50257, "bf16", ignored=True, masked=True),
        # the gradient of a training step in 32 bits
        _rows_case("backward", "train 4096x131072 f32", 1, 4096, 131072, "f32", ignored=True),
        # the gradients of a few small adapters
        _ragged_case("adapters 10 f32", 10, 64, 8192, "f32", 1),
        # every gradient of a model with 12 layers of width 1024
        _layers_case("model 12 layers bf16", 1024, 12, 32000, "bf16"),
        # many tensors of any size one after the other in two buckets, one of 16-bit and one of 32-bit gradients
        _ragged_case("buckets 1000 mixed", 1000, 1, 1000000, "mixed", 2),
        # every gradient of a model with 20 layers of width 2048
        _layers_case("model 20 layers bf16", 2048, 20, 32000, "bf16"),
    ]


def _between(rng, low, high):
    """A whole number in [low, high], spread evenly over its logarithm; half of them odd."""
    n = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    return min(high, max(low, n | 1 if rng.random() < 0.5 else n))


def draw(rng):
    op = rng.choice(["logprobs", "logprobs", "backward", "clip"])
    if op == "clip":
        count = _between(rng, 1, 1500)
        largest = _between(rng, 2, min(1 << 26, (1 << 29) // count))
        return {"op": op, "form": "ragged", "count": count, "smallest": rng.choice([1, max(1, largest // 50)]),
                "largest": largest, "pick": rng.randrange(1 << 20), "dtype": rng.choice(["bf16", "f16", "f32", "mixed"]),
                "kind": rng.choice(["l2", "l2", "l2", "l1", "max"]), "clips": rng.random() < 0.75}
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    vocab = _between(rng, 33, 262144)
    top = rng.choice([0, rng.randint(1, 32)]) if op == "logprobs" else 0
    batch = rng.choice([1, 1, rng.randint(2, 8)])
    rows = _between(rng, 1, max(1, min(16384, ((1 << 26) if top else (1 << 28)) // vocab // batch)))
    return {"op": op, "batch": batch, "rows": rows, "vocab": vocab, "dtype": dtype, "top": top,
            "scale": rng.choice([1.0, 1.0, round(rng.uniform(0.5, 2.0), 3)]), "masked": rng.random() < 0.3,
            "ignored": rng.random() < 0.5}


def _sizes(case):
    """[(elements, dtype)] of a clip case's tensors, in order."""
    if case["form"] == "layers":
        w = case["width"]
        layer = [w, w * w, w * w, w * w, w * w, w, 4 * w * w, 4 * w * w]
        return [(n, case["dtype"]) for n in [case["vocab"] * w] + layer * case["layers"] + [w]]
    r = random.Random(case["pick"])
    low, high = math.log(case["smallest"]), math.log(case["largest"])
    sizes = [int(round(math.exp(r.uniform(low, high)))) for _ in range(case["count"])]
    return [(n, r.choice(["bf16", "f32"]) if case["dtype"] == "mixed" else case["dtype"]) for n in sizes]


# ------------------------------------------------------------------------------------------------------ states
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return _prepare_clip(case, g) if case["op"] == "clip" else _prepare_rows(case, g)


def _empty_rows(case, dtype):
    """Storage for the case's logits, or for their gradient: (rows, vocab), or (batch, rows, vocab) of longer ones."""
    b, n, v = case["batch"], case["rows"], case["vocab"]
    if b == 1:
        return torch.zeros(n, v, dtype=dtype, device="cuda")
    return torch.zeros(b, n + 1, v, dtype=dtype, device="cuda")[:, :-1]


def _prepare_rows(case, g):
    v, dtype = case["vocab"], _DTYPE[case["dtype"]]
    logits = _empty_rows(case, dtype)
    shape = logits.shape[:-1]
    flat = [logits] if case["batch"] == 1 else list(logits)
    targets = torch.randint(0, v, shape, generator=g, device="cuda")
    for part, goal in zip(flat, targets.view(len(flat), -1)):
        for lo in range(0, part.shape[0], 1024):  # in pieces: the random numbers are made in 32 bits
            x = torch.randn(part[lo:lo + 1024].shape, generator=g, device="cuda").mul_(2.5)
            # most tokens are likely ones
            x.scatter_add_(-1, goal[lo:lo + 1024, None], 6 * torch.rand(x.shape[0], 1, generator=g, device="cuda"))
            if case["masked"]:
                x.masked_fill_(torch.rand(x.shape, generator=g, device="cuda") < 0.3, -math.inf)
            part[lo:lo + 1024] = x.to(dtype)
            del x
    if case["ignored"]:
        targets.masked_fill_(torch.rand(shape, generator=g, device="cuda") < 0.2, -100)
    f32 = {"dtype": torch.float32, "device": "cuda"}
    s = {"case": case, "logits": logits, "targets": targets}
    if case["op"] == "logprobs":
        s |= {"logp": torch.empty(shape, **f32), "entropy": torch.empty(shape, **f32), "lse": torch.empty(shape, **f32),
              "top_logp": torch.empty(*shape, case["top"], **f32),
              "top_index": torch.empty(*shape, case["top"], dtype=torch.int64, device="cuda")}
        return s
    # what the forward pass left, and what arrives from the loss
    lse, entropy = torch.empty(shape, **f32), torch.empty(shape, **f32)
    for part, a, b in zip(flat, lse.view(len(flat), -1), entropy.view(len(flat), -1)):
        for lo in range(0, part.shape[0], 256):
            got = _exact_rows(part[lo:lo + 256], case["scale"])
            a[lo:lo + 256], b[lo:lo + 256] = got["lse"].float(), got["entropy"].float()
    grads = [torch.randn(shape, generator=g, device="cuda") for _ in range(3)]
    return s | {"lse": lse, "entropy": entropy, "grad_logp": grads[0], "grad_entropy": grads[1].mul_(0.01),
                "grad_lse": grads[2].mul_(0.001), "grad_logits": _empty_rows(case, dtype)}


def _prepare_clip(case, g):
    sizes = _sizes(case)
    flat, out, at = {}, {}, {}
    for d in sorted({d for _, d in sizes}):
        n = sum(k for k, t in sizes if t == d)
        flat[d] = torch.empty(n, dtype=_DTYPE[d], device="cuda")
        for lo in range(0, n, 1 << 27):
            part = flat[d][lo:lo + (1 << 27)]
            part.copy_(torch.randn(part.shape, generator=g, device="cuda").mul_(0.02))
        out[d], at[d] = torch.zeros_like(flat[d]), 0
    ins, outs = [], []
    for k, d in sizes:  # the tensors of a bucket follow one another without gaps
        ins.append(flat[d][at[d]:at[d] + k])
        outs.append(out[d][at[d]:at[d] + k])
        at[d] += k
    total = sum(k for k, _ in sizes)
    expect = {"l2": 0.02 * math.sqrt(total), "l1": 0.016 * total, "max": 0.05}[case["kind"]]
    s = {"case": case, "ins": ins, "outs": outs, "flat_out": out, "max_norm": expect * (0.25 if case["clips"] else 4.0),
         "norm": torch.empty(1, dtype=torch.float32, device="cuda")}
    if own:  # the list that a training program makes once for its gradient buffers
        s["list"] = _framework().TensorList(ins, outs)
    return s


# -------------------------------------------------------------------------------------------------- one pass
def run(s):
    if own:
        return _own(s)
    op = s["case"]["op"]
    return _plain_clip(s) if op == "clip" else _plain_backward(s) if op == "backward" else _plain_logprobs(s)


@functools.cache
def _framework():
    from alpaka3_b200 import algo
    return algo


def _own(s):
    algo, case = _framework(), s["case"]
    if case["op"] == "clip":
        algo.clip_grad_norm(s["norm"], s["list"], s["max_norm"], case["kind"])
        return {"norm": s["norm"], "grads": s["flat_out"]}
    if case["op"] == "backward":
        algo.token_logprobs_backward(s["grad_logits"], s["logits"], s["targets"], s["lse"], entropy=s["entropy"],
                                     grad_logp=s["grad_logp"], grad_entropy=s["grad_entropy"],
                                     grad_lse=s["grad_lse"], scale=case["scale"])
        return {"grad_logits": s["grad_logits"]}
    top = {"top_logp": s["top_logp"], "top_index": s["top_index"]} if case["top"] else {}
    algo.token_logprobs(s["logp"], s["logits"], s["targets"], entropy=s["entropy"], lse=s["lse"], scale=case["scale"],
                        **top)
    return {"logp": s["logp"], "entropy": s["entropy"], "lse": s["lse"], **top}


def _plain_logprobs(s):
    case = s["case"]
    z = s["logits"].float()
    if case["scale"] != 1.0:
        z = z * case["scale"]
    high = z.amax(-1, keepdim=True)
    high = torch.where(high == -math.inf, torch.zeros_like(high), high)  # a row with nothing left
    e = torch.exp(z - high)
    total = e.sum(-1, keepdim=True)
    lse = high + torch.log(total)
    z = z - torch.where(lse == -math.inf, torch.zeros_like(lse), lse)  # the log probabilities
    p = e / torch.where(total == 0, torch.ones_like(total), total)
    entropy = -torch.where(p > 0, p * z, torch.zeros_like(p)).sum(-1)
    t = s["targets"]
    counts = (t >= 0) & (t < case["vocab"])
    logp = z.gather(-1, torch.where(counts, t, torch.zeros_like(t))[..., None])[..., 0]
    out = {"logp": torch.where(counts, logp, torch.zeros_like(logp)), "entropy": entropy, "lse": lse[..., 0]}
    if case["top"]:
        # by the logits as they are, a tie to the lowest index
        order = torch.sort(s["logits"].float(), dim=-1, descending=True, stable=True)[1][..., :case["top"]].contiguous()
        out |= {"top_logp": z.gather(-1, order), "top_index": order}
    return out


def _plain_backward(s):
    case = s["case"]
    t, v = s["targets"], case["vocab"]
    counts = (t >= 0) & (t < v)
    some = s["lse"] != -math.inf
    lse = torch.where(some, s["lse"], torch.zeros_like(s["lse"]))
    zero = torch.zeros_like(lse)
    z = s["logits"].float()
    if case["scale"] != 1.0:
        z = z * case["scale"]
    z = z - lse[..., None]
    p = torch.exp(z)
    g = torch.where(counts & some, s["grad_logp"], zero)
    plogp = torch.where(p > 0, p * (z + s["entropy"][..., None]), torch.zeros_like(p))
    d = p * (s["grad_lse"] - g)[..., None] - plogp * s["grad_entropy"][..., None]
    d.scatter_add_(-1, torch.where(counts, t, torch.zeros_like(t))[..., None], g[..., None])
    if case["scale"] != 1.0:
        d = d * case["scale"]
    return {"grad_logits": d.to(s["logits"].dtype)}


def _plain_clip(s):
    kind = s["case"]["kind"]
    named = {torch.bfloat16: "bf16", torch.float16: "f16", torch.float32: "f32"}
    flats = {d: torch.cat([x for x in s["ins"] if named[x.dtype] == d]).float() for d in s["flat_out"]}
    if kind == "max":
        norm = torch.stack([x.abs().amax() for x in flats.values()]).amax().double()
    elif kind == "l1":
        norm = torch.stack([x.abs().sum(dtype=torch.float64) for x in flats.values()]).sum()
    else:
        norm = torch.stack([x.square().sum(dtype=torch.float64) for x in flats.values()]).sum().sqrt()
    factor = torch.clamp(s["max_norm"] / (norm + 1e-6), max=1.0).float()
    return {"norm": norm.float().reshape(1), "grads": {d: (x * factor).to(_DTYPE[d]) for d, x in flats.items()}}


# ---------------------------------------------------------------------------------------------- what it costs
def work(case):
    """Every input read once and every output written once; the operations on each element counted by hand."""
    if case["op"] == "clip":
        n = sum(k for k, _ in _sizes(case))
        return {"bytes": 2 * sum(k * _SIZE[d] for k, d in _sizes(case)) + 4, "flops": 3 * n}
    rows = case["batch"] * case["rows"]
    n = rows * case["vocab"]
    if case["op"] == "backward":
        return {"bytes": 2 * n * _SIZE[case["dtype"]] + rows * (8 + 5 * 4), "flops": 8 * n}
    return {"bytes": n * _SIZE[case["dtype"]] + rows * (8 + 3 * 4 + case["top"] * 12), "flops": 7 * n}


# ------------------------------------------------------------------------------------------------ in 64 bits
def _exact_rows(logits, scale):
    """Log-sum-exp, entropy and log probabilities of 2-D logits, by their definition in 64 bits."""
    z = logits.double() * scale
    lse = torch.logsumexp(z, -1)
    q = z - torch.where(lse == -math.inf, torch.zeros_like(lse), lse)[:, None]
    return {"lse": lse, "q": q, "entropy": -torch.nan_to_num(q * q.exp(), nan=0.0, neginf=0.0).sum(-1)}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "clip":
        big = {"l2": lambda x: x.double().square().sum(), "l1": lambda x: x.double().abs().sum(),
               "max": lambda x: x.double().abs().max()}[case["kind"]]
        parts = torch.stack([big(x) for x in s["ins"]])
        norm = {"l2": parts.sum().sqrt(), "l1": parts.sum(), "max": parts.max()}[case["kind"]].item()
        factor = min(1.0, s["max_norm"] / (norm + 1e-6))
        named = {torch.bfloat16: "bf16", torch.float16: "f16", torch.float32: "f32"}
        grads = {d: torch.cat([x.double() * factor for x in s["ins"] if named[x.dtype] == d]) for d in s["flat_out"]}
        return {"norm": torch.tensor([norm], dtype=torch.float64), "grads": grads}
    shape, v = s["logits"].shape, case["vocab"]
    flat, targets = s["logits"].reshape(-1, v), s["targets"].reshape(-1)
    step = max(1, (1 << 26) // v)
    if case["op"] == "backward":
        out = torch.empty(flat.shape, dtype=torch.float64, device="cuda")
        cols = {k: s[k].reshape(-1).double() for k in ("lse", "entropy", "grad_logp", "grad_entropy", "grad_lse")}
        for lo in range(0, flat.shape[0], step):
            c = {k: x[lo:lo + step, None] for k, x in cols.items()}
            t = targets[lo:lo + step, None]
            q = flat[lo:lo + step].double() * case["scale"] - c["lse"]
            empty = c["lse"] == -math.inf
            hit = (torch.arange(v, device="cuda")[None] == t).double()
            counts = ((t >= 0) & (t < v)).double()
            pq = torch.nan_to_num(q.exp() * (q + c["entropy"]), nan=0.0)
            d = c["grad_logp"] * (hit - counts * q.exp()) + c["grad_lse"] * q.exp() - c["grad_entropy"] * pq
            out[lo:lo + step] = torch.where(empty, torch.zeros_like(d), d * case["scale"])
        return {"grad_logits": out.reshape(shape)}
    parts = []
    for lo in range(0, flat.shape[0], step):
        got = _exact_rows(flat[lo:lo + step], case["scale"])
        t = targets[lo:lo + step]
        counts = (t >= 0) & (t < v)
        here = got["q"][torch.arange(len(t), device="cuda"), t.clamp(0, v - 1)]
        row = {"logp": torch.where(counts, here, torch.zeros_like(here)), "entropy": got["entropy"], "lse": got["lse"]}
        if case["top"]:
            # the rank of an element: how many are larger, or as large and further left
            order = torch.argsort(flat[lo:lo + step].double(), dim=-1, descending=True, stable=True)[:, :case["top"]]
            row |= {"top_logp": got["q"].gather(-1, order), "top_index": order}
        parts.append(row)
    out = {k: torch.cat([p[k] for p in parts]) for k in parts[0]}
    return {k: x.reshape(*shape[:-1], *x.shape[1:]) for k, x in out.items()}
