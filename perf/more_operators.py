"""What the operators around a language model's layers are measured on: tokens to rows, rows to normed rows, drafted
tokens to accepted ones.

* ``norm``       ``algo.rms_norm``: rows plus residual, divided by their root mean square, times a weight; in the rows'
                 type, or in 8 bits with scales.
* ``norm_back``  ``algo.rms_norm_backward``: the gradients with respect to the rows and to the weight.
* ``embed``      ``algo.embedding``: the rows of a table that tokens name, scaled.
* ``embed_back`` ``algo.embedding_backward``: the gradient with respect to the table.
* ``verify``     ``algo.verify_drafts``: how many drafted tokens stand against the target's probabilities, and the token
                 drawn behind them, from given random numbers.

``run`` computes them in plain torch operations, or, where ``own`` is true, with the framework's kernels.
"""
import functools
import math

import torch

own = False

_DTYPE = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32, "e4m3": torch.float8_e4m3fn,
          "e5m2": torch.float8_e5m2}
_SIZE = {"bf16": 2, "f16": 2, "f32": 4, "e4m3": 1, "e5m2": 1}
_LARGEST = {"e4m3": 448.0, "e5m2": 57344.0}
_EPS = 1e-6


# ------------------------------------------------------------------------------------------------------- cases
def _norm_case(name, rows, width, dtype, out=None, group=0, residual=True, gap=0, weight=None):
    """out: the outputs' type; group: elements that share a scale (0: a row's). gap: elements between two rows of x, as
    where x is a part of a wider product."""
    return {"op": "norm", "name": name, "rows": rows, "width": width, "dtype": dtype, "out": out or dtype, "group": group,
            "residual": residual, "gap": gap, "weight": weight or dtype}


def _norm_back_case(name, rows, width, dtype, residual=True, weight=None):
    return {"op": "norm_back", "name": name, "rows": rows, "width": width, "dtype": dtype, "residual": residual,
            "weight": weight or dtype}


def _embed_case(op, name, tokens, width, vocab, dtype, scale=1.0, to=None, ignored=False, add=False):
    """to: the type of the output (embed), or of the table's gradient (embed_back)."""
    return {"op": op, "name": name, "tokens": tokens, "width": width, "vocab": vocab, "dtype": dtype, "scale": scale,
            "to": to or dtype, "ignored": ignored, "add": add}


def _verify_case(name, batch, drafts, vocab, dtype, model=True, scale=1.0, masked=False, ragged=False):
    """model: the drafts come from a model whose logits are given, not from a search that is sure of them."""
    return {"op": "verify", "name": name, "batch": batch, "drafts": drafts, "vocab": vocab, "dtype": dtype, "model": model,
            "scale": scale, "masked": masked, "ragged": ragged}


def listed():
    return [
        # one token being decoded: the layer's output joins the residual stream
        _norm_case("norm decode 1x4096 bf16", 1, 4096, "bf16"),
        # queries of every head of a prompt, a part of a wider product's rows
        _norm_case("norm heads 65536x128 bf16", 65536, 128, "bf16", residual=False, gap=64, weight="f32"),
        # a prompt in front of an 8-bit product: scales for groups of 128
        _norm_case("norm prompt 8192x8192 bf16 e4m3", 8192, 8192, "bf16", out="e4m3", group=128),
        # the backward pass of a training step, with the gradient that comes along the residual stream
        _norm_back_case("norm back 16384x2048 bf16", 16384, 2048, "bf16"),
        # that of a small model of an odd width in 32 bits
        _norm_back_case("norm back 2000x1001 f32", 2000, 1001, "f32", residual=False),
        # a batch being decoded
        _embed_case("embed", "embed decode 64x2048 bf16", 64, 2048, 32000, "bf16"),
        # the prompts of a batch, table in 32 bits, padding among the tokens
        _embed_case("embed", "embed 32768x4096 f32 to bf16", 32768, 4096, 50257, "f32", scale=64.0, to="bf16",
                    ignored=True),
        # the gradient of an episode's few tokens
        _embed_case("embed_back", "embed back 512x1024 f32", 512, 1024, 32000, "f32"),
        # that of a training step, into a table of an odd vocabulary
        _embed_case("embed_back", "embed back 65536x2048 bf16", 65536, 2048, 50257, "bf16", scale=2.0, ignored=True),
        # one sequence whose drafts were looked up in its own text
        _verify_case("verify 1x4 32000 bf16 looked up", 1, 4, 32000, "bf16", model=False, scale=1.25),
        # a batch whose drafts come from a small model
        _verify_case("verify 64x4 131072 bf16", 64, 4, 131072, "bf16"),
        # many sequences in 32 bits, vocabulary of an odd size, some ruled out, drafts of several lengths
        _verify_case("verify 256x3 50257 f32", 256, 3, 50257, "f32", masked=True, ragged=True),
    ]


def _between(rng, low, high):
    """A whole number in [low, high], spread evenly over its logarithm; half of them odd."""
    n = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    return min(high, max(low, n | 1 if rng.random() < 0.5 else n))


def _width(rng, high):
    n = _between(rng, 16, high)
    return n if rng.random() < 0.4 else max(16, n // 16 * 16)


def draw(rng):
    op = rng.choice(["norm", "norm", "norm_back", "embed", "embed_back", "verify", "verify"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op == "verify":
        vocab, drafts = _between(rng, 33, 262144), rng.choice([0, 1, 2, 3, 4, 5, 7, 8])
        batch = _between(rng, 1, max(1, min(512, (1 << 25) // vocab // (drafts + 1))))
        case = _verify_case("", batch, drafts, vocab, dtype, rng.random() < 0.6, rng.choice([1.0, round(rng.uniform(0.6, 1.6), 3)]),
                            rng.random() < 0.3, rng.random() < 0.5)
    elif op in ("norm", "norm_back"):
        width = _width(rng, 32768)
        rows = _between(rng, 1, max(1, min(65536, (1 << 25) // width)))
        weight = rng.choice([dtype, dtype, "f32"])
        if op == "norm_back":
            case = _norm_back_case("", rows, width, dtype, rng.random() < 0.6, weight)
        else:
            out = rng.choice([dtype, dtype, "e4m3", "e5m2"])
            case = _norm_case("", rows, width, dtype, out, rng.choice([0, 32, 64, 128]) if out[0] == "e" else 0,
                              rng.random() < 0.6, rng.choice([0, 0, 16, 5]), weight)
    else:
        width = _width(rng, 8192)
        vocab = _between(rng, 33, max(33, min(262144, (1 << 26) // width)))
        tokens = _between(rng, 1, max(1, min(131072, (1 << 26) // width)))
        to = rng.choice([dtype, dtype, "f32"]) if dtype != "f32" or op == "embed_back" else rng.choice(["f32", "bf16", "f16"])
        case = _embed_case(op, "", tokens, width, vocab, dtype, rng.choice([1.0, round(math.sqrt(width), 3)]), to,
                           rng.random() < 0.4, op == "embed_back" and rng.random() < 0.3)
    del case["name"]
    return case


# ------------------------------------------------------------------------------------------------------ states
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return {"norm": _prepare_norm, "norm_back": _prepare_norm_back, "embed": _prepare_embed, "embed_back": _prepare_embed_back,
            "verify": _prepare_verify}[case["op"]](case, g)


def _normal(g, rows, width, dtype, scale=1.0, gap=0):
    """Random rows; `gap` elements lie between one and the next."""
    out = torch.zeros(rows, width + gap, dtype=_DTYPE[dtype], device="cuda")[:, :width]
    for lo in range(0, rows, max(1, (1 << 25) // width)):
        part = out[lo:lo + max(1, (1 << 25) // width)]
        part.copy_(torch.randn(part.shape, generator=g, device="cuda").mul_(scale))
    return out


def _blank(shape, dtype):
    return torch.zeros(shape, dtype=_DTYPE.get(dtype, dtype), device="cuda")


def _groups(case):
    return 1 if case["group"] == 0 else -(-case["width"] // case["group"])


def _prepare_norm(case, g):
    rows, width, dtype = case["rows"], case["width"], case["dtype"]
    s = {"case": case, "x": _normal(g, rows, width, dtype, 0.7, case["gap"]),
         "weight": (1 + 0.2 * torch.randn(width, generator=g, device="cuda")).to(_DTYPE[case["weight"]]),
         "out": _blank((rows, width), case["out"]), "rstd": _blank(rows, "f32")}
    if case["residual"]:  # the stream grows from layer to layer
        s |= {"residual": _normal(g, rows, width, dtype, 3.0), "total": _blank((rows, width), dtype)}
    if case["out"][0] == "e":
        s["scales"] = _blank((rows, _groups(case)), "f32")
    return s


def _prepare_norm_back(case, g):
    rows, width, dtype = case["rows"], case["width"], case["dtype"]
    x = _normal(g, rows, width, dtype, 2.0)
    s = {"case": case, "x": x, "grad_out": _normal(g, rows, width, dtype, 0.01),
         "weight": (1 + 0.2 * torch.randn(width, generator=g, device="cuda")).to(_DTYPE[case["weight"]]),
         "rstd": torch.cat([torch.rsqrt(p.float().square().mean(-1) + _EPS) for p in x.split(max(1, (1 << 25) // width))]),
         "grad_x": _blank((rows, width), dtype), "grad_weight": _blank(width, case["weight"])}
    if case["residual"]:
        s["grad_total"] = _normal(g, rows, width, dtype, 0.01)
    return s


def _tokens(case, g):
    """Tokens as text has them: few are frequent, most are rare."""
    v = case["vocab"]
    rank = torch.exp(torch.rand(case["tokens"], generator=g, device="cuda", dtype=torch.float64) * math.log(v + 1)) - 1
    t = (rank.long().clamp(0, v - 1) * 7919 + 13) % v
    if case["ignored"]:
        t.masked_fill_(torch.rand(t.shape, generator=g, device="cuda") < 0.1, -100)
    return t


def _prepare_embed(case, g):
    return {"case": case, "tokens": _tokens(case, g), "weight": _normal(g, case["vocab"], case["width"], case["dtype"], 0.02),
            "out": _blank((case["tokens"], case["width"]), case["to"])}


def _prepare_embed_back(case, g):
    shape = (case["vocab"], case["width"])
    s = {"case": case, "tokens": _tokens(case, g),
         "grad_out": _normal(g, case["tokens"], case["width"], case["dtype"], 0.01), "grad_weight": _blank(shape, case["to"])}
    if case["add"]:  # what the same table's other use, as the head, already gave
        s["add"] = _normal(g, *shape, case["to"], 0.01)
    return s


def _lse(logits, scale):
    return torch.stack([torch.logsumexp(x.double() * scale, -1).float() for x in logits]) if logits.shape[1] else \
        torch.zeros(logits.shape[:2], device="cuda")


def _prepare_verify(case, g):
    b, k, v, dtype, scale = case["batch"], case["drafts"], case["vocab"], _DTYPE[case["dtype"]], case["scale"]
    logits = torch.empty(b, k + 1, v, dtype=dtype, device="cuda")
    guess = torch.empty(b, k, v, dtype=dtype, device="cuda")
    drafts = torch.empty(b, k, dtype=torch.int64, device="cuda")
    for i in range(b):
        x = torch.randn(k + 1, v, generator=g, device="cuda").mul_(2.5)
        y = x[:k] + 0.7 * torch.randn(k, v, generator=g, device="cuda")
        if case["masked"]:
            out = torch.rand(1, v, generator=g, device="cuda") < 0.3
            out[0, v // 2] = False
            x.masked_fill_(out, -math.inf)
            y.masked_fill_(out, -math.inf)
        logits[i], guess[i] = x.to(dtype), y.to(dtype)
        race = torch.empty(k, v, device="cuda").exponential_(generator=g)
        drafts[i] = (torch.softmax(guess[i].float() * scale, -1) / race).argmax(-1)
    if case["ragged"] and k:  # some sequences have fewer drafts
        length = torch.randint(0, k + 1, (b, 1), generator=g, device="cuda")
        drafts.masked_fill_(torch.arange(k, device="cuda")[None] >= length, -1)
    s = {"case": case, "logits": logits, "lse": _lse(logits, scale), "drafts": drafts,
         "uniform": torch.rand(b, k, generator=g, device="cuda"),
         "noise": torch.empty(b, v, device="cuda").exponential_(generator=g).clamp_(min=1e-30),
         "tokens": torch.zeros(b, k + 1, dtype=torch.int64, device="cuda"),
         "accepted": torch.zeros(b, dtype=torch.int64, device="cuda")}
    if case["model"]:
        s |= {"draft_logits": guess, "draft_lse": _lse(guess, scale)}
    return s


# -------------------------------------------------------------------------------------------------- one pass
def run(s):
    if own:
        return _own(s)
    return {"norm": _plain_norm, "norm_back": _plain_norm_back, "embed": _plain_embed, "embed_back": _plain_embed_back,
            "verify": _plain_verify}[s["case"]["op"]](s)


@functools.cache
def _framework():
    from alpaka3_b200 import algo
    return algo


def _own(s):
    algo, case = _framework(), s["case"]
    op = case["op"]
    if op == "norm":
        algo.rms_norm(s["out"], s["x"], s["weight"], residual=s.get("residual"), total=s.get("total"), rstd=s["rstd"],
                      scales=s.get("scales"), group=case["group"] or None, eps=_EPS)
        return {k: s[k] for k in ("out", "total", "rstd", "scales") if k in s}
    if op == "norm_back":
        algo.rms_norm_backward(s["grad_x"], s["grad_out"], s["x"], s["weight"], s["rstd"], grad_weight=s["grad_weight"],
                               grad_total=s.get("grad_total"))
        return {"grad_x": s["grad_x"], "grad_weight": s["grad_weight"]}
    if op == "embed":
        algo.embedding(s["out"], s["weight"], s["tokens"], scale=case["scale"])
        return {"out": s["out"]}
    if op == "embed_back":
        algo.embedding_backward(s["grad_weight"], s["grad_out"], s["tokens"], scale=case["scale"], add=s.get("add"))
        return {"grad_weight": s["grad_weight"]}
    algo.verify_drafts(s["tokens"], s["accepted"], s["drafts"], s["logits"], s["lse"], s["uniform"], s["noise"],
                       draft_logits=s.get("draft_logits"), draft_lse=s.get("draft_lse"), scale=case["scale"])
    return {"tokens": s["tokens"], "accepted": s["accepted"]}


def _plain_norm(s):
    case = s["case"]
    h = s["x"].float()
    out = {}
    if case["residual"]:
        out["total"] = (h + s["residual"].float()).to(_DTYPE[case["dtype"]])
        h = out["total"].float()
    out["rstd"] = torch.rsqrt(h.square().mean(-1) + _EPS)
    y = h * out["rstd"][:, None] * s["weight"].float()
    if case["out"][0] != "e":
        return out | {"out": y.to(_DTYPE[case["out"]])}
    size = case["group"] or case["width"]
    pad = -case["width"] % size
    parts = torch.nn.functional.pad(y, (0, pad)).view(case["rows"], -1, size)
    out["scales"] = parts.abs().amax(-1) / _LARGEST[case["out"]]
    inverse = torch.where(out["scales"] > 0, 1 / out["scales"], torch.zeros_like(out["scales"]))
    q = (parts * inverse[..., None]).view(case["rows"], -1)[:, :case["width"]]
    return out | {"out": q.clamp(-_LARGEST[case["out"]], _LARGEST[case["out"]]).to(_DTYPE[case["out"]])}


def _plain_norm_back(s):
    hat = s["x"].float() * s["rstd"][:, None]
    g = s["grad_out"].float()
    part = g * s["weight"].float()
    d = s["rstd"][:, None] * (part - hat * (part * hat).mean(-1, keepdim=True))
    if "grad_total" in s:
        d = d + s["grad_total"].float()
    return {"grad_x": d.to(s["x"].dtype), "grad_weight": (g * hat).sum(0).to(s["weight"].dtype)}


def _plain_embed(s):
    t, case = s["tokens"], s["case"]
    known = (t >= 0) & (t < case["vocab"])
    rows = s["weight"][torch.where(known, t, torch.zeros_like(t))].float()
    if case["scale"] != 1.0:
        rows = rows * case["scale"]
    return {"out": torch.where(known[:, None], rows, torch.zeros_like(rows)).to(_DTYPE[case["to"]])}


def _plain_embed_back(s):
    t, case = s["tokens"], s["case"]
    known = (t >= 0) & (t < case["vocab"])
    d = torch.zeros(case["vocab"] + 1, case["width"], device="cuda")  # the last row takes what has no token
    d.index_add_(0, torch.where(known, t, torch.full_like(t, case["vocab"])), s["grad_out"].float())
    d = d[:-1]
    if case["scale"] != 1.0:
        d = d * case["scale"]
    if "add" in s:
        d = d + s["add"].float()
    return {"grad_weight": d.to(_DTYPE[case["to"]])}


def _plain_verify(s):
    case = s["case"]
    b, k, v, scale = case["batch"], case["drafts"], case["vocab"], case["scale"]
    t = s["drafts"]
    known = (t >= 0) & (t < v)
    at = torch.where(known, t, torch.zeros_like(t))
    # in 64 bits: both the comparison and the largest quotient may be close
    p = torch.exp(s["logits"][:, :k].gather(-1, at[..., None])[..., 0].double() * scale - s["lse"][:, :k].double())
    q = torch.ones_like(p)
    if case["model"]:
        q = torch.exp(s["draft_logits"].gather(-1, at[..., None])[..., 0].double() * scale - s["draft_lse"].double())
    stands = (known & (s["uniform"].double() * q < p)).long().cumprod(-1)
    count = stands.sum(-1)
    each = torch.arange(b, device="cuda")
    row = torch.exp(s["logits"][each, count].double() * scale - s["lse"][each, count].double()[:, None])
    rest = row
    if k:
        here = count.clamp(max=k - 1)
        refused = (count < k) & known[each, here]
        if case["model"]:
            taken = torch.exp(s["draft_logits"][each, here].double() * scale - s["draft_lse"][each, here].double()[:, None])
        else:
            taken = torch.zeros_like(row)
            taken[each, at[each, here]] = 1.0
        rest = row - torch.where(refused[:, None], taken, torch.zeros_like(taken))
        rest = torch.where((rest > 0).any(-1, keepdim=True), rest, row)
    score = torch.where(rest > 0, rest / s["noise"].double(), torch.zeros_like(rest))
    drawn = torch.where(score.amax(-1) > 0, score.argmax(-1), torch.full_like(count, -1))
    place = torch.arange(k + 1, device="cuda")[None]
    padded = torch.nn.functional.pad(t, (0, 1), value=-1)
    tokens = torch.where(place < count[:, None], padded, torch.where(place == count[:, None], drawn[:, None], -1))
    return {"tokens": tokens, "accepted": count}


# ---------------------------------------------------------------------------------------------- what it costs
def work(case):
    """Every input read once and every output written once; the operations on each element counted by hand."""
    op = case["op"]
    if op == "norm":
        n, size = case["rows"] * case["width"], _SIZE[case["dtype"]]
        scales = case["rows"] * _groups(case) * 4 if case["out"][0] == "e" else 0
        return {"bytes": n * (size * (3 if case["residual"] else 1) + _SIZE[case["out"]]) + scales + 4 * case["rows"]
                + case["width"] * _SIZE[case["weight"]], "flops": 5 * n}
    if op == "norm_back":
        n, size = case["rows"] * case["width"], _SIZE[case["dtype"]]
        return {"bytes": n * size * (4 if case["residual"] else 3) + 4 * case["rows"]
                + 2 * case["width"] * _SIZE[case["weight"]], "flops": 9 * n}
    if op == "embed":
        # of the table at least one row; how many more are named depends on the tokens
        n = case["tokens"] * case["width"]
        return {"bytes": n * _SIZE[case["to"]] + case["width"] * _SIZE[case["dtype"]] + 8 * case["tokens"], "flops": n}
    if op == "embed_back":
        n, size = case["vocab"] * case["width"], _SIZE[case["to"]]
        share = 0.9 if case["ignored"] else 1.0
        return {"bytes": n * size * (2 if case["add"] else 1) + 8 * case["tokens"]
                + case["tokens"] * case["width"] * _SIZE[case["dtype"]] * share, "flops": case["tokens"] * case["width"]}
    # one row of the target and of the noise for every sequence; of the draft only where a token is refused (not counted)
    n = case["batch"] * case["vocab"]
    return {"bytes": n * (_SIZE[case["dtype"]] + 4) + case["batch"] * (case["drafts"] + 1) * 32, "flops": 5 * n}


# ------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "norm_back": _exact_norm_back, "embed": _exact_embed, "embed_back": _exact_embed_back,
            "verify": _exact_verify}[case["op"]](s)


def _rounded(x, dtype):
    """x in 64 bits, rounded once to `dtype`: what is stored of it."""
    return x.to(_DTYPE[dtype]).double()


def _exact_norm(s):
    case = s["case"]
    h = s["x"].double()
    out = {}
    if case["residual"]:  # the norm is that of the sum as it is stored
        out["total"] = h = _rounded(h + s["residual"].double(), case["dtype"])
    mean = torch.linalg.vector_norm(h, dim=-1) ** 2 / case["width"]
    out["rstd"] = 1.0 / torch.sqrt(mean + _EPS)
    y = h / torch.sqrt(mean + _EPS)[:, None] * s["weight"].double()[None]
    if case["out"][0] != "e":
        return out | {"out": y}
    size, parts, scales = case["group"] or case["width"], [], []
    for part in y.split(size, -1):
        scale = part.abs().max(-1, keepdim=True)[0] / _LARGEST[case["out"]]
        parts.append(torch.where(scale > 0, part / scale, torch.zeros_like(part)))
        scales.append(scale)
    return out | {"out": torch.cat(parts, -1), "scales": torch.cat(scales, -1)}


def _exact_norm_back(s):
    n = s["case"]["width"]
    h, g, w, r = s["x"].double(), s["grad_out"].double(), s["weight"].double(), s["rstd"].double()[:, None]
    # d/dh_j of sum_i g_i w_i h_i r with r = (mean h^2 + eps)^(-1/2), dr/dh_j = -r^3 h_j / n
    dot = torch.einsum("rn,rn->r", g * w, h)[:, None]
    d = g * w * r - r ** 3 * h * dot / n
    if "grad_total" in s:
        d += s["grad_total"].double()
    return {"grad_x": d, "grad_weight": torch.einsum("rn,rn->n", g, h * r)}


def _exact_embed(s):
    t, v = s["tokens"], s["case"]["vocab"]
    out = torch.zeros(len(t), s["case"]["width"], dtype=torch.float64, device="cuda")
    here = ((t >= 0) & (t < v)).nonzero()[:, 0]
    out[here] = s["weight"].index_select(0, t[here]).double() * s["case"]["scale"]
    return {"out": out}


def _exact_embed_back(s):
    t, case = s["tokens"], s["case"]
    here = ((t >= 0) & (t < case["vocab"])).nonzero()[:, 0]
    d = torch.zeros(case["vocab"], case["width"], dtype=torch.float64, device="cuda")
    d.index_put_((t[here],), s["grad_out"][here].double() * case["scale"], accumulate=True)
    if "add" in s:
        d += s["add"].double()
    return {"grad_weight": d}


def _exact_verify(s):
    case = s["case"]
    k, v, scale = case["drafts"], case["vocab"], case["scale"]
    tokens = torch.full((case["batch"], k + 1), -1, dtype=torch.int64, device="cuda")
    counts = torch.zeros(case["batch"], dtype=torch.int64, device="cuda")
    drafts, uniform = s["drafts"].tolist(), s["uniform"].double().tolist()
    for b, row in enumerate(drafts):
        n, rest = 0, None
        while rest is None:
            left = (s["logits"][b, n].double() * scale - s["lse"][b, n].double()).exp()
            if n == k or not 0 <= row[n] < v:
                rest = left
                break
            if case["model"]:
                drafted = (s["draft_logits"][b, n].double() * scale - s["draft_lse"][b, n].double()).exp()
            else:
                drafted = torch.nn.functional.one_hot(torch.tensor(row[n], device="cuda"), v).double()
            ratio = left[row[n]] / drafted[row[n]]
            if uniform[b][n] < ratio.item():
                tokens[b, n] = row[n]
                n += 1
            else:
                rest = torch.clamp(left - drafted, min=0)
                rest = left if rest.max() == 0 else rest
        counts[b] = n
        if rest.nan_to_num(nan=0.0).max() > 0:
            # the first of exponential clocks with these rates
            tokens[b, n] = torch.where(rest > 0, s["noise"][b].double() / rest, math.inf).argmin()
    return {"tokens": tokens, "accepted": counts}
