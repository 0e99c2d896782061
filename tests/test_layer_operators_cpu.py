"""CPU: the checks of arguments of the norm of rows, the embedding and the verification of drafts (they run before any CUDA
call), the layout of their argument structures, and which arrays count as apart."""
import ctypes
import math
import os
import random
import subprocess

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
A, B, C, D = 0x10000000, 0x20000000, 0x30000000, 0x40000000  # stand for device addresses: nothing below may use them
W, R, S, T = 0x50000000, 0x60000000, 0x70000000, 0x80000000


@pytest.fixture(scope="module")
def L():
    if torch.cuda.is_available():
        pytest.skip("the addresses in these calls are made up: only where no GPU could use one")
    from alpaka3_b200 import capi
    return capi.lib()


def rows(at, outer=0, inner=64):
    return [at, outer, inner]


def norm(L, **kw):
    from alpaka3_b200 import capi
    a = dict(outer=1, inner=4, n=64, x=rows(A), residual=rows(0), total=rows(0), out=rows(B), weight=W, rstd=R, scales=0,
             eps=1e-6, dtype=capi.BF16, out_dtype=capi.BF16, weight_dtype=capi.F32, group=0)
    assert set(kw) <= set(a), kw
    a.update(kw)
    flat = [v for k in a.values() for v in (k if isinstance(k, list) else [k])]
    return L.a3b_rms_norm(None, capi.RMS_NORM_ARGS.pack(*flat))


def norm_backward(L, **kw):
    from alpaka3_b200 import capi
    a = dict(outer=1, inner=4, n=64, grad_out=rows(A), x=rows(B), grad_total=rows(0), grad_x=rows(C), weight=W, rstd=R,
             grad_weight=S, workspace=T, workspace_bytes=1 << 20, dtype=capi.BF16, weight_dtype=capi.F32,
             grad_weight_dtype=capi.F32, reserved=0)
    assert set(kw) <= set(a), kw
    a.update(kw)
    flat = [v for k in a.values() for v in (k if isinstance(k, list) else [k])]
    return L.a3b_rms_norm_backward(None, capi.RMS_NORM_BACKWARD_ARGS.pack(*flat))


def embed(L, **kw):
    from alpaka3_b200 import capi
    a = dict(outer=1, inner=4, n=64, vocab=100, first=0, table=A, stride=64, tokens=T, out=rows(B), scale=1.0,
             table_dtype=capi.BF16, index=capi.I64, out_dtype=capi.BF16, reserved=0)
    assert set(kw) <= set(a), kw
    a.update(kw)
    flat = [v for k in a.values() for v in (k if isinstance(k, list) else [k])]
    return L.a3b_embedding(None, capi.EMBEDDING_ARGS.pack(*flat))


def embed_backward(L, **kw):
    from alpaka3_b200 import capi
    a = dict(outer=1, inner=4, n=64, vocab=100, first=0, grad_out=rows(A), tokens=T, add=0, add_stride=0, grad_table=B,
             stride=64, workspace=W, workspace_bytes=1 << 20, scale=1.0, grad_dtype=capi.BF16, index=capi.I64,
             table_dtype=capi.BF16, reserved=0)
    assert set(kw) <= set(a), kw
    a.update(kw)
    flat = [v for k in a.values() for v in (k if isinstance(k, list) else [k])]
    return L.a3b_embedding_backward(None, capi.EMBEDDING_BACKWARD_ARGS.pack(*flat))


def verify(L, **kw):
    from alpaka3_b200 import capi
    a = dict(batch=2, length=3, vocab=64, logits=rows(A, 256, 64), draft=rows(B, 192, 64), lse=C, draft_lse=D, scale=1.0,
             draft_scale=1.0, drafts=W, top=0, uniform=R, noise=S, noise_stride=64, tokens=T, accepted=T + 0x1000,
             dtype=capi.BF16, index=capi.I64)
    assert set(kw) <= set(a), kw
    a.update(kw)
    flat = [v for k in a.values() for v in (k if isinstance(k, list) else [k])]
    return L.a3b_verify_drafts(None, capi.VERIFY_DRAFTS_ARGS.pack(*flat))


def refused(rc, code=None):
    from alpaka3_b200 import capi
    assert rc == (capi.ERR_INVALID if code is None else code), (rc, capi.last_error())
    assert capi.last_error()


def past_the_checks(rc):
    """what is sound ends at the lack of a GPU"""
    from alpaka3_b200 import capi
    assert rc in (capi.ERR_CUDA, capi.ERR_UNSUPPORTED), (rc, capi.last_error())


def test_structures_match_the_header(tmp_path):
    """Sizes, and the offsets of the last fields, as a C compiler lays the structures out."""
    from alpaka3_b200 import capi
    pairs = {"a3b_rms_norm_args": (capi.RMS_NORM_ARGS, "group"),
             "a3b_rms_norm_backward_args": (capi.RMS_NORM_BACKWARD_ARGS, "reserved"),
             "a3b_embedding_args": (capi.EMBEDDING_ARGS, "reserved"),
             "a3b_embedding_backward_args": (capi.EMBEDDING_BACKWARD_ARGS, "reserved"),
             "a3b_verify_drafts_args": (capi.VERIFY_DRAFTS_ARGS, "index_dtype")}
    body = "".join(f'printf("%zu %zu\\n", sizeof({k}), offsetof({k}, {last}));' for k, (_, last) in pairs.items())
    source = tmp_path / "sizes.c"
    source.write_text(f"#include <stdio.h>\n#include <stddef.h>\n#include <alpaka3_b200.h>\nint main(void) {{ {body} return 0; }}\n")
    exe = tmp_path / "sizes"
    subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), str(source), "-o", str(exe)])
    lines = subprocess.check_output([str(exe)], text=True).split("\n")
    for (name, (packed, _)), line in zip(pairs.items(), lines):
        size, last = map(int, line.split())
        assert packed.size == size == last + 4, name


def test_norm_refusals(L):
    from alpaka3_b200 import capi
    F, H, E4 = capi.F32, capi.F16, capi.E4M3
    refused(L.a3b_rms_norm(None, None))
    for kw in (dict(dtype=capi.F64), dict(dtype=99), dict(n=0), dict(eps=-1.0), dict(eps=math.nan), dict(eps=math.inf),
               dict(x=rows(0)), dict(out=rows(0)), dict(total=rows(C)), dict(out_dtype=F), dict(out_dtype=capi.I32),
               dict(weight_dtype=H), dict(group=64), dict(scales=S), dict(out_dtype=E4), dict(out_dtype=E4, scales=S, group=16),
               dict(out_dtype=E4, scales=S, group=48), dict(x=rows(A + 1)), dict(residual=rows(A + 1)), dict(out=rows(B + 1)),
               dict(weight=W + 2), dict(rstd=R + 2), dict(out_dtype=E4, scales=S + 2), dict(inner=1 << 62, outer=8),
               dict(out=rows(B, 0, 63)), dict(out=rows(B, 0, 0)), dict(out=rows(A + 2)), dict(out=rows(A, 0, 65)),
               dict(out=rows(A + 128 * 3)), dict(residual=rows(C), total=rows(B)), dict(residual=rows(C), total=rows(C + 2)),
               dict(out=rows(W)), dict(out=rows(R - 64)), dict(rstd=A),
               dict(out_dtype=E4, out=rows(A), scales=S), dict(out_dtype=E4, scales=R), dict(out_dtype=E4, scales=B),
               dict(outer=3, out=rows(B, 64, 64)), dict(outer=3, inner=2, out=rows(B, 100, 64)), dict(rstd=B + 16)):
        refused(norm(L, **kw))
    for kw in (dict(n=1 << 31), dict(inner=1 << 31), dict(inner=1 << 16, outer=1 << 16)):
        refused(norm(L, **kw), capi.ERR_TOO_LARGE)
    assert norm(L, inner=0, x=rows(0), out=rows(0)) == capi.OK
    for kw in ({}, dict(out=rows(A)), dict(residual=rows(C), total=rows(C)), dict(residual=rows(C), total=rows(A)),
               dict(residual=rows(C), total=rows(D), out=rows(C)), dict(x=rows(A, 0, 192), out=rows(A + 128, 0, 192)),
               dict(weight=0, rstd=0), dict(out_dtype=E4, scales=S, group=32), dict(residual=rows(A)),
               dict(outer=3, inner=2, out=rows(B, 64, 200)), dict(x=rows(A, 0, 0))):
        past_the_checks(norm(L, **kw))


def test_norm_backward_refusals(L):
    from alpaka3_b200 import capi
    F, H = capi.F32, capi.F16
    refused(L.a3b_rms_norm_backward(None, None))
    for kw in (dict(dtype=capi.F64), dict(n=0), dict(grad_out=rows(0)), dict(x=rows(0)), dict(grad_x=rows(0)), dict(rstd=0),
               dict(weight_dtype=H), dict(grad_weight_dtype=H), dict(grad_weight_dtype=capi.BF16), dict(grad_x=rows(C + 1)),
               dict(grad_weight=S + 2), dict(rstd=R + 1), dict(grad_x=rows(C, 0, 63)), dict(grad_x=rows(A + 2)),
               dict(grad_total=rows(C + 64)), dict(grad_weight=A), dict(grad_weight=W), dict(grad_weight=C),
               dict(workspace=C), dict(workspace=A), dict(workspace=S), dict(grad_x=rows(W)), dict(grad_x=rows(R)),
               dict(grad_x=rows(B, 0, 65))):
        refused(norm_backward(L, **kw))
    for kw in (dict(n=1 << 31), dict(inner=1 << 31)):
        refused(norm_backward(L, **kw), capi.ERR_TOO_LARGE)
    for kw in ({}, dict(grad_x=rows(A)), dict(grad_x=rows(B)), dict(grad_total=rows(D), grad_x=rows(D)),
               dict(grad_weight=0, workspace=0, workspace_bytes=0), dict(weight=0, grad_weight_dtype=F)):
        past_the_checks(norm_backward(L, **kw))
    assert norm_backward(L, inner=0, grad_weight=0) == capi.OK


def test_embedding_refusals(L):
    from alpaka3_b200 import capi
    F, H = capi.F32, capi.F16
    refused(L.a3b_embedding(None, None))
    refused(L.a3b_embedding_backward(None, None))
    for kw in (dict(table_dtype=capi.I32), dict(out_dtype=capi.F64), dict(out_dtype=H), dict(index=capi.U32), dict(n=0),
               dict(scale=math.inf), dict(scale=math.nan), dict(scale=1e39), dict(table=0), dict(tokens=0), dict(out=rows(0)),
               dict(table=A + 1), dict(out=rows(B + 1)), dict(tokens=T + 4), dict(out=rows(B, 0, 63)), dict(out=rows(A)),
               dict(out=rows(A + 64 * 2 * 99)), dict(out=rows(T)), dict(outer=1 << 62, inner=8)):
        refused(embed(L, **kw))
    for kw in (dict(vocab=1 << 31), dict(inner=1 << 31), dict(n=1 << 31)):
        refused(embed(L, **kw), capi.ERR_TOO_LARGE)
        refused(embed_backward(L, **kw), capi.ERR_TOO_LARGE)
    assert embed(L, inner=0, tokens=0, out=rows(0)) == capi.OK
    for kw in ({}, dict(table_dtype=F), dict(out_dtype=F), dict(vocab=0, table=0), dict(stride=0),
               dict(index=capi.I32, tokens=T + 4), dict(table=A, stride=128, out=rows(A + 128, 0, 128))):
        past_the_checks(embed(L, **kw))
    for kw in (dict(table_dtype=capi.I32), dict(grad_dtype=H), dict(index=capi.U32), dict(n=0), dict(scale=math.inf),
               dict(grad_out=rows(0)), dict(tokens=0), dict(grad_table=0), dict(grad_table=B + 1), dict(add=C + 1),
               dict(stride=63), dict(stride=0), dict(add=B, add_stride=65), dict(add=B + 128, add_stride=64),
               dict(grad_table=A), dict(grad_table=T), dict(grad_table=W), dict(workspace=A), dict(workspace=T),
               dict(add=W, add_stride=64)):
        refused(embed_backward(L, **kw))
    assert embed_backward(L, vocab=0) == capi.OK
    for kw in ({}, dict(add=C, add_stride=64), dict(add=B, add_stride=64), dict(grad_out=rows(A, 0, 0)),
               dict(inner=0, grad_out=rows(0), tokens=0, workspace=0, workspace_bytes=0)):
        past_the_checks(embed_backward(L, **kw))


def test_verify_refusals(L):
    from alpaka3_b200 import capi
    refused(L.a3b_verify_drafts(None, None))
    for kw in (dict(dtype=capi.F64), dict(index=capi.U32), dict(vocab=0), dict(tokens=0), dict(accepted=0), dict(drafts=0),
               dict(logits=rows(0)), dict(lse=0), dict(uniform=0), dict(noise=0), dict(draft_lse=0), dict(scale=0.0),
               dict(scale=math.nan), dict(scale=1e9), dict(draft_scale=-1.0), dict(logits=rows(A + 1, 256, 64)),
               dict(draft=rows(B + 1, 192, 64)), dict(lse=C + 2), dict(uniform=R + 1), dict(noise=S + 2), dict(drafts=W + 4),
               dict(tokens=T + 4), dict(accepted=T + 8), dict(tokens=W), dict(tokens=A + 64), dict(accepted=S + 8),
               dict(accepted=C), dict(top=T), dict(logits=rows(0), draft=rows(0), top=0)):
        refused(verify(L, **kw))
    for kw in (dict(vocab=(1 << 31) - 64), dict(batch=1 << 31), dict(length=1 << 31), dict(batch=1 << 20, length=1 << 12)):
        refused(verify(L, **kw), capi.ERR_TOO_LARGE)
    refused(verify(L, batch=1 << 62, length=8))
    assert verify(L, batch=0, tokens=0, drafts=0) == capi.OK
    for kw in ({}, dict(draft=rows(0)), dict(length=0, drafts=0, uniform=0), dict(top=D + 0x1000), dict(logits=rows(A, 0, 0)),
               dict(logits=rows(0), draft=rows(0), lse=0, uniform=0, noise=0, top=D), dict(noise_stride=0)):
        past_the_checks(verify(L, **kw))


def test_apart_against_all_bytes(L):
    """Random small layouts of two arrays of rows in one buffer: never accepted where they share a byte and are not the same
    rows, and always where one ends before the other begins or both step alike and lie beside one another."""
    from alpaka3_b200 import capi
    r = random.Random(7)
    seen = {True: 0, False: 0, "beside": 0}
    for _ in range(4000):
        outer, inner, n = r.randint(1, 3), r.randint(1, 3), r.randint(1, 4)
        unit = r.choice([n, 2 * n, 2 * n + 1, 10])
        si = max(unit, n)
        so = r.choice([si * inner, si * (inner + 1), si * inner + 3])
        other = r.choice([(so, si), (so, si), (si * inner, si), (r.randint(0, 12), r.randint(0, 12))])
        off = r.randint(-30, 30)
        xa, oa = A + 4 * off, A
        cells = lambda base, s: {base + 4 * (o * s[0] + i * s[1] + e)  # noqa: E731
                                 for o in range(outer) for i in range(inner) for e in range(n)}
        mine, theirs = cells(oa, (so, si)), cells(xa, other)
        same = off == 0 and (outer == 1 or other[0] == so) and (inner == 1 or other[1] == si)
        rc = norm(L, outer=outer, inner=inner, n=n, x=rows(xa, *other), out=rows(oa, so, si), dtype=capi.F32,
                  out_dtype=capi.F32)
        ok = rc in (capi.ERR_CUDA, capi.ERR_UNSUPPORTED)
        assert ok or "overlap" in capi.last_error(), capi.last_error()
        touching = bool(mine & theirs)
        if touching and not same:
            assert not ok, (outer, inner, n, so, si, other, off)
        if same or max(theirs) < min(mine) or max(mine) < min(theirs):
            assert ok, (outer, inner, n, so, si, other, off)
        if other == (so, si) and so % si == 0 and not touching and abs(off) % si >= n and si - abs(off) % si >= n:
            assert ok
            seen["beside"] += 1
        seen[touching] += 1
    assert min(seen.values()) > 200, seen


def test_python_refusals():
    """Before anything reaches the library: CPU tensors, wrong types and shapes."""
    from alpaka3_b200 import algo
    x = torch.zeros(2, 8)
    i = torch.zeros(2, dtype=torch.int64)
    for call in (lambda: algo.rms_norm(x, x), lambda: algo.rms_norm_backward(x, x, x, None, torch.zeros(2)),
                 lambda: algo.embedding(x, x, i), lambda: algo.embedding_backward(x, x, i),
                 lambda: algo.verify_drafts(torch.zeros(2, 3, dtype=torch.int64), i, torch.zeros(2, 2, dtype=torch.int64),
                                            top_index=torch.zeros(2, 3, dtype=torch.int64))):
        with pytest.raises(ValueError, match="CUDA"):
            call()
    for call in (lambda: algo.rms_norm(x, x.double()), lambda: algo.embedding(x, x.long(), i),
                 lambda: algo.verify_drafts(i, i, x)):
        with pytest.raises(TypeError):
            call()


def test_joint_rows():
    from alpaka3_b200 import algo
    x = torch.empty(4, 6, 10)
    wide = torch.empty(4, 6, 30)
    assert algo._joint_rows((x, "x"), (None, "r"), (wide[..., 10:20], "o")) == (1, 24, 10, [(0, 10), (0, 0), (0, 30)])
    back = torch.empty(6, 4, 10).transpose(0, 1)
    assert algo._joint_rows((x, "x"), (back, "o")) == (4, 6, 10, [(60, 10), (10, 40)])
    assert algo._joint_rows((x[:0], "x"), (wide[:0, :, :10], "o")) == (0, 0, 10, [(0, 0)] * 2)
    assert algo._joint_rows((x[0, 0], "x"), (x[1, 2], "o")) == (1, 1, 10, [(0, 0)] * 2)
    assert algo._joint_rows((torch.empty(3, 1, 10), "x"), (torch.empty(1, 3, 10).transpose(0, 1), "o"))[:3] == (1, 3, 10)
    for bad in (x.transpose(1, 2), x[..., ::2], torch.empty(())):
        with pytest.raises(ValueError):
            algo._joint_rows((bad, "x"))
    with pytest.raises(ValueError, match="two strides"):
        algo._joint_rows((torch.empty(3, 4, 5, 8)[:, :3, :4], "x"))
