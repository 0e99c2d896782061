"""Python mirror of alpaka3's onHost algorithm entry points for the primitive path, over the C ABI.

Device buffers are torch CUDA tensors (plumbing only: allocation, streams); every computation is one call into
``libalpaka3_b200.so``. Names and argument meaning follow include/alpaka/onHost/algo/*.hpp:

* :func:`transform`           onHost::transform            (algo/transform.hpp:50-88)
* :func:`transform_reduce`    onHost::transformReduce      (algo/transformReduce.hpp:59-114)
* :func:`reduce`              onHost::reduce               (algo/reduce.hpp:28-79)
* :func:`inclusive_scan` / :func:`exclusive_scan` (+ ``in_place``), :func:`get_scan_buffer_size`
                              onHost::*Scan[InPlace], getScanBufferSize (algo/scan.hpp:26-218)
* :func:`fill`, :func:`iota`  onHost::fill (Queue.hpp:346), onHost::iota (algo/iota.hpp:29-85)
* :func:`babelstream`         the BabelStream kernels (benchmark/babelstream/src/babelStreamMainTest.cpp:78-141)
* :func:`nbody_step`, :func:`nbody_update_velocities`, :func:`nbody_update_positions`  (example/nBody)
* :func:`heat_step`, :func:`heat_init`  (example/heatEquation2D)

Reductions of a language model's training and decoding steps, which alpaka3 does not have:

* :func:`token_logprobs`, :func:`token_logprobs_backward`  per row of logits: the log probability of its token, entropy,
                              log-sum-exp and most likely alternatives, and their gradient
* :class:`TensorList`, :func:`grad_norm`, :func:`clip_grads`, :func:`clip_grad_norm`  norm and clipping of a list of
                              gradients
* :func:`rms_norm`, :func:`rms_norm_backward`  root-mean-square norm of rows with the residual's addition, also with an
                              output in 8 bits, and its gradient
* :func:`embedding`, :func:`embedding_backward`  rows of a table by tokens, and the table's gradient
* :func:`verify_drafts`       drafted tokens against the target's probabilities, from given random numbers

Errors raise :class:`alpaka3_b200.capi.A3BError` (the reference throws std::runtime_error on backend errors).
"""
import ctypes
import functools

import numpy as np
import torch

from . import capi

_DT = {torch.int32: capi.I32, torch.uint32: capi.U32, torch.int64: capi.I64, torch.uint64: capi.U64,
       torch.float32: capi.F32, torch.float64: capi.F64}
_NP = {capi.I32: np.int32, capi.U32: np.uint32, capi.I64: np.int64, capi.U64: np.uint64, capi.F32: np.float32,
       capi.F64: np.float64}
REDUCE = {"plus": capi.PLUS, "min": capi.MIN, "max": capi.MAX}
XFORM = {"identity": capi.IDENTITY, "square": capi.SQUARE, "product": capi.PRODUCT}
STREAM = {"init": capi.INIT, "copy": capi.COPY, "mul": capi.MUL, "add": capi.ADD, "triad": capi.TRIAD,
          "nstream": capi.NSTREAM}
NORM = {"l2": capi.NORM_L2, "l1": capi.NORM_L1, "max": capi.NORM_MAX}
_LOGITS_DT = {torch.float32: capi.F32, torch.float16: capi.F16, torch.bfloat16: capi.BF16}
_GRAD_DT = {**_LOGITS_DT, torch.float64: capi.F64}
_INDEX_DT = {torch.int64: capi.I64, torch.int32: capi.I32}
_NORM_OUT_DT = {**_LOGITS_DT, torch.float8_e4m3fn: capi.E4M3, torch.float8_e5m2: capi.E5M2}
MAP = {"copy": capi.MAP_COPY, "scale": capi.MAP_SCALE, "add": capi.MAP_ADD, "mul": capi.MAP_MUL,
       "axpy": capi.MAP_AXPY, "square": capi.MAP_SQUARE}


def dtype_code(t):
    try:
        return _DT[t.dtype]
    except KeyError:
        raise TypeError(f"unsupported dtype {t.dtype}") from None


def stream_handle(stream=None):
    s = stream if stream is not None else torch.cuda.current_stream()
    return ctypes.c_void_p(s.cuda_stream)


def _ptr(t):
    if t is None:
        return None
    if not t.is_cuda:
        raise ValueError("expected a CUDA tensor")
    if not t.is_contiguous():
        raise ValueError("expected a contiguous tensor")
    return ctypes.c_void_p(t.data_ptr())


def _host_scalar(value, code):
    arr = np.array([value], dtype=_NP[code])
    return arr, arr.ctypes.data_as(ctypes.c_void_p)


def _neutral(op, code):
    dt = np.dtype(_NP[code])
    if op == "plus":
        return 0
    if dt.kind == "f":
        return np.inf if op == "min" else -np.inf
    info = np.iinfo(dt)
    return info.max if op == "min" else info.min


# ------------------------------------------------------------------------------------------------ element-wise
def babelstream(kind, a, b, c, scalar=0.4, init=(0.1, 0.2, 0.0), stream=None):
    code = dtype_code(a)
    ini = (ctypes.c_double * 3)(*init)
    capi.call("a3b_babelstream", stream_handle(stream), STREAM[kind], code, _ptr(a), _ptr(b), _ptr(c), a.numel(),
              float(scalar), ini)


def transform(kind, out, in0, in1=None, alpha=1.0, stream=None):
    capi.call("a3b_transform", stream_handle(stream), MAP[kind], dtype_code(out), _ptr(out), _ptr(in0), _ptr(in1),
              out.numel(), float(alpha))
    return out


def fill(out, value, stream=None):
    code = dtype_code(out)
    keep, p = _host_scalar(value, code)
    capi.call("a3b_fill", stream_handle(stream), code, _ptr(out), out.numel(), p)
    return out


def iota(out, start=0, stream=None):
    code = dtype_code(out)
    keep, p = _host_scalar(start, code)
    capi.call("a3b_iota", stream_handle(stream), code, _ptr(out), out.numel(), p)
    return out


def random_u32(out, seed, start=0, shift=0, stream=None):
    capi.call("a3b_random_u32", stream_handle(stream), _ptr(out), out.numel(), seed, start, shift)
    return out


def random_u64(out, seed, start=0, stream=None):
    capi.call("a3b_random_u64", stream_handle(stream), _ptr(out), out.numel(), seed, start)
    return out


def random_f32(out, seed, lo=-1.0, hi=1.0, start=0, stream=None):
    capi.call("a3b_random_f32", stream_handle(stream), _ptr(out), out.numel(), seed, start, lo, hi)
    return out


# -------------------------------------------------------------------------------------------------- reductions
def set_early_start(enable=True, stream=None):
    """Let the reductions on `stream` start while the previous kernel of the stream still runs (programmatic
    dependent launch; off by default). Enable it only when no kernel on the stream signals its dependents early
    (griddepcontrol.launch_dependents) before writing its output."""
    capi.call("a3b_set_early_start", stream_handle(stream), 1 if enable else 0)


def transform_reduce(neutral, out, reduce_fn, transform_fn, in0, in1=None, stream=None):
    """onHost::transformReduce(queue, neutral, out, reduceFn, transformFn, in0[, in1]); out: 1-element tensor."""
    code = dtype_code(in0)
    if out.dtype != in0.dtype or out.numel() < 1:
        raise ValueError("out must hold one element of the input dtype")
    if neutral is None:
        neutral = _neutral(reduce_fn, code)
    keep, p = _host_scalar(neutral, code)
    capi.call("a3b_transform_reduce", stream_handle(stream), code, REDUCE[reduce_fn], XFORM[transform_fn], _ptr(in0),
              _ptr(in1), in0.numel(), p, _ptr(out))
    return out


def transform_reduce_partial(reduce_fn, transform_fn, in0, in1=None, partial=None, neutral=None, stream=None):
    """Un-rounded 8-byte partial (float64 for float inputs, int64/uint64 for integers) for cross-GPU combination."""
    code = dtype_code(in0)
    if partial is None:
        pdt = torch.float64 if code in (capi.F32, capi.F64) else (torch.int64 if code in (capi.I32, capi.I64)
                                                                   else torch.uint64)
        partial = torch.empty(1, dtype=pdt, device=in0.device)
    if neutral is None:
        neutral = _neutral(reduce_fn, code)
    keep, p = _host_scalar(neutral, code)
    capi.call("a3b_transform_reduce_partial", stream_handle(stream), code, REDUCE[reduce_fn], XFORM[transform_fn],
              _ptr(in0), _ptr(in1), in0.numel(), p, _ptr(partial))
    return partial


def reduce(neutral, out, reduce_fn, data, stream=None):
    """onHost::reduce over a 1-D..N-D tensor; a tensor whose rows (last dim) are strided by a constant pitch is
    passed as a pitched 2-D view without copying."""
    code = dtype_code(data)
    if neutral is None:
        neutral = _neutral(reduce_fn, code)
    keep, p = _host_scalar(neutral, code)
    if data.is_contiguous():
        rows, row_len, pitch = 1, data.numel(), data.numel() * data.element_size()
    else:
        if data.dim() != 2 or data.stride(1) != 1:
            raise ValueError("non-contiguous input must be a 2-D view with unit stride in the last dimension")
        rows, row_len, pitch = data.shape[0], data.shape[1], data.stride(0) * data.element_size()
    capi.call("a3b_reduce_2d", stream_handle(stream), code, REDUCE[reduce_fn], ctypes.c_void_p(data.data_ptr()),
              rows, row_len, pitch, p, _ptr(out))
    return out


# -------------------------------------------------------------------------------------------------------- scan
def get_scan_buffer_size(dtype, n):
    code = _DT[dtype]
    return capi.lib().a3b_scan_buffer_size(code, n)


def _scan(inclusive, out, data, buffer=None, carry=None, stream=None):
    code = dtype_code(data)
    if out.dtype != data.dtype or out.numel() != data.numel():
        raise ValueError("output must match the input's dtype and size")
    bp = _ptr(buffer) if buffer is not None else None
    bb = buffer.numel() * buffer.element_size() if buffer is not None else 0
    capi.call("a3b_scan", stream_handle(stream), code, 1 if inclusive else 0, _ptr(data), _ptr(out), data.numel(),
              _ptr(carry), bp, bb)
    return out


def inclusive_scan(out, data, buffer=None, carry=None, stream=None):
    return _scan(True, out, data, buffer, carry, stream)


def exclusive_scan(out, data, buffer=None, carry=None, stream=None):
    return _scan(False, out, data, buffer, carry, stream)


def inclusive_scan_in_place(data, buffer=None, stream=None):
    return _scan(True, data, data, buffer, None, stream)


def exclusive_scan_in_place(data, buffer=None, stream=None):
    return _scan(False, data, data, buffer, None, stream)


# ------------------------------------------------------------------------------------- token log probabilities
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)  # the address alone, without a Stream object


@functools.cache
def _entry(name):
    return getattr(capi.lib(), name)


@functools.cache
def _one_device():
    return torch.cuda.device_count() == 1


def _call_on(index, stream, name, *args):
    """Entry point `name` on `stream` (default: the current stream of device `index`) with that device current."""
    if stream is None:
        handle = _raw_stream(index) if _raw_stream else torch.cuda.current_stream(index).cuda_stream
    elif stream.device_index != index:
        raise ValueError(f"the stream belongs to device {stream.device_index}, the tensors to device {index}")
    else:
        handle = stream.cuda_stream
    if _one_device() or torch.cuda.current_device() == index:
        rc = _entry(name)(handle, *args)
    else:
        with torch.cuda.device(index):
            rc = _entry(name)(handle, *args)
    if rc:
        capi.check(rc, name)


def _rows(t, name):
    """(outer, inner, outer stride, inner stride) of the rows (last dimension) of t: all other dimensions together must
    step through memory with at most two strides, as those of logits[:, :-1] do."""
    if t.dim() < 1 or (t.shape[-1] > 1 and t.stride(-1) != 1):
        raise ValueError(f"{name}: rows must be contiguous in the last dimension")
    levels = []
    for size, stride in zip(t.shape[:-1], t.stride()[:-1]):
        if size == 1:
            continue
        if levels and levels[-1][1] == size * stride:
            levels[-1] = (levels[-1][0] * size, stride)
        else:
            levels.append((size, stride))
    if t.numel() == 0:
        levels = [(t.numel(), 0)]
    if len(levels) > 2:
        raise ValueError(f"{name}: the dimensions before the last do not collapse to two strides")
    (outer, so), (inner, si) = [(1, 0)] * (2 - len(levels)) + levels
    return outer, inner, so, si


def _per_row(t, name, count, index, dtypes):
    """Address of a dense array of `count` elements on device `index` (None stays None)."""
    if t is None:
        return None
    if t.dtype not in dtypes:
        raise TypeError(f"{name}: unsupported dtype {t.dtype}")
    if t.get_device() != index or not t.is_contiguous():
        raise ValueError(f"{name}: expected a contiguous tensor on CUDA device {index}")
    if t.numel() != count:
        raise ValueError(f"{name}: expected {count} elements, got {t.numel()}")
    return t.data_ptr()


def _logits(t, name="logits"):
    """(dtype code, device index, outer, inner, vocab, outer stride, inner stride)"""
    code = _LOGITS_DT.get(t.dtype)
    if code is None:
        raise TypeError(f"unsupported {name} dtype {t.dtype}")
    index = t.get_device()
    if index < 0:
        raise ValueError(f"{name}: expected a CUDA tensor")
    if t.dim() > 0 and t.is_contiguous():
        vocab = t.shape[-1]
        return code, index, 1, t.numel() // max(vocab, 1), vocab, 0, vocab
    outer, inner, so, si = _rows(t, name)
    return code, index, outer, inner, t.shape[-1], so, si


_F32 = (torch.float32,)


def token_logprobs(logp, logits, targets, entropy=None, lse=None, top_logp=None, top_index=None, scale=1.0,
                   stream=None):
    """Per row of logits (..., vocab), float32 / float16 / bfloat16, z = scale * logits: writes the log probability of
    the row's token to `logp`, the entropy of its distribution to `entropy`, ln sum e^z to `lse` (float32, one per row,
    each optional; logp may be None) and the k most likely alternatives to `top_logp` and `top_index` (k = their last
    dimension, up to 32; largest first, a tie to the lower index). One launch, one pass over the logits.

    targets: int64 or int32, one per row (None without logp); outside [0, vocab) there is no token: logp 0. top_index:
    dtype of targets, or int64 / int32 without them. The logits' rows may be strided (logits[:, :-1], a padded
    vocabulary); the other tensors are contiguous. Infinities and NaN: see a3b_token_logprobs. Returns logp."""
    code, dev, outer, inner, vocab, so, si = _logits(logits)
    rows = outer * inner
    top, index = 0, capi.I64
    if top_logp is not None or top_index is not None:
        if top_logp is None or top_index is None:
            raise ValueError("top_logp and top_index belong together")
        top = top_logp.shape[-1]
        index = _INDEX_DT.get(top_index.dtype, -1)
    if targets is not None:
        if top and top_index.dtype != targets.dtype:
            raise TypeError("top_index and targets must have the same dtype")
        index = _INDEX_DT.get(targets.dtype, -1)
    elif logp is not None:
        raise ValueError("logp needs targets")
    _call_on(dev, stream, "a3b_token_logprobs", code, logits.data_ptr(), outer, inner, vocab, so, si, scale, index,
             _per_row(targets, "targets", rows, dev, _INDEX_DT), _per_row(logp, "logp", rows, dev, _F32),
             _per_row(entropy, "entropy", rows, dev, _F32), _per_row(lse, "lse", rows, dev, _F32), top,
             _per_row(top_logp, "top_logp", rows * top, dev, _F32),
             _per_row(top_index, "top_index", rows * top, dev, _INDEX_DT))
    return logp


def token_logprobs_backward(grad_logits, logits, targets, lse, entropy=None, grad_logp=None, grad_entropy=None,
                            grad_lse=None, scale=1.0, stream=None):
    """Gradient of token_logprobs' logp, entropy and lse with respect to the logits: given lse (and entropy, for
    grad_entropy) as token_logprobs wrote them and the gradients of a loss with respect to them (float32, one per row;
    None is zero), writes that with respect to the logits to `grad_logits` (shape and dtype of logits; any row strides;
    may be `logits` itself). Rows without a token get nothing from grad_logp. Returns grad_logits."""
    code, dev, outer, inner, vocab, so, si = _logits(logits)
    if grad_logits.shape != logits.shape or grad_logits.dtype != logits.dtype or grad_logits.get_device() != dev:
        raise ValueError("grad_logits must have the shape, dtype and device of logits")
    _, _, go, gi, _, gso, gsi = _logits(grad_logits, "grad_logits")
    if go != outer:  # one of the two collapses further than the other
        if outer == 1:
            outer, inner, so = go, gi, si * gi
        elif go == 1:
            gso = gsi * inner
    if go * gi != outer * inner or (go != 1 and gi != inner):
        raise ValueError("logits and grad_logits do not collapse to the same two dimensions")
    rows = outer * inner
    if lse is None:
        raise ValueError("lse is needed")
    index = capi.I64 if targets is None else _INDEX_DT.get(targets.dtype, -1)
    _call_on(dev, stream, "a3b_token_logprobs_backward", code, logits.data_ptr(), outer, inner, vocab, so, si, scale,
             index, _per_row(targets, "targets", rows, dev, _INDEX_DT), _per_row(lse, "lse", rows, dev, _F32),
             _per_row(entropy, "entropy", rows, dev, _F32), _per_row(grad_logp, "grad_logp", rows, dev, _F32),
             _per_row(grad_entropy, "grad_entropy", rows, dev, _F32), _per_row(grad_lse, "grad_lse", rows, dev, _F32),
             grad_logits.data_ptr(), gso, gsi)
    return grad_logits


# ------------------------------------------------------------------------------------ norm and clipping of a list
def _is_dense(t):
    """Whether t's elements fill one stretch of memory, in any order of the dimensions."""
    if t.is_contiguous():
        return True
    want = 1
    for stride, size in sorted((st, sz) for sz, st in zip(t.shape, t.stride()) if sz != 1):
        if stride != want:
            return False
        want *= size
    return True


class TensorList:
    """A list of CUDA tensors (float32, float64, float16, bfloat16, mixed as needed, of one device) for grad_norm,
    clip_grads and clip_grad_norm, with the tensors that receive the clipped values: `outputs`, with the dtypes, shapes
    and strides of `inputs`, or the inputs themselves (in place). Each tensor must be dense (its elements fill one
    stretch of memory, in any order of dimensions). A None among the inputs (a parameter without a gradient) is left out,
    and what stands in its place in `outputs` with it.

    Making one costs the host about a microsecond per tensor; a program whose gradients stay where they are makes it
    once. It holds the addresses of the tensors as they are now, and keeps those tensors alive."""

    def __init__(self, inputs, outputs=None):
        self._handle = None
        ins = list(inputs)
        outs = ins if outputs is None else list(outputs)
        if len(outs) != len(ins):
            raise ValueError("inputs and outputs must be equally many")
        if any(t is None for t in ins):
            given = [k for k, t in enumerate(ins) if t is not None]
            same = outs is ins
            ins = [ins[k] for k in given]
            outs = ins if same else [outs[k] for k in given]
        self.inputs, self.outputs = ins, outs
        n = len(ins)
        self.device = ins[0].device if n else None
        index = ins[0].get_device() if n else -1
        codes = [_GRAD_DT.get(t.dtype, -1) for t in ins]
        if -1 in codes:
            raise TypeError(f"unsupported dtype {ins[codes.index(-1)].dtype}")
        if n and (index < 0 or any(t.get_device() != index for t in ins)):
            raise ValueError("expected CUDA tensors of one device")
        if not all(t.is_contiguous() or _is_dense(t) for t in ins):
            raise ValueError("expected dense tensors")
        sizes = [t.numel() for t in ins]
        addresses = [t.data_ptr() for t in ins]
        keep = [t.untyped_storage() for t in ins]  # alive even if a tensor moves on
        if outs is ins:
            targets = None
        else:
            for t, o in zip(ins, outs):
                if (o.dtype != t.dtype or o.get_device() != index or o.shape != t.shape
                        or not (o.is_contiguous() and t.is_contiguous() or o.stride() == t.stride())):
                    raise ValueError("an output must have the dtype, device, shape and strides of its input")
            targets = (ctypes.c_void_p * n)(*[o.data_ptr() for o in outs])
            keep += [o.untyped_storage() for o in outs]
        handle = ctypes.c_void_p()
        capi.call("a3b_tensor_list_create", (ctypes.c_void_p * n)(*addresses), targets, (ctypes.c_uint64 * n)(*sizes),
                  (ctypes.c_int * n)(*codes), n, ctypes.byref(handle))
        self._handle = handle
        self._storages = keep
        self._workspace = None

    def __del__(self):
        if getattr(self, "_handle", None) is not None and capi is not None:
            capi.lib().a3b_tensor_list_destroy(self._handle)
            self._handle = None

    def __len__(self):
        return len(self.inputs)

    def _scratch(self, index, stream):
        """Scratch for one call, from torch's allocator in the order of the call's stream."""
        if self._workspace is None:
            with torch.cuda.device(index):
                self._workspace = capi.lib().a3b_grad_norm_workspace(self._handle)
        if stream is None:
            return torch.empty(self._workspace, dtype=torch.uint8, device=torch.device("cuda", index))
        with torch.cuda.stream(stream):
            return torch.empty(self._workspace, dtype=torch.uint8, device=torch.device("cuda", index))


def _scalar(t, name, index, dtypes):
    """Address of one element on device `index` (None stays None)."""
    if t is None:
        return None
    if t.dtype not in dtypes:
        raise TypeError(f"unsupported dtype {t.dtype} of {name}")
    if t.get_device() != index or t.numel() != 1:
        raise ValueError(f"{name}: expected a tensor of one element on CUDA device {index}")
    return t.data_ptr()


_NORM_DT = {torch.float32: capi.F32, torch.float64: capi.F64}


def _list_args(norm, tensors, kind, partial=None):
    """(TensorList, device index, kind code, address of partial, norm's dtype code, norm's address)"""
    if kind not in NORM:
        raise ValueError(f"unknown norm {kind!r}: one of {', '.join(NORM)}")
    if not isinstance(tensors, TensorList):
        tensors = TensorList(tensors)
    index = tensors.device.index if tensors.device is not None else -1
    for t in (norm, partial):
        if index < 0 and t is not None:
            index = t.get_device()
    if index < 0:
        raise ValueError("expected CUDA tensors")
    p = _scalar(partial, "partial", index, (torch.float64,))
    if norm is None:
        return tensors, index, NORM[kind], p, capi.F32, None
    n = _scalar(norm, "norm", index, _NORM_DT)
    return tensors, index, NORM[kind], p, _NORM_DT[norm.dtype], n


def grad_norm(norm, tensors, kind="l2", partial=None, stream=None):
    """Norm over all elements of a list of tensors ("l2", "l1" or "max"; a TensorList or any sequence of tensors) into
    `norm`, one float32 or float64 element on the device. partial: one float64 element that receives the sum of squares,
    the sum of magnitudes or the largest magnitude unrounded, for combination across ranks; either may be None."""
    if norm is None and partial is None:
        raise ValueError("nothing to compute: no output is given")
    tensors, dev, k, p, code, n = _list_args(norm, tensors, kind, partial)
    ws = tensors._scratch(dev, stream)
    _call_on(dev, stream, "a3b_grad_norm", tensors._handle, k, ws.data_ptr(), ws.numel(), p, code, n)
    return norm


def clip_grads(norm, tensors, partial, max_norm, kind="l2", stream=None):
    """Multiplies every tensor of the list by min(1, max_norm / (norm + 1e-6)), with the norm that `partial` stands for
    (as grad_norm wrote it, or combined across ranks), and writes that norm to `norm` (None: not written)."""
    if partial is None:
        raise ValueError("partial is needed")
    tensors, dev, k, p, code, n = _list_args(norm, tensors, kind, partial)
    _call_on(dev, stream, "a3b_clip_grads", tensors._handle, k, p, max_norm, code, n)
    return norm


def clip_grad_norm(norm, tensors, max_norm, kind="l2", stream=None):
    """grad_norm and clip_grads in one call: the tensors of the list scaled down so that their common norm is at most
    `max_norm`, written to the list's outputs (a plain sequence: in place); the norm before goes to `norm`."""
    tensors, dev, k, _, code, n = _list_args(norm, tensors, kind)
    ws = tensors._scratch(dev, stream)
    _call_on(dev, stream, "a3b_clip_grad_norm", tensors._handle, k, max_norm, ws.data_ptr(), ws.numel(), code, n)
    return norm


# ------------------------------------------------------------------------------------------- norm of rows
def _joint_rows(*tensors):
    """(outer, inner, n, [(outer stride, inner stride) of each]) of tensors of one shape, in two levels of rows that fit all
    of them; each is (tensor or None, name), the first never None. None has strides 0."""
    x, name = tensors[0]
    shape = x.shape
    for t, label in tensors:
        if t is not None and (t.dim() < 1 or (t.shape[-1] > 1 and t.stride(-1) != 1)):
            raise ValueError(f"{label}: rows must be contiguous in the last dimension")
    if x.numel() == 0:
        return 0, 0, shape[-1], [(0, 0)] * len(tensors)
    if len(shape) == 2:
        return 1, shape[0], shape[1], [(0, 0) if t is None else (0, t.stride(0)) for t, _ in tensors]
    given = [t for t, _ in tensors if t is not None]
    levels = []  # (size, the strides of each)
    for d in range(x.dim() - 1):
        size, strides = shape[d], tuple(t.stride(d) for t in given)
        if size == 1:
            continue
        if levels and all(a == size * b for a, b in zip(levels[-1][1], strides)):
            levels[-1] = (levels[-1][0] * size, strides)
        else:
            levels.append((size, strides))
    if len(levels) > 2:
        raise ValueError(f"{name}: the dimensions before the last do not collapse to two strides")
    none = (0,) * len(given)
    (outer, so), (inner, si) = [(1, none)] * (2 - len(levels)) + levels
    steps = iter(zip(so, si))
    return outer, inner, shape[-1], [(0, 0) if t is None else next(steps) for t, _ in tensors]


def _like(t, name, shape, dev, dtype):
    if t.shape != shape or t.dtype != dtype or t.get_device() != dev:
        raise ValueError(f"{name} must have the shape and device of the rows, and dtype {dtype}")


def _row_tensor(x, name):
    """(dtype code, device index) of a CUDA tensor of rows"""
    code = _LOGITS_DT.get(x.dtype)
    if code is None:
        raise TypeError(f"unsupported {name} dtype {x.dtype}")
    dev = x.get_device()
    if dev < 0:
        raise ValueError(f"{name}: expected a CUDA tensor")
    if x.dim() < 1:
        raise ValueError(f"{name}: expected at least one dimension")
    return code, dev


def _weight(weight, dtype, n, dev, name="weight"):
    """dtype code of a weight of rows of n elements of `dtype`"""
    if weight.dtype != dtype and weight.dtype != torch.float32:
        raise TypeError(f"{name} must have the dtype of the rows, or float32")
    if weight.get_device() != dev or weight.numel() != n or not weight.is_contiguous():
        raise ValueError(f"{name}: expected {n} contiguous elements on CUDA device {dev}")
    return _LOGITS_DT[weight.dtype]


@functools.lru_cache(maxsize=256)
def _workspace_bytes(entry, dev, *sizes):
    with torch.cuda.device(dev):
        size = getattr(capi.lib(), entry)(*sizes)
    if size == 0:
        raise capi.A3BError(capi.ERR_CUDA, capi.last_error(), entry)
    return size


def _workspace(entry, device, stream, *sizes):
    """(scratch for one call, from torch's allocator in the order of the call's stream; its size in bytes)"""
    size = _workspace_bytes(entry, device.index, *sizes)
    if stream is None:
        return torch.empty(size, dtype=torch.uint8, device=device), size
    with torch.cuda.stream(stream):
        return torch.empty(size, dtype=torch.uint8, device=device), size


def rms_norm(out, x, weight=None, residual=None, total=None, rstd=None, scales=None, group=None, eps=1e-6, stream=None):
    """Per row of x (..., n), float32 / float16 / bfloat16: h = x + residual (rounded to x's dtype), written to `total`;
    1 / sqrt(mean h^2 + eps), written to `rstd` (float32, one per row); out = h * rstd * weight. residual, total, weight and
    rstd are optional. weight: n elements of x's dtype or float32.

    out has x's dtype, or torch.float8_e4m3fn or float8_e5m2 with `scales` (float32, contiguous, one for each `group` = 32,
    64 or 128 elements of a row, or one a row with group None): the values are out * scale.

    Rows of all tensors may be strided (heads of a wider product); out may be x or residual, and total may be residual or x
    (in place). For the gradient keep `total` (x without a residual) and rstd. Infinities, NaN and what may overlap: see
    a3b_rms_norm. Returns out."""
    dtype, dev, shape = x.dtype, x.get_device(), x.shape
    code = _LOGITS_DT.get(dtype)
    if code is None or dev < 0 or not shape:
        _row_tensor(x, "x")
    target = _NORM_OUT_DT.get(out.dtype)
    if target is None:
        raise TypeError(f"unsupported out dtype {out.dtype}")
    n = shape[-1]
    if out.shape != shape or out.get_device() != dev:
        raise ValueError("out must have the shape and device of x")
    flat = x.is_contiguous() and out.is_contiguous()
    res = tot = 0
    if residual is not None:
        _like(residual, "residual", shape, dev, dtype)
        res = residual.data_ptr()
        flat = flat and residual.is_contiguous()
    if total is not None:
        if residual is None:
            raise ValueError("total needs a residual")
        _like(total, "total", shape, dev, dtype)
        tot = total.data_ptr()
        flat = flat and total.is_contiguous()
    wcode, wat = code, 0
    if weight is not None:
        wcode, wat = _weight(weight, dtype, n, dev), weight.data_ptr()
    if flat:
        outer, inner = 1, x.numel() // n if n else 0
        xo = ro = to = oo = 0
        xi = ri = ti = oi = n
    else:
        outer, inner, _, ((xo, xi), (ro, ri), (to, ti), (oo, oi)) = _joint_rows((x, "x"), (residual, "residual"),
                                                                                (total, "total"), (out, "out"))
    size = group or 0
    rat = sat = 0
    if rstd is not None:
        rat = _per_row(rstd, "rstd", outer * inner, dev, _F32)
    if scales is not None:
        sat = _per_row(scales, "scales", outer * inner * (-(-n // size) if size else 1), dev, _F32)
    _call_on(dev, stream, "a3b_rms_norm",
             capi.RMS_NORM_ARGS.pack(outer, inner, n, x.data_ptr(), xo, xi, res, ro, ri, tot, to, ti, out.data_ptr(), oo, oi,
                                     wat, rat, sat, eps, code, target, wcode, size))
    return out


def rms_norm_backward(grad_x, grad_out, x, weight, rstd, grad_weight=None, grad_total=None, stream=None):
    """Gradient of rms_norm's out: given the rows that were normed (`x`: the total, where a residual was added), rstd as
    rms_norm wrote it, and the gradients of a loss with respect to out and to the total itself (grad_total, None: zero),
    writes that with respect to the rows to `grad_x` and that with respect to the weight to `grad_weight` (the weight's
    dtype; None: not computed). With a residual, grad_x is the gradient of both summands. grad_out, grad_total, grad_x have
    the shape and dtype of x, each any row strides; grad_x may be grad_out, x or grad_total. Returns grad_x."""
    code, dev = _row_tensor(x, "x")
    shape, dtype = x.shape, x.dtype
    n = shape[-1]
    _like(grad_out, "grad_out", shape, dev, dtype)
    _like(grad_x, "grad_x", shape, dev, dtype)
    flat = x.is_contiguous() and grad_out.is_contiguous() and grad_x.is_contiguous()
    tot = 0
    if grad_total is not None:
        _like(grad_total, "grad_total", shape, dev, dtype)
        tot = grad_total.data_ptr()
        flat = flat and grad_total.is_contiguous()
    wcode, wat = code, 0
    if weight is not None:
        wcode, wat = _weight(weight, dtype, n, dev), weight.data_ptr()
    if rstd is None:
        raise ValueError("rstd is needed")
    if flat:
        outer, inner = 1, x.numel() // n if n else 0
        xo = go = to = oo = 0
        xi = gi = ti = oi = n
    else:
        outer, inner, _, ((xo, xi), (go, gi), (to, ti), (oo, oi)) = _joint_rows((x, "x"), (grad_out, "grad_out"),
                                                                                (grad_total, "grad_total"), (grad_x, "grad_x"))
    rows = outer * inner
    gcode, gat, at, size = wcode, 0, 0, 0
    if grad_weight is not None:
        gcode, gat = _weight(grad_weight, dtype, n, dev, "grad_weight"), grad_weight.data_ptr()
        if weight is not None and gcode != wcode:
            raise TypeError("grad_weight must have the dtype of the weight")
        ws, size = _workspace("a3b_rms_norm_backward_workspace", x.device, stream, rows, n)
        at = ws.data_ptr()
    _call_on(dev, stream, "a3b_rms_norm_backward",
             capi.RMS_NORM_BACKWARD_ARGS.pack(outer, inner, n, grad_out.data_ptr(), go, gi, x.data_ptr(), xo, xi, tot, to, ti,
                                              grad_x.data_ptr(), oo, oi, wat, _per_row(rstd, "rstd", rows, dev, _F32), gat, at,
                                              size, code, wcode, gcode, 0))
    return grad_x


# ----------------------------------------------------------------------------------------- rows of a table
def _table(t, name, dev):
    """(dtype code, row stride) of a 2-D table of rows on device `dev`"""
    code, where = _row_tensor(t, name)
    if where != dev:
        raise ValueError(f"{name}: expected a tensor on CUDA device {dev}")
    if t.dim() != 2 or (t.shape[1] > 1 and t.stride(1) != 1):
        raise ValueError(f"{name}: expected two dimensions, rows contiguous")
    return code, t.stride(0)


def _token_rows(t, tokens, dev, table, tcode, name):
    """(dtype code, outer, inner, n, outer stride, inner stride, index code, address of the tokens) of rows (..., n) that
    belong to tokens (...) and to rows of `table`"""
    code, where = _row_tensor(t, name)
    if where != dev:
        raise ValueError(f"{name}: expected a tensor on CUDA device {dev}")
    shape = t.shape
    n = shape[-1]
    if shape[:-1] != tokens.shape:
        raise ValueError(f"{name} must have the tokens' shape, and one dimension behind it")
    if table.shape[1] != n:
        raise ValueError(f"{name} and the table must have rows of the same length")
    if code != tcode and capi.F32 not in (code, tcode):
        raise TypeError("rows and table have one dtype, or one of them is float32")
    if t.is_contiguous():
        outer, inner, so, si = 1, tokens.numel(), 0, n
    else:
        outer, inner, _, ((so, si),) = _joint_rows((t, name))
    return (code, outer, inner, n, so, si, _INDEX_DT.get(tokens.dtype, -1),
            _per_row(tokens, "tokens", outer * inner, dev, _INDEX_DT))


def _lookup(table, table_name, rows, name, tokens):
    """(device index, dtype code and row stride of the table, and what _token_rows gives) of rows, their tokens and the table"""
    dev = table.get_device()
    shape = table.shape
    # The usual call, told by one question after the other; any other answer goes the long way, which also says what is wrong.
    if len(shape) == 2 and shape[1] and rows.is_contiguous() and tokens.is_contiguous() and table.is_contiguous():
        code, tcode, index = _LOGITS_DT.get(rows.dtype), _LOGITS_DT.get(table.dtype), _INDEX_DT.get(tokens.dtype)
        if (code is not None and tcode is not None and index is not None and dev >= 0 and rows.get_device() == dev
                and tokens.get_device() == dev and (code == tcode or code == capi.F32 or tcode == capi.F32)
                and rows.shape == tokens.shape + shape[1:]):
            n = shape[1]
            return dev, tcode, n, code, 1, tokens.numel(), n, 0, n, index, tokens.data_ptr()
    tcode, stride = _table(table, table_name, dev)
    return dev, tcode, stride, *_token_rows(rows, tokens, dev, table, tcode, name)


def embedding(out, weight, tokens, scale=1.0, first=0, stream=None):
    """out[...] = scale * weight[tokens[...] - first], one row of the table `weight` (rows, n) for each token (int64 or
    int32, contiguous, any shape; out: that shape and n). A token outside [first, first + rows) gives a row of zeros: padding
    such as -100, or the tokens of other ranks where the table is cut over ranks. Types: float32 / float16 / bfloat16, both
    alike or one of them float32. Rows may be strided. Returns out."""
    dev, tcode, stride, code, outer, inner, n, so, si, index, at = _lookup(weight, "weight", out, "out", tokens)
    _call_on(dev, stream, "a3b_embedding",
             capi.EMBEDDING_ARGS.pack(outer, inner, n, weight.shape[0], first, weight.data_ptr(), stride, at, out.data_ptr(),
                                      so, si, scale, tcode, index, code, 0))
    return out


def embedding_backward(grad_weight, grad_out, tokens, scale=1.0, add=None, first=0, stream=None):
    """Gradient of embedding's out with respect to the table: every row of `grad_weight` (rows, n) is add's row (zero without
    `add`) plus scale times the sum of grad_out's rows over the places of its token. `add` has the dtype and shape of
    grad_weight (the gradient from the table's use as a head); it may be grad_weight itself, of which then only rows of
    tokens that occur are touched. The same bits in every call. Returns grad_weight."""
    dev, tcode, stride, code, outer, inner, n, so, si, index, at = _lookup(grad_weight, "grad_weight", grad_out, "grad_out",
                                                                           tokens)
    more = more_stride = 0
    if add is not None:
        acode, more_stride = _table(add, "add", dev)
        if acode != tcode or add.shape != grad_weight.shape:
            raise ValueError("add must have the dtype and shape of grad_weight")
        more = add.data_ptr()
    vocab = grad_weight.shape[0]
    ws, size = _workspace("a3b_embedding_backward_workspace", grad_weight.device, stream, outer * inner, n, vocab)
    _call_on(dev, stream, "a3b_embedding_backward",
             capi.EMBEDDING_BACKWARD_ARGS.pack(outer, inner, n, vocab, first, grad_out.data_ptr(), so, si, at, more, more_stride,
                                               grad_weight.data_ptr(), stride, ws.data_ptr(), size, scale, code, index, tcode, 0))
    return grad_weight


# ------------------------------------------------------------------------------------------ drafted tokens
def _draft_rows(t, name, batch, length, dev, dtype):
    """(address, batch stride, row stride) of logits (batch, length, vocab)"""
    shape = t.shape
    if t.dtype != dtype or t.get_device() != dev:
        raise ValueError(f"{name} must have the dtype of the logits and lie on CUDA device {dev}")
    if len(shape) != 3 or shape[0] != batch or shape[1] != length or (shape[2] > 1 and t.stride(2) != 1):
        raise ValueError(f"{name}: expected shape ({batch}, {length}, vocab), rows contiguous")
    so, si, _ = t.stride()
    return t.data_ptr(), so, si


def verify_drafts(tokens, accepted, drafts, logits=None, lse=None, uniform=None, noise=None, draft_logits=None,
                  draft_lse=None, scale=1.0, draft_scale=None, top_index=None, stream=None):
    """For every sequence of a batch: how many of its drafted tokens stand against the target's probabilities, to `accepted`
    (batch), and those tokens, the one drawn behind them, and -1 for the rest, to `tokens` (batch, length + 1).

    drafts (batch, length): the first one outside [0, vocab) ends a sequence's draft. logits (batch, length + 1, vocab),
    float32 / float16 / bfloat16, and lse (batch, length + 1) as token_logprobs writes it at the same `scale`: position i's
    row predicts draft i. draft_logits (batch, length, vocab) and draft_lse (batch, length) are those the drafts were drawn
    from, at draft_scale (None: scale); without them the drafts were certain (looked up). uniform (batch, length): float32 in
    [0, 1); noise (batch, vocab): float32 exponential variates. Tokens are then distributed as if drawn from the target one
    by one. length may be 0: one token is drawn from each row.

    top_index (batch, length + 1): the target's most likely token of every row (token_logprobs with one alternative);
    sequences whose first entry is a token are verified greedily, without random numbers; all of them if logits is None.
    drafts, tokens, accepted and top_index have one dtype, int64 or int32. See a3b_verify_drafts. Returns tokens."""
    index = _INDEX_DT.get(drafts.dtype)
    if index is None:
        raise TypeError(f"unsupported drafts dtype {drafts.dtype}")
    dev = drafts.get_device()
    if dev < 0:
        raise ValueError("drafts: expected a CUDA tensor")
    shape = drafts.shape
    if len(shape) != 2:
        raise ValueError("drafts: expected shape (batch, length)")
    batch, length = shape
    same = (drafts.dtype,)
    places = batch * (length + 1)
    code, vocab, at, lb, ls = capi.F32, (1 << 31) - 65, 0, 0, 0
    other, db, ds, noise_at, noise_stride = 0, 0, 0, 0, 0
    if logits is not None:
        code = _LOGITS_DT.get(logits.dtype)
        if code is None:
            raise TypeError(f"unsupported logits dtype {logits.dtype}")
        if lse is None or noise is None or (uniform is None and length):
            raise ValueError("logits need lse, uniform and noise")
        at, lb, ls = _draft_rows(logits, "logits", batch, length + 1, dev, logits.dtype)
        vocab = logits.shape[2]
        if draft_logits is not None:
            if draft_lse is None:
                raise ValueError("draft_logits need draft_lse")
            if draft_logits.shape[-1] != vocab:
                raise ValueError("logits and draft_logits must have the same vocabulary")
            other, db, ds = _draft_rows(draft_logits, "draft_logits", batch, length, dev, logits.dtype)
        if (noise.dtype != torch.float32 or noise.get_device() != dev or noise.shape != (batch, vocab)
                or (vocab > 1 and noise.stride(1) != 1)):
            raise ValueError(f"noise: expected float32 of shape ({batch}, {vocab}) on CUDA device {dev}, rows contiguous")
        noise_at, noise_stride = noise.data_ptr(), noise.stride(0)
    elif top_index is None:
        raise ValueError("neither logits nor top_index is given")
    elif draft_logits is not None:
        raise ValueError("draft_logits need logits")
    _call_on(dev, stream, "a3b_verify_drafts",
             capi.VERIFY_DRAFTS_ARGS.pack(batch, length, vocab, at, lb, ls, other, db, ds,
                                          _per_row(lse, "lse", places, dev, _F32) or 0,
                                          _per_row(draft_lse, "draft_lse", batch * length, dev, _F32) or 0, scale,
                                          scale if draft_scale is None else draft_scale,
                                          _per_row(drafts, "drafts", batch * length, dev, same),
                                          _per_row(top_index, "top_index", places, dev, same) or 0,
                                          _per_row(uniform, "uniform", batch * length, dev, _F32) or 0, noise_at, noise_stride,
                                          _per_row(tokens, "tokens", places, dev, same),
                                          _per_row(accepted, "accepted", batch, dev, same), code, index))
    return tokens


# ------------------------------------------------------------------------------------------------------- nBody
def nbody_update_velocities(m, x, y, z, vx, vy, vz, dt, eps, i_begin=0, stream=None):
    capi.call("a3b_nbody_update_velocities", stream_handle(stream), _ptr(m), _ptr(x), _ptr(y), _ptr(z), m.numel(),
              i_begin, vx.numel(), _ptr(vx), _ptr(vy), _ptr(vz), float(dt), float(eps))


def nbody_update_positions(x, y, z, vx, vy, vz, dt, stream=None):
    capi.call("a3b_nbody_update_positions", stream_handle(stream), _ptr(x), _ptr(y), _ptr(z), _ptr(vx), _ptr(vy),
              _ptr(vz), x.numel(), float(dt))


def nbody_step(m, x, y, z, vx, vy, vz, dt, eps, i_begin=0, stream=None):
    capi.call("a3b_nbody_step", stream_handle(stream), _ptr(m), _ptr(x), _ptr(y), _ptr(z), m.numel(), i_begin,
              vx.numel(), _ptr(vx), _ptr(vy), _ptr(vz), float(dt), float(eps))


# -------------------------------------------------------------------------------------------------------- heat
def haccmk_step10(xx, yy, zz, mass, vx2, vy2, vz2, n1, fsrrmax2, mp_rsm2, fcoeff, stream=None):
    """HACCmk's Step10 short-range force for the first n1 particles against all of xx/yy/zz/mass (float32)."""
    capi.call("a3b_haccmk_step10", stream_handle(stream), _ptr(xx), _ptr(yy), _ptr(zz), _ptr(mass), int(n1),
              xx.numel(), float(fsrrmax2), float(mp_rsm2), float(fcoeff), _ptr(vx2), _ptr(vy2), _ptr(vz2))


def heat_step(cur, nxt, rX, rY, row_begin=1, row_end=None, stream=None):
    """cur/nxt: (rows+2, cols+2) float64 tensors (rows may be pitched: stride(0) >= cols + 2)."""
    rows, cols = cur.shape[0] - 2, cur.shape[1] - 2
    if row_end is None:
        row_end = rows + 1
    if cur.stride(1) != 1 or nxt.stride() != cur.stride():
        raise ValueError("grids must share a row pitch and be contiguous within rows")
    capi.call("a3b_heat_step", stream_handle(stream), ctypes.c_void_p(cur.data_ptr()),
              ctypes.c_void_p(nxt.data_ptr()), rows, cols, cur.stride(0), row_begin, row_end, float(rX), float(rY))


def heat_init(u, dx, dy, row_offset=0, global_rows=None, stream=None):
    rows, cols = u.shape[0] - 2, u.shape[1] - 2
    if global_rows is None:
        global_rows = rows
    capi.call("a3b_heat_init", stream_handle(stream), ctypes.c_void_p(u.data_ptr()), rows, cols, u.stride(0),
              row_offset, global_rows, float(dx), float(dy))


def heat_exact(u, t, dx, dy, ring_only=False, row_offset=0, global_rows=None, stream=None):
    """The heatEquation2D example's exact solution at time t on every cell, or on the global ring only."""
    rows, cols = u.shape[0] - 2, u.shape[1] - 2
    if global_rows is None:
        global_rows = rows
    capi.call("a3b_heat_exact", stream_handle(stream), ctypes.c_void_p(u.data_ptr()), rows, cols, u.stride(0),
              row_offset, global_rows, float(t), float(dx), float(dy), 1 if ring_only else 0)


def heat_problem(n, steps, t_max, device, stream=None):
    """Runs the heatEquation2D example's own problem (heatEquation2D.cpp:97-196) on the device: exact initial field,
    `steps` Jacobi steps with the exact solution re-imposed on the ring after each; returns the final field."""
    extent = n + 2
    dx = 1.0 / (extent - 1)
    dy = 1.0 / (extent - 1)
    dt = t_max / steps
    rX = dt / (dx * dx)
    rY = dt / (dy * dy)
    cur = torch.empty((extent, extent), dtype=torch.float64, device=device)
    heat_exact(cur, 0.0, dx, dy, stream=stream)
    nxt = cur.clone()
    for step in range(1, steps + 1):
        heat_step(cur, nxt, rX, rY, stream=stream)
        heat_exact(nxt, float(step) * dt, dx, dy, ring_only=True, stream=stream)
        cur, nxt = nxt, cur
    return cur
