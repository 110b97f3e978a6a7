"""Operators of image networks beside their convolutions, through the C ABI
(rdv_group_norm, rdv_cross_attention, rdv_dropout and the backward calls).
Build-defined: the reference has no counterpart.

The functions take GPU tensors (torch tensors or RDVObjects) of float32,
float16 or bfloat16, read strided views in place where the innermost dimension
is contiguous (any other layout is copied first), return fresh contiguous
tensors unless the caller passes `out`, and launch on torch's current stream.
Gradients are explicit calls, as mse_backward's are.  The TensorOperation forms
are in nn.py.  There is no CPU path."""
from __future__ import annotations

import ctypes as C
import math

import torch

from . import _lib
from .core import RDVObject, current_stream_handle, launch_scope

_DTYPES = {torch.float32: _lib.DTYPE_F32, torch.float16: _lib.DTYPE_F16, torch.bfloat16: _lib.DTYPE_BF16}
_ACTIVATIONS = {"none": _lib.ACT_NONE, "relu": _lib.ACT_RELU, "silu": _lib.ACT_SILU}


def _tensor(t, what: str) -> torch.Tensor:
    if isinstance(t, RDVObject):
        return t.as_tensor("torch")
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{what} must be a torch tensor, got {type(t).__name__}")
    return t


def _data(t, what: str) -> torch.Tensor:
    t = _tensor(t, what)
    if t.dtype not in _DTYPES:
        raise TypeError(f"{what} must be float32, float16 or bfloat16, got {t.dtype}")
    return t


def _like(t, x: torch.Tensor, what: str) -> torch.Tensor:
    """t as a tensor of x's shape and type."""
    t = _data(t, what)
    assert t.shape == x.shape, f"{what} must have shape {list(x.shape)}, got {list(t.shape)}"
    if t.dtype != x.dtype:
        raise TypeError(f"{what} must be {x.dtype}, got {t.dtype}")
    return t


def _on_gpu(*named) -> None:
    """Every tensor on the current GPU: launches go there, on its current stream."""
    for t, what in named:
        if t is None:
            continue
        if not t.is_cuda:
            raise TypeError(f"{what} must be a GPU tensor, got device {t.device}")
        if t.device.index != torch.cuda.current_device():
            raise TypeError(f"{what} is on {t.device}, the current GPU is cuda:{torch.cuda.current_device()}")


def _out_tensor(out, shape, dtype, device, what: str = "out", aligned: bool = True) -> torch.Tensor:
    """The caller's buffer, checked to be what the kernels write, or a fresh one."""
    if out is None:
        return torch.empty(shape, dtype=dtype, device=device)
    out = _tensor(out, what)
    assert tuple(out.shape) == tuple(shape), f"{what} must have shape {list(shape)}, got {list(out.shape)}"
    if out.dtype != dtype or out.device != device:
        raise TypeError(f"{what} must be {dtype} on {device}, got {out.dtype} on {out.device}")
    assert out.is_contiguous(), f"{what} must be contiguous"
    assert not aligned or out.data_ptr() % 16 == 0, f"{what} must be 16-byte aligned"
    return out


def _grad_tensors(grads, shapes, dtypes, device, names):
    if grads is None:
        grads = (None,) * len(shapes)
    if not isinstance(grads, (list, tuple)) or len(grads) != len(shapes):
        raise TypeError(f"grads must be ({', '.join(names)})")
    return tuple(_out_tensor(g, s, t, device, n) for g, s, t, n in zip(grads, shapes, dtypes, names))


def _apart(out: torch.Tensor, *inputs) -> None:
    """The kernels read inputs after they have begun to write: no sharing of memory."""
    for t, what in inputs:
        if t is not None and t.numel() and out.numel():
            span = sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1
            a, b = out.data_ptr(), t.data_ptr()
            assert a >= b + span * t.element_size() or b >= a + out.numel() * out.element_size(), \
                f"out must not share memory with {what}"


def _workspace(nbytes: int, what: str, device) -> tuple:
    """(tensor, pointer, bytes): scratch of one call, from the allocator so that calls on other streams get their own."""
    if nbytes < 0:
        _lib.check(int(nbytes), what)
    if nbytes == 0:
        return None, 0, 0
    ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
    return ws, ws.data_ptr(), nbytes


def _ptr(t) -> int:
    return 0 if t is None else t.data_ptr()


# ------------------------------------------------------------ group normalisation


def _image_rows(t: torch.Tensor) -> tuple:
    """(t or its contiguous copy, image stride, row stride) of t [images, ..., channels] or [rows, channels]."""
    if not t.is_contiguous():
        shape, stride = t.shape, t.stride()
        first = 1 if t.dim() > 2 else 0
        merged = stride[-1] == 1 or shape[-1] == 1
        step, count = None, 1
        for i in range(t.dim() - 2, first - 1, -1):  # the dimensions of the rows, innermost first
            if shape[i] == 1:
                continue
            if step is None:
                step = stride[i]
            merged = merged and stride[i] == step * count
            count *= shape[i]
        if merged:
            return t, (stride[0] if first else 0), (step or 0)
        t = t.contiguous()
    channels = t.shape[-1]
    return t, (t.numel() // max(1, t.shape[0]) if t.dim() > 2 else 0), channels


def _norm_inputs(x, weight, bias, groups, eps, activation):
    x = _data(x, "x")
    assert x.dim() >= 2, "x must be [rows, channels] (one image) or [images, ..., channels]"
    channels = int(x.shape[-1])
    assert channels >= 1 and int(groups) >= 1 and channels % int(groups) == 0, \
        f"groups ({groups}) must divide the channels ({channels})"
    if activation not in _ACTIVATIONS:
        raise ValueError(f"activation must be one of {sorted(_ACTIVATIONS)}, got {activation!r}")
    params = []
    for p, what in ((weight, "weight"), (bias, "bias")):
        if p is not None:
            p = _tensor(p, what)
            assert tuple(p.shape) == (channels,), f"{what} must be [channels]"
            if p.dtype != torch.float32:
                raise TypeError(f"{what} must be float32, got {p.dtype}")
            p = p.contiguous()
        params.append(p)
    d = _lib.GroupNormDesc()
    d.images = int(x.shape[0]) if x.dim() > 2 else 1
    d.rows = math.prod(x.shape[1:-1]) if x.dim() > 2 else int(x.shape[0])
    d.channels, d.groups, d.eps = channels, int(groups), float(eps)
    d.act, d.dtype = _ACTIVATIONS[activation], _DTYPES[x.dtype]
    return x, params[0], params[1], d


def _group_norm_into(d, x, weight, bias, y, stats) -> None:
    """Launches rdv_group_norm into y and stats (or None)."""
    x, d.x_image_stride, d.x_row_stride = _image_rows(x)
    lib = _lib.load()
    ws, wp, wn = _workspace(lib.rdv_group_norm_workspace_bytes(C.byref(d), 0), "group_norm", x.device)
    _lib.check(lib.rdv_group_norm(C.byref(d), x.data_ptr(), _ptr(weight), _ptr(bias), y.data_ptr(), _ptr(stats), wp,
                                  wn, current_stream_handle()), "group_norm")


def group_norm(x, weight, bias, groups: int, eps: float = 1e-5, activation: str = "none", out=None,
               return_stats: bool = False):
    """activation(weight * (x - mean) / sqrt(var + eps) + bias) over channels-last
    images, with mean and (biased) variance over an image's rows and each of
    `groups` equal runs of channels.  x: [rows, channels] (one image, the
    tensor operations' layout) or [images, ..., channels]; weight and bias:
    float32 [channels] or None; activation: "none", "relu" (a NaN gives 0, as
    ReLUTensorOp does) or "silu".  Returns y like x, contiguous, and with
    return_stats also stats [images, groups, 2] = (mean, 1 / std) in float32,
    which group_norm_backward takes."""
    x, weight, bias, d = _norm_inputs(x, weight, bias, groups, eps, activation)
    _on_gpu((x, "x"), (weight, "weight"), (bias, "bias"))
    y = _out_tensor(out, x.shape, x.dtype, x.device)
    if out is not None:
        _apart(y, (x, "x"), (weight, "weight"), (bias, "bias"))
    stats = torch.empty((d.images, d.groups, 2), dtype=torch.float32, device=x.device) if return_stats else None
    with launch_scope():
        _group_norm_into(d, x, weight, bias, y, stats)
    return (y, stats) if return_stats else y


def group_norm_backward(grad, x, weight, bias, groups: int, stats, activation: str = "none", grads=None):
    """(dx, dweight, dbias) of group_norm for grad = dL/dy, given the stats it
    returned for the same x, weight, bias, groups and activation.  dx is like
    x, dweight and dbias are float32 [channels]; `grads` supplies the three
    buffers."""
    x, weight, bias, d = _norm_inputs(x, weight, bias, groups, 0.0, activation)
    grad = _like(grad, x, "grad")
    stats = _tensor(stats, "stats")
    assert tuple(stats.shape) == (d.images, d.groups, 2) and stats.is_contiguous(), \
        f"stats must be a contiguous [{d.images}, {d.groups}, 2] tensor, as group_norm returns it"
    if stats.dtype != torch.float32:
        raise TypeError(f"stats must be float32, got {stats.dtype}")
    _on_gpu((x, "x"), (grad, "grad"), (weight, "weight"), (bias, "bias"), (stats, "stats"))
    dx, dw, db = _grad_tensors(grads, (x.shape, (d.channels,), (d.channels,)), (x.dtype, torch.float32, torch.float32),
                               x.device, ("dx", "dweight", "dbias"))
    if grads is not None:
        for t in (dx, dw, db):
            _apart(t, (x, "x"), (grad, "grad"), (weight, "weight"), (bias, "bias"), (stats, "stats"))
    lib = _lib.load()
    with launch_scope():
        x, d.x_image_stride, d.x_row_stride = _image_rows(x)
        grad, d.g_image_stride, d.g_row_stride = _image_rows(grad)
        ws, wp, wn = _workspace(lib.rdv_group_norm_workspace_bytes(C.byref(d), 1), "group_norm_backward", x.device)
        _lib.check(lib.rdv_group_norm_backward(C.byref(d), grad.data_ptr(), x.data_ptr(), _ptr(weight), _ptr(bias),
                                               stats.data_ptr(), dx.data_ptr(), dw.data_ptr(), db.data_ptr(), wp, wn,
                                               current_stream_handle()), "group_norm_backward")
    return dx, dw, db


# ------------------------------------------------------------ cross attention


def _innermost(t: torch.Tensor) -> torch.Tensor:
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _rows_in_place(t: torch.Tensor) -> torch.Tensor:
    """t [batch, length, heads, dim] as the library reads it: the innermost dimension contiguous and, as rows whose
    strides are multiples of 16 bytes are read in pieces of that size, such a tensor itself aligned to it."""
    t = _innermost(t)
    return t if t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.contiguous_format)


def _attention_inputs(q, k, v, key_lengths, key_mask, scale):
    q, k, v = _data(q, "q"), _data(k, "k"), _data(v, "v")
    assert q.dim() == 4, "q must be [batch, queries, heads, dim]"
    assert k.dim() == 4 and k.shape == v.shape, "k and v must both be [batch, keys, kv_heads, dim]"
    b, lq, hq, dim = (int(n) for n in q.shape)
    lk, hkv = int(k.shape[1]), int(k.shape[2])
    assert int(k.shape[0]) == b, f"q has a batch of {b}, k and v of {k.shape[0]}"
    assert int(k.shape[3]) == dim, f"q has heads of {dim} dimensions, k and v of {k.shape[3]}"
    assert hkv >= 1 and hq >= 1 and hq % hkv == 0, f"kv_heads ({hkv}) must divide heads ({hq})"
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError(f"q, k and v must have one type, got {q.dtype}, {k.dtype} and {v.dtype}")
    if key_lengths is not None:
        key_lengths = _tensor(key_lengths, "key_lengths")
        assert tuple(key_lengths.shape) == (b,), f"key_lengths must be [batch] = [{b}]"
        if key_lengths.dtype not in (torch.int32, torch.int64):
            raise TypeError(f"key_lengths must be int32 or int64, got {key_lengths.dtype}")
    if key_mask is not None:
        key_mask = _tensor(key_mask, "key_mask")
        assert tuple(key_mask.shape) == (b, lk), f"key_mask must be [batch, keys] = [{b}, {lk}]"
        if key_mask.dtype != torch.bool:
            raise TypeError(f"key_mask must be bool, got {key_mask.dtype}")
    scale = 1.0 / math.sqrt(dim) if scale is None else float(scale)
    if not math.isfinite(scale):
        raise ValueError(f"scale must be finite, got {scale}")
    _on_gpu((q, "q"), (k, "k"), (v, "v"), (key_lengths, "key_lengths"), (key_mask, "key_mask"))
    q, k, v = _rows_in_place(q), _rows_in_place(k), _rows_in_place(v)
    d = _lib.AttentionDesc()
    d.batch, d.queries, d.keys, d.heads, d.kv_heads, d.dim = b, lq, lk, hq, hkv, dim
    d.dtype, d.scale = _DTYPES[q.dtype], scale
    d.q_stride[:], d.k_stride[:], d.v_stride[:] = q.stride()[:3], k.stride()[:3], v.stride()[:3]
    if key_lengths is not None:
        key_lengths = key_lengths.clamp(0, lk).to(torch.int32) if key_lengths.dtype == torch.int64 else key_lengths
        key_lengths = key_lengths.contiguous()
    if key_mask is not None:
        key_mask = _innermost(key_mask) if lk else None
        d.mask_stride = key_mask.stride(0) if lk else 0
    return q, k, v, key_lengths, key_mask, d


def _cross_attention_into(d, q, k, v, key_lengths, key_mask, out, lse) -> None:
    """Launches rdv_cross_attention into out and lse (or None)."""
    lib = _lib.load()
    ws, wp, wn = _workspace(lib.rdv_cross_attention_workspace_bytes(C.byref(d), 0), "cross_attention", q.device)
    _lib.check(lib.rdv_cross_attention(C.byref(d), q.data_ptr(), k.data_ptr(), v.data_ptr(), _ptr(key_lengths),
                                       _ptr(key_mask), out.data_ptr(), _ptr(lse), wp, wn, current_stream_handle()),
               "cross_attention")


def cross_attention(q, k, v, key_lengths=None, key_mask=None, scale: float | None = None, out=None,
                    return_lse: bool = False):
    """softmax(scale q k^T) v from q [batch, queries, heads, dim] to the states of
    another sequence, k and v [batch, keys, kv_heads, dim] (views of one
    projection's output, say); head h reads state head h // (heads // kv_heads);
    dim at most 128; scale defaults to 1 / sqrt(dim).  Of item b the states
    j < key_lengths[b] (int32 or int64 [batch]) with key_mask[b, j] (bool
    [batch, keys]) count; what k and v hold elsewhere has no effect.  A query
    with no state gets 0.  Returns out [batch, queries, heads, dim] and with
    return_lse also lse [batch, heads, queries] float32, the logarithm of each
    softmax's denominator (-inf where no state counts), which
    cross_attention_backward takes.  float16 and bfloat16 inputs: the matrix
    cores take softmax terms rounded to that type; float32: float32
    throughout."""
    q, k, v, key_lengths, key_mask, d = _attention_inputs(q, k, v, key_lengths, key_mask, scale)
    given = out is not None
    out = _out_tensor(out, q.shape, q.dtype, q.device)
    if given:
        _apart(out, (q, "q"), (k, "k"), (v, "v"), (key_lengths, "key_lengths"), (key_mask, "key_mask"))
    lse = torch.empty((d.batch, d.heads, d.queries), dtype=torch.float32, device=q.device) if return_lse else None
    with launch_scope():
        _cross_attention_into(d, q, k, v, key_lengths, key_mask, out, lse)
    return (out, lse) if return_lse else out


def cross_attention_backward(grad, q, k, v, out, lse, key_lengths=None, key_mask=None, scale: float | None = None,
                             grads=None):
    """(dq, dk, dv) of cross_attention for grad = dL/dout, given the out and lse
    it returned for the same arguments.  dk and dv are summed over the heads
    that share a state head and are 0 at states that do not count; `grads`
    supplies the three buffers."""
    q, k, v, key_lengths, key_mask, d = _attention_inputs(q, k, v, key_lengths, key_mask, scale)
    grad, out = _like(grad, q, "grad"), _like(out, q, "out").contiguous()
    lse = _tensor(lse, "lse")
    assert tuple(lse.shape) == (d.batch, d.heads, d.queries) and lse.is_contiguous(), \
        f"lse must be a contiguous [{d.batch}, {d.heads}, {d.queries}] tensor, as cross_attention returns it"
    if lse.dtype != torch.float32:
        raise TypeError(f"lse must be float32, got {lse.dtype}")
    _on_gpu((grad, "grad"), (out, "out"), (lse, "lse"))
    grad = _rows_in_place(grad)
    d.g_stride[:] = grad.stride()[:3]
    given = grads is not None
    grads = _grad_tensors(grads, (q.shape, k.shape, v.shape), (q.dtype,) * 3, q.device, ("dq", "dk", "dv"))
    if given:
        for t in grads:
            _apart(t, (grad, "grad"), (q, "q"), (k, "k"), (v, "v"), (out, "out"), (lse, "lse"),
                   (key_lengths, "key_lengths"), (key_mask, "key_mask"))
    dq, dk, dv = grads
    lib = _lib.load()
    with launch_scope():
        ws, wp, wn = _workspace(lib.rdv_cross_attention_workspace_bytes(C.byref(d), 1), "cross_attention_backward",
                                q.device)
        _lib.check(lib.rdv_cross_attention_backward(C.byref(d), grad.data_ptr(), q.data_ptr(), k.data_ptr(),
                                                    v.data_ptr(), out.data_ptr(), lse.data_ptr(), _ptr(key_lengths),
                                                    _ptr(key_mask), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), wp,
                                                    wn, current_stream_handle()), "cross_attention_backward")
    return dq, dk, dv


# ------------------------------------------------------------ dropout


def _dropout_inputs(x, p, seed, subsequence):
    x = _data(x, "x")
    p, seed, subsequence = float(p), int(seed), int(subsequence)
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"p must be in [0, 1], got {p}")
    for value, what in ((seed, "seed"), (subsequence, "subsequence")):
        if not 0 <= value < 1 << 64:
            raise ValueError(f"{what} must be in [0, 2^64), got {value}")
    return x, p, seed, subsequence


def _dropout_into(x, p, seed, subsequence, residual, y) -> None:
    """Launches rdv_dropout into y."""
    x = x.contiguous()
    residual = None if residual is None else residual.contiguous()
    _lib.check(_lib.load().rdv_dropout(x.data_ptr(), _ptr(residual), y.data_ptr(), x.numel(), _DTYPES[x.dtype], p,
                                       seed, subsequence, current_stream_handle()), "dropout")


def dropout(x, p: float, seed: int, subsequence: int = 0, residual=None, out=None):
    """residual + x * keep / (1 - p): each element of x is dropped with
    probability p.  The mask is a function of (seed, subsequence, the element's
    row-major index) alone -- word i % 4 of Philox4x32-10 at counter (i // 4,
    subsequence) under key seed keeps element i where it is at least
    floor(p 2^32) -- and is never stored: dropout_backward makes it again.  Give every layer and step its
    own subsequence.  residual: a tensor like x, added after.  `out` may be x
    or residual itself."""
    x, p, seed, subsequence = _dropout_inputs(x, p, seed, subsequence)
    if residual is not None:
        residual = _like(residual, x, "residual")
    _on_gpu((x, "x"), (residual, "residual"))
    y = _out_tensor(out, x.shape, x.dtype, x.device, aligned=False)
    if out is not None:
        for t, what in ((x, "x"), (residual, "residual")):
            if t is not None and not (t.data_ptr() == y.data_ptr() and t.is_contiguous()):
                _apart(y, (t, what))
    with launch_scope():
        _dropout_into(x, p, seed, subsequence, residual, y)
    return y


def dropout_backward(grad, p: float, seed: int, subsequence: int = 0, out=None):
    """The gradient of x of dropout(x, p, seed, subsequence): grad * keep / (1 - p)
    with the same mask.  (The residual's gradient is grad itself.)"""
    return dropout(grad, p, seed, subsequence, out=out)
