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
import functools
import math

import torch

from . import _lib
from .core import RDVObject, launch_scope

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


def _gpu_index() -> int:
    """The current GPU, or -1 where there is none (arguments are still checked there)."""
    return torch._C._cuda_getDevice() if torch.cuda.is_initialized() else -1


def _stream(device: int) -> int:
    """The handle of the device's current stream."""
    return torch._C._cuda_getCurrentRawStream(device)


def _on_gpu(device: int, *named) -> None:
    """Every tensor (followed by its name) on the current GPU: launches go there, on its current stream."""
    for i in range(0, len(named), 2):
        t = named[i]
        if t is not None and (t.get_device() != device or device < 0):
            if not t.is_cuda:
                raise TypeError(f"{named[i + 1]} must be a GPU tensor, got device {t.device}")
            raise TypeError(f"{named[i + 1]} is on {t.device}, the current GPU is cuda:{device}")


def _like_out(out, x: torch.Tensor, aligned: bool = True) -> torch.Tensor:
    """The caller's buffer for a result like x, or a fresh contiguous one."""
    if out is None:
        return torch.empty_like(x) if x.is_contiguous() else x.new_empty(x.shape)
    return _out_tensor(out, x.shape, x.dtype, x.device, "out", aligned)


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


def _grad_tensors(grads, likes, names):
    """The caller's buffers for gradients of `likes`, or fresh contiguous ones."""
    if grads is None:
        return tuple(_like_out(None, t) for t in likes)
    if not isinstance(grads, (list, tuple)) or len(grads) != len(likes):
        raise TypeError(f"grads must be ({', '.join(names)})")
    grads = tuple(_out_tensor(g, t.shape, t.dtype, t.device, n) for g, t, n in zip(grads, likes, names))
    for i, g in enumerate(grads):
        _apart(g, *zip(grads[:i], names))
    return grads


def _apart(out: torch.Tensor, *inputs) -> None:
    """The kernels read inputs after they have begun to write: no sharing of memory."""
    for t, what in inputs:
        if t is not None and t.numel() and out.numel():
            span = sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1
            a, b = out.data_ptr(), t.data_ptr()
            assert a >= b + span * t.element_size() or b >= a + out.numel() * out.element_size(), \
                f"out must not share memory with {what}"


def _check(rc: int, what: str) -> None:
    if rc:
        _lib.check(rc, what)


def _ptr(t) -> int:
    return 0 if t is None else t.data_ptr()


# ------------------------------------------------------------ group normalisation


def _image_rows(shape, stride):
    """(image stride, row stride) of a tensor [images, ..., channels] or [rows, channels] of these strides, or None
    where its rows do not lie at one distance with contiguous channels."""
    if stride[-1] != 1 and shape[-1] != 1:
        return None
    first = 1 if len(shape) > 2 else 0
    step, count = None, 1
    for i in range(len(shape) - 2, first - 1, -1):  # the dimensions of the rows, innermost first
        if shape[i] == 1:
            continue
        if step is None:
            step = stride[i]
        elif stride[i] != step * count:
            return None
        count *= shape[i]
    return (stride[0] if first else 0), (step or 0)


@functools.lru_cache(maxsize=4096)
def _norm_plan(shape, x_stride, g_stride, dtype, groups, eps, activation, device):
    """What a call on tensors of this layout needs, by layout alone: (descriptor, whether x and grad have to be copied
    first, workspace bytes).  g_stride is None for the forward call; `device` is the GPU it is planned for."""
    channels = shape[-1]
    assert channels >= 1 and groups >= 1 and channels % groups == 0, \
        f"groups ({groups}) must divide the channels ({channels})"
    if activation not in _ACTIVATIONS:
        raise ValueError(f"activation must be one of {sorted(_ACTIVATIONS)}, got {activation!r}")
    images = shape[0] if len(shape) > 2 else 1
    rows = math.prod(shape[1:-1]) if len(shape) > 2 else shape[0]
    dense = (rows * channels if len(shape) > 2 else 0, channels)
    d = _lib.GroupNormDesc()
    d.images, d.rows, d.channels, d.groups, d.eps = images, rows, channels, groups, eps
    d.act, d.dtype = _ACTIVATIONS[activation], _DTYPES[dtype]
    at = _image_rows(shape, x_stride)
    d.x_image_stride, d.x_row_stride = at or dense
    g_at = dense if g_stride is None else _image_rows(shape, g_stride)
    d.g_image_stride, d.g_row_stride = g_at or dense
    nbytes = _lib.load().rdv_group_norm_workspace_bytes(C.byref(d), 0 if g_stride is None else 1)
    if nbytes < 0:
        _lib.check(int(nbytes), "group_norm")
    return d, at is None, g_at is None, nbytes


def _norm_param(p, x, what: str):
    if p is None:
        return None
    p = _tensor(p, what)
    assert p.dim() == 1 and p.shape[0] == x.shape[-1], f"{what} must be [channels]"
    if p.dtype != torch.float32:
        raise TypeError(f"{what} must be float32, got {p.dtype}")
    return p.contiguous()


def _norm_inputs(x, weight, bias):
    x = _data(x, "x")
    assert x.dim() >= 2, "x must be [rows, channels] (one image) or [images, ..., channels]"
    return x, _norm_param(weight, x, "weight"), _norm_param(bias, x, "bias")


def _group_norm_into(plan, x, weight, bias, y, stats, device: int) -> None:
    """Launches rdv_group_norm into y and stats (or None)."""
    d, copy, _, nbytes = plan
    if copy:
        x = x.contiguous()
    ws = torch.empty(nbytes, dtype=torch.uint8, device=x.device) if nbytes else None
    _check(_lib.load().rdv_group_norm(C.byref(d), x.data_ptr(), _ptr(weight), _ptr(bias), y.data_ptr(), _ptr(stats),
                                      _ptr(ws), nbytes, _stream(device)), "group_norm")


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
    x, weight, bias = _norm_inputs(x, weight, bias)
    device = _gpu_index()
    plan = _norm_plan(x.shape, x.stride(), None, x.dtype, int(groups), float(eps), activation, device)
    _on_gpu(device, x, "x", weight, "weight", bias, "bias")
    y = _like_out(out, x)
    if out is not None:
        _apart(y, (x, "x"), (weight, "weight"), (bias, "bias"))
    stats = None
    if return_stats:
        stats = torch.empty((plan[0].images, plan[0].groups, 2), dtype=torch.float32, device=x.device)
    with launch_scope():
        _group_norm_into(plan, x, weight, bias, y, stats, device)
    return (y, stats) if return_stats else y


def group_norm_backward(grad, x, weight, bias, groups: int, stats, activation: str = "none", grads=None):
    """(dx, dweight, dbias) of group_norm for grad = dL/dy, given the stats it
    returned for the same x, weight, bias, groups and activation.  dx is like
    x, dweight and dbias are float32 [channels]; `grads` supplies the three
    buffers."""
    x, weight, bias = _norm_inputs(x, weight, bias)
    grad = _like(grad, x, "grad")
    device = _gpu_index()
    d, copy_x, copy_g, nbytes = _norm_plan(x.shape, x.stride(), grad.stride(), x.dtype, int(groups), 0.0, activation,
                                           device)
    stats = _tensor(stats, "stats")
    assert tuple(stats.shape) == (d.images, d.groups, 2) and stats.is_contiguous(), \
        f"stats must be a contiguous [{d.images}, {d.groups}, 2] tensor, as group_norm returns it"
    if stats.dtype != torch.float32:
        raise TypeError(f"stats must be float32, got {stats.dtype}")
    _on_gpu(device, x, "x", grad, "grad", weight, "weight", bias, "bias", stats, "stats")
    param = weight if weight is not None else bias
    if param is None:
        param = torch.empty(d.channels, dtype=torch.float32, device=x.device)
    dx, dw, db = _grad_tensors(grads, (x, param, param), ("dx", "dweight", "dbias"))
    if grads is not None:
        for t in (dx, dw, db):
            _apart(t, (x, "x"), (grad, "grad"), (weight, "weight"), (bias, "bias"), (stats, "stats"))
    with launch_scope():
        if copy_x:
            x = x.contiguous()
        if copy_g:
            grad = grad.contiguous()
        ws = torch.empty(nbytes, dtype=torch.uint8, device=x.device) if nbytes else None
        _check(_lib.load().rdv_group_norm_backward(C.byref(d), grad.data_ptr(), x.data_ptr(), _ptr(weight), _ptr(bias),
                                                   stats.data_ptr(), dx.data_ptr(), dw.data_ptr(), db.data_ptr(),
                                                   _ptr(ws), nbytes, _stream(device)), "group_norm_backward")
    return dx, dw, db


# ------------------------------------------------------------ cross attention


def _rows_in_place(t: torch.Tensor) -> torch.Tensor:
    """t [batch, length, heads, dim] as the library reads it: the innermost dimension contiguous and, as rows whose
    strides are multiples of 16 bytes are read in pieces of that size, such a tensor itself aligned to it."""
    if t.stride(-1) != 1 and t.shape[-1] != 1:
        t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.contiguous_format)


@functools.lru_cache(maxsize=4096)
def _attention_plan(q_shape, k_shape, v_shape, q_stride, k_stride, v_stride, g_stride, mask_stride, dtype, scale, device):
    """What a call on tensors of this layout needs, by layout alone: (descriptor, workspace bytes).  g_stride is None
    for the forward call; `device` is the GPU it is planned for."""
    assert len(q_shape) == 4, "q must be [batch, queries, heads, dim]"
    assert len(k_shape) == 4 and k_shape == v_shape, "k and v must both be [batch, keys, kv_heads, dim]"
    b, lq, hq, dim = q_shape
    _, lk, hkv, k_dim = k_shape
    assert k_shape[0] == b, f"q has a batch of {b}, k and v of {k_shape[0]}"
    assert k_dim == dim, f"q has heads of {dim} dimensions, k and v of {k_dim}"
    assert hkv >= 1 and hq >= 1 and hq % hkv == 0, f"kv_heads ({hkv}) must divide heads ({hq})"
    scale = 1.0 / math.sqrt(dim) if scale is None else scale
    if not math.isfinite(scale):
        raise ValueError(f"scale must be finite, got {scale}")
    d = _lib.AttentionDesc()
    d.batch, d.queries, d.keys, d.heads, d.kv_heads, d.dim = b, lq, lk, hq, hkv, dim
    d.dtype, d.scale, d.mask_stride = _DTYPES[dtype], scale, mask_stride
    d.q_stride[:], d.k_stride[:], d.v_stride[:] = q_stride[:3], k_stride[:3], v_stride[:3]
    if g_stride is not None:
        d.g_stride[:] = g_stride[:3]
    nbytes = _lib.load().rdv_cross_attention_workspace_bytes(C.byref(d), 0 if g_stride is None else 1)
    if nbytes < 0:
        _lib.check(int(nbytes), "cross_attention")
    return d, nbytes


def _attention_inputs(q, k, v, key_lengths, key_mask, scale, grad=None):
    """The checked inputs as the library reads them, and the plan."""
    q, k, v = _data(q, "q"), _data(k, "k"), _data(v, "v")
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError(f"q, k and v must have one type, got {q.dtype}, {k.dtype} and {v.dtype}")
    if q.dim() == k.dim() == v.dim() == 4:  # else the plan refuses
        q, k, v = _rows_in_place(q), _rows_in_place(k), _rows_in_place(v)
    if grad is not None:
        grad = _rows_in_place(_like(grad, q, "grad"))
    mask_stride = 0
    if key_mask is not None:
        key_mask = _tensor(key_mask, "key_mask")
        assert key_mask.dim() == 2 and k.dim() == 4 and key_mask.shape == k.shape[:2], "key_mask must be [batch, keys]"
        if key_mask.dtype != torch.bool:
            raise TypeError(f"key_mask must be bool, got {key_mask.dtype}")
        if key_mask.stride(1) != 1:
            key_mask = key_mask.contiguous()
        mask_stride = key_mask.stride(0)
    device = _gpu_index()
    plan = _attention_plan(q.shape, k.shape, v.shape, q.stride(), k.stride(), v.stride(),
                           None if grad is None else grad.stride(), mask_stride, q.dtype,
                           None if scale is None else float(scale), device)
    if key_lengths is not None:
        key_lengths = _tensor(key_lengths, "key_lengths")
        assert tuple(key_lengths.shape) == (q.shape[0],), f"key_lengths must be [batch] = [{q.shape[0]}]"
        if key_lengths.dtype not in (torch.int32, torch.int64):
            raise TypeError(f"key_lengths must be int32 or int64, got {key_lengths.dtype}")
    _on_gpu(device, q, "q", k, "k", v, "v", key_lengths, "key_lengths", key_mask, "key_mask", grad, "grad")
    if key_lengths is not None:
        if key_lengths.dtype == torch.int64:
            key_lengths = key_lengths.clamp(0, k.shape[1]).to(torch.int32)
        key_lengths = key_lengths.contiguous()
    return q, k, v, key_lengths, key_mask, grad, plan, device


def _cross_attention_into(plan, q, k, v, key_lengths, key_mask, out, lse, device: int) -> None:
    """Launches rdv_cross_attention into out and lse (or None)."""
    d, nbytes = plan
    ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device) if nbytes else None
    _check(_lib.load().rdv_cross_attention(C.byref(d), q.data_ptr(), k.data_ptr(), v.data_ptr(), _ptr(key_lengths),
                                           _ptr(key_mask), out.data_ptr(), _ptr(lse), _ptr(ws), nbytes,
                                           _stream(device)), "cross_attention")


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
    given = q, k, v
    q, k, v, key_lengths, key_mask, _, plan, device = _attention_inputs(q, k, v, key_lengths, key_mask, scale)
    y = _like_out(out, q)
    if out is not None:
        _apart(y, (_tensor(given[0], "q"), "q"), (_tensor(given[1], "k"), "k"), (_tensor(given[2], "v"), "v"),
               (key_lengths, "key_lengths"), (key_mask, "key_mask"))
    lse = None
    if return_lse:
        d = plan[0]
        lse = torch.empty((d.batch, d.heads, d.queries), dtype=torch.float32, device=q.device)
    with launch_scope():
        _cross_attention_into(plan, q, k, v, key_lengths, key_mask, y, lse, device)
    return (y, lse) if return_lse else y


def cross_attention_backward(grad, q, k, v, out, lse, key_lengths=None, key_mask=None, scale: float | None = None,
                             grads=None):
    """(dq, dk, dv) of cross_attention for grad = dL/dout, given the out and lse
    it returned for the same arguments.  dk and dv are summed over the heads
    that share a state head and are 0 at states that do not count; `grads`
    supplies the three buffers.  float16 and bfloat16 inputs: the matrix cores
    take softmax terms and the scores' gradients rounded to that type, and each
    row's sum of grad * out is of `out` as it was rounded."""
    q, k, v, key_lengths, key_mask, grad, (d, nbytes), device = _attention_inputs(q, k, v, key_lengths, key_mask, scale,
                                                                                  grad)
    out = _like(out, q, "out").contiguous()
    lse = _tensor(lse, "lse")
    assert tuple(lse.shape) == (d.batch, d.heads, d.queries) and lse.is_contiguous(), \
        f"lse must be a contiguous [{d.batch}, {d.heads}, {d.queries}] tensor, as cross_attention returns it"
    if lse.dtype != torch.float32:
        raise TypeError(f"lse must be float32, got {lse.dtype}")
    _on_gpu(device, out, "out", lse, "lse")
    given = grads is not None
    dq, dk, dv = _grad_tensors(grads, (q, k, v), ("dq", "dk", "dv"))
    if given:
        for t in (dq, dk, dv):
            _apart(t, (grad, "grad"), (q, "q"), (k, "k"), (v, "v"), (out, "out"), (lse, "lse"),
                   (key_lengths, "key_lengths"), (key_mask, "key_mask"))
    with launch_scope():
        ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device) if nbytes else None
        _check(_lib.load().rdv_cross_attention_backward(C.byref(d), grad.data_ptr(), q.data_ptr(), k.data_ptr(),
                                                        v.data_ptr(), out.data_ptr(), lse.data_ptr(),
                                                        _ptr(key_lengths), _ptr(key_mask), dq.data_ptr(),
                                                        dk.data_ptr(), dv.data_ptr(), _ptr(ws), nbytes,
                                                        _stream(device)), "cross_attention_backward")
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


def _dropout_into(x, p, seed, subsequence, residual, y, device: int) -> None:
    """Launches rdv_dropout into y."""
    x = x.contiguous()
    residual = None if residual is None else residual.contiguous()
    _check(_lib.load().rdv_dropout(x.data_ptr(), _ptr(residual), y.data_ptr(), x.numel(), _DTYPES[x.dtype], p, seed,
                                   subsequence, _stream(device)), "dropout")


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
    device = _gpu_index()
    _on_gpu(device, x, "x", residual, "residual")
    y = _like_out(out, x, aligned=False)
    if out is not None:
        for t, what in ((x, "x"), (residual, "residual")):
            if t is not None and not (t.data_ptr() == y.data_ptr() and t.is_contiguous()):
                _apart(y, (t, what))
    with launch_scope():
        _dropout_into(x, p, seed, subsequence, residual, y, device)
    return y


def dropout_backward(grad, p: float, seed: int, subsequence: int = 0, out=None):
    """The gradient of x of dropout(x, p, seed, subsequence): grad * keep / (1 - p)
    with the same mask.  (The residual's gradient is grad itself.)"""
    return dropout(grad, p, seed, subsequence, out=out)
