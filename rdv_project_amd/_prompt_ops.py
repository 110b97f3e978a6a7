"""Operators of a prompt's encoder, whose states cross_attention reads, through the
C ABI (rdv_embedding, rdv_rms_norm, rdv_causal_attention and the backward
calls).  Build-defined: the reference has no counterpart.

The functions take GPU tensors (torch tensors or RDVObjects) of float32,
float16 or bfloat16, read strided views in place where the innermost dimension
is contiguous (any other layout is copied first), return fresh contiguous
tensors unless the caller passes buffers, and launch on torch's current stream.
Gradients are explicit calls, as mse_backward's are.  The TensorOperation forms
are in nn.py.  There is no CPU path."""
from __future__ import annotations

import ctypes as C
import functools
import math
import threading
from typing import NamedTuple, Optional

import torch

from . import _lib
from ._image_ops import (_DTYPES, _apart, _check, _data, _gpu_index, _grad_tensors, _image_rows, _like, _like_out,
                         _on_gpu, _out_tensor, _ptr, _rows_in_place, _stream, _tensor)
from .core import launch_scope


def _workspace(nbytes: int, like: torch.Tensor):
    return torch.empty(nbytes, dtype=torch.uint8, device=like.device) if nbytes else None


def _bytes(n: int, what: str) -> int:
    if n < 0:
        _lib.check(int(n), what)
    return n


def _row_stride(shape, stride):
    """The distance of the rows of a tensor [..., width], or None where they do not lie at one distance with contiguous
    elements."""
    at = _image_rows((1, *shape), (0, *stride))
    return None if at is None else at[1]


def _same_or_apart(out, *inputs) -> None:
    """out is one of the tensors itself, element for element, or shares no memory with it."""
    for t, what in inputs:
        if t is not None and not (t.data_ptr() == out.data_ptr() and t.is_contiguous() and t.dtype == out.dtype):
            _apart(out, (t, what))


# ------------------------------------------------------------ embedding


def _tokens(tokens) -> torch.Tensor:
    tokens = _tensor(tokens, "tokens")
    if tokens.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"tokens must be int32 or int64, got {tokens.dtype}")
    return tokens


@functools.lru_cache(maxsize=4096)
def _embedding_plan(n, wide, vocab, dim, dtype, scale, w_stride, g_stride, device):
    """What a call of this kind needs, by layout alone: (reference to the descriptor, workspace bytes); g_stride is None
    for the forward call, `device` the GPU it is planned for."""
    if not math.isfinite(scale):
        raise ValueError(f"scale must be finite, got {scale}")
    d = _lib.EmbeddingDesc()
    d.tokens, d.vocab, d.dim, d.dtype, d.wide_tokens, d.scale = n, vocab, dim, _DTYPES[dtype], wide, scale
    d.w_row_stride, d.g_row_stride = w_stride or 0, g_stride or 0
    nbytes = 0 if g_stride is None else _bytes(_lib.load().rdv_embedding_workspace_bytes(C.byref(d)), "embedding")
    return C.byref(d), nbytes


def _embedding_into(tokens, weight, scale: float, y, device: int) -> None:
    """Launches rdv_embedding into y."""
    tokens = tokens.contiguous()
    vocab, dim = weight.shape
    if weight.stride(1) != 1 and dim != 1:
        weight = weight.contiguous()
    d, _ = _embedding_plan(tokens.numel(), tokens.dtype == torch.int64, vocab, dim, weight.dtype, scale,
                           weight.stride(0), None, device)
    _check(_lib.load().rdv_embedding(d, tokens.data_ptr(), weight.data_ptr(), y.data_ptr(), _stream(device)), "embedding")


def _embedding_inputs(tokens, weight):
    tokens, weight = _tokens(tokens), _data(weight, "weight")
    assert weight.dim() == 2 and min(weight.shape) >= 1, "weight must be [vocab, dim]"
    return tokens, weight


def embedding(tokens, weight, scale: float = 1.0, out=None):
    """scale * weight[token] for tokens of any shape (int32 or int64) from weight
    [vocab, dim]; a token outside [0, vocab), -1 for padding say, gives a row of
    zeros.  Returns [*tokens.shape, dim] in weight's type."""
    tokens, weight = _embedding_inputs(tokens, weight)
    device = _gpu_index()
    _on_gpu(device, tokens, "tokens", weight, "weight")
    if out is None:
        y = weight.new_empty((*tokens.shape, weight.shape[1]))
    else:
        y = _out_tensor(out, (*tokens.shape, weight.shape[1]), weight.dtype, weight.device, aligned=False)
        _apart(y, (tokens, "tokens"), (weight, "weight"))
    with launch_scope():
        _embedding_into(tokens, weight, float(scale), y, device)
    return y


def embedding_backward(grad, tokens, vocab: int, scale: float = 1.0, out=None):
    """The gradient of weight of embedding(tokens, weight, scale) for grad =
    dL/dy [*tokens.shape, dim]: [vocab, dim] in grad's type, row v scale times the
    sum of the rows of grad whose token is v, in float32 (partial sums of very
    frequent tokens in float64) and rounded once; zeros for tokens that do not
    occur.  The order of a sum follows from the tokens alone, so the same call
    gives the same bits."""
    grad, tokens = _data(grad, "grad"), _tokens(tokens)
    assert grad.dim() == tokens.dim() + 1 and grad.shape[:-1] == tokens.shape and grad.shape[-1] >= 1, \
        f"grad must be [{', '.join(map(str, tokens.shape))}, dim], got {list(grad.shape)}"
    vocab, dim = int(vocab), grad.shape[-1]
    stride = dim if grad.is_contiguous() else _row_stride(grad.shape, grad.stride())
    device = _gpu_index()
    d, nbytes = _embedding_plan(tokens.numel(), tokens.dtype == torch.int64, vocab, dim, grad.dtype, float(scale), None,
                                dim if stride is None else stride, device)
    _on_gpu(device, grad, "grad", tokens, "tokens")
    if out is None:
        dw = grad.new_empty((vocab, dim))
    else:
        dw = _out_tensor(out, (vocab, dim), grad.dtype, grad.device, aligned=False)
        _apart(dw, (grad, "grad"), (tokens, "tokens"))
    with launch_scope():
        if stride is None:
            grad = grad.contiguous()
        tokens = tokens.contiguous()
        ws = _workspace(nbytes, grad)
        _check(_lib.load().rdv_embedding_backward(d, grad.data_ptr(), tokens.data_ptr(), dw.data_ptr(), _ptr(ws),
                                                  nbytes, _stream(device)), "embedding_backward")
    return dw


# ------------------------------------------------------------ root-mean-square normalisation


@functools.lru_cache(maxsize=4096)
def _rms_plan(shape, dtype, eps, strides, backward, device):
    """What a call on rows [..., width] of these layouts needs, by layout alone: (reference to the descriptor, whether each
    tensor has to be copied first, workspace bytes).  strides: of x and residual, or of h, grad and grad_sum (None where
    there is none); `device`: the GPU it is planned for."""
    width = shape[-1]
    assert width >= 1, "x must be [..., width]"
    d = _lib.RmsNormDesc()
    d.rows, d.width, d.dtype, d.eps = math.prod(shape[:-1]), width, _DTYPES[dtype], eps
    at = [0 if s is None else _row_stride(shape, s) for s in strides]
    copies = [a is None for a in at]
    at = [width if a is None else a for a in at]
    if not backward:
        d.x_row_stride, d.r_row_stride = at
        return C.byref(d), copies, 0
    d.x_row_stride, d.g_row_stride, d.s_row_stride = at
    return C.byref(d), copies, _bytes(_lib.load().rdv_rms_norm_workspace_bytes(C.byref(d)), "rms_norm")


def _rms_param(p, x):
    if p is None:
        return None
    p = _tensor(p, "weight")
    assert p.dim() == 1 and p.shape[0] == x.shape[-1], "weight must be [width]"
    if p.dtype != torch.float32:
        raise TypeError(f"weight must be float32, got {p.dtype}")
    return p.contiguous()


def _rms_inputs(x, weight):
    x = _data(x, "x")
    assert x.dim() >= 1, "x must be [..., width]"
    return x, _rms_param(weight, x)


def _rms_norm_into(x, weight, residual, eps: float, y, h, scales, stats, device: int) -> None:
    """Launches rdv_rms_norm into y, and into h, scales and stats (or None)."""
    d, copies, _ = _rms_plan(x.shape, x.dtype, eps, (x.stride(), None if residual is None else residual.stride()), False,
                             device)
    if copies[0]:
        x = x.contiguous()
    if copies[1]:
        residual = residual.contiguous()
    _check(_lib.load().rdv_rms_norm(d, x.data_ptr(), _ptr(residual), _ptr(weight), _ptr(h), y.data_ptr(), _ptr(scales),
                                    _ptr(stats), _stream(device)), "rms_norm")


def rms_norm(x, weight, residual=None, eps: float = 1e-6, out=None, sum_out=None, return_stats: bool = False,
             eight_bits: bool = False):
    """weight * h / sqrt(mean(h^2) + eps) over the rows of x [..., width], where h
    is x, or x + residual (a tensor like x) as it is stored; weight: float32
    [width] or None.

    Returns y like x; (y, h) with residual; and with return_stats also stats [...]
    = 1 / sqrt(mean(h^2) + eps) in float32, which rms_norm_backward takes.
    `sum_out` is h's buffer, which may be x or residual itself; `out` is y's, which
    may be x itself where there is no residual.  eight_bits: in y's place stands
    (values, scales), float8_e4m3fn [..., width] and float32 [...], for products in
    8 bits: y is scales times values, scales = max |y| / 448 of the row, NaN where a
    y is (`out`: the two buffers)."""
    x, weight = _rms_inputs(x, weight)
    eps = float(eps)
    if not 0.0 <= eps < math.inf:
        raise ValueError(f"eps must be finite and >= 0, got {eps}")
    if residual is not None:
        residual = _like(residual, x, "residual")
    elif sum_out is not None:
        raise TypeError("sum_out is for a call with a residual")
    device = _gpu_index()
    _on_gpu(device, x, "x", residual, "residual", weight, "weight")
    rows, dev = x.shape[:-1], x.device
    inputs = (x, "x"), (residual, "residual")
    scales = None
    if eight_bits:
        if out is not None and (not isinstance(out, (list, tuple)) or len(out) != 2):
            raise TypeError("out must be (values, scales)")
        values, scales = out if out is not None else (None, None)
        y = _out_tensor(values, x.shape, torch.float8_e4m3fn, dev, "values", aligned=False)
        scales = _out_tensor(scales, rows, torch.float32, dev, "scales", aligned=False)
        if out is not None:
            _apart(y, *inputs, (weight, "weight"))
            _apart(scales, *inputs, (weight, "weight"), (y, "values"))
    else:
        y = _like_out(out, x, aligned=False)
        if out is not None:
            (_same_or_apart if residual is None else _apart)(y, inputs[0])
            _apart(y, inputs[1], (weight, "weight"))
    h = None
    if residual is not None:
        if sum_out is None:
            h = _like_out(None, x)
        else:
            h = _out_tensor(sum_out, x.shape, x.dtype, dev, "sum_out", aligned=False)
            _same_or_apart(h, *inputs)
            _apart(h, (weight, "weight"), (y, "out"), (scales, "scales"))
    stats = torch.empty(rows, dtype=torch.float32, device=dev) if return_stats else None
    with launch_scope():
        _rms_norm_into(x, weight, residual, eps, y, h, scales, stats, device)
    result = ((y, scales) if eight_bits else y,) + (() if h is None else (h,)) + ((stats,) if return_stats else ())
    return result[0] if len(result) == 1 else result


def rms_norm_backward(grad, h, weight, stats, grad_sum=None, grads=None):
    """(dx, dweight) of rms_norm for grad = dL/dy, and with a residual grad_sum =
    dL/dh of what else reads h; h is x, or the sum that the call returned, and
    stats what it returned with return_stats.  dx is the gradient of x and, where
    there was one, of residual alike; dweight is float32 [width]; `grads` supplies
    the two buffers."""
    h, weight = _rms_inputs(h, weight)
    grad = _like(grad, h, "grad")
    if grad_sum is not None:
        grad_sum = _like(grad_sum, h, "grad_sum")
    stats = _tensor(stats, "stats")
    assert stats.shape == h.shape[:-1] and stats.is_contiguous(), \
        f"stats must be a contiguous {list(h.shape[:-1])} tensor, as rms_norm returns it"
    if stats.dtype != torch.float32:
        raise TypeError(f"stats must be float32, got {stats.dtype}")
    device = _gpu_index()
    _on_gpu(device, h, "h", grad, "grad", weight, "weight", stats, "stats", grad_sum, "grad_sum")
    if grads is None:
        dx = _like_out(None, h)
        dw = torch.empty(h.shape[-1], dtype=torch.float32, device=h.device)
    else:
        if not isinstance(grads, (list, tuple)) or len(grads) != 2:
            raise TypeError("grads must be (dx, dweight)")
        dx = _out_tensor(grads[0], h.shape, h.dtype, h.device, "dx", aligned=False)
        dw = _out_tensor(grads[1], (h.shape[-1],), torch.float32, h.device, "dweight", aligned=False)
        for t in (dx, dw):
            _apart(t, (grad, "grad"), (h, "h"), (weight, "weight"), (stats, "stats"), (grad_sum, "grad_sum"))
        _apart(dw, (dx, "dx"))
    with launch_scope():
        d, copies, nbytes = _rms_plan(h.shape, h.dtype, 0.0, (h.stride(), grad.stride(),
                                                              None if grad_sum is None else grad_sum.stride()), True, device)
        if any(copies):
            h, grad, grad_sum = (t.contiguous() if c else t for t, c in zip((h, grad, grad_sum), copies))
        ws = _workspace(nbytes, h)
        _check(_lib.load().rdv_rms_norm_backward(d, grad.data_ptr(), _ptr(grad_sum), h.data_ptr(), _ptr(weight),
                                                 stats.data_ptr(), dx.data_ptr(), dw.data_ptr(), _ptr(ws), nbytes,
                                                 _stream(device)), "rms_norm_backward")
    return dx, dw


# ------------------------------------------------------------ causal attention


_CAPTURED: list = []  # lists of work that graphs read
_CAPTURED_LOCK = threading.Lock()


class PackedSequences:
    """Sequences packed one after the other, for causal_attention: sequence s is
    lengths[s] rows of q, after those of the sequences before it, and states[s] rows
    of k and v (as many where states is None: whole prompts).  More states than
    tokens: the next tokens of a sequence whose earlier states are there, single
    ones among them; fewer: its first tokens see nothing.  starts[s] is the row of
    k and v where the sequence's states begin, for states that lie in the slots of
    a cache, say (None: one after the other).

    It holds the lists of work that the kernels take, made on the host at the first
    call of each kind (heads, dimensions, type, direction) on each GPU and copied
    there: keep it for all layers and steps on sequences of these lengths.  That
    first call waits for the copy, and cannot be captured into a graph.  Lists that a
    graph has captured are kept, also when the PackedSequences is gone, until
    release() or the end of the process: nothing tells when a graph is."""

    def __init__(self, lengths, states=None, starts=None) -> None:
        self.lengths = _counts(lengths, "lengths")
        self.states = self.lengths if states is None else _counts(states, "states")
        if len(self.states) != len(self.lengths):
            raise ValueError(f"{len(self.lengths)} lengths, but {len(self.states)} states")
        token, state, rows = 0, 0, []
        self.starts = None if starts is None else _counts(starts, "starts")
        if self.starts is not None and len(self.starts) != len(self.lengths):
            raise ValueError(f"{len(self.lengths)} lengths, but {len(self.starts)} starts")
        for i, (t, s) in enumerate(zip(self.lengths, self.states)):
            at = state if self.starts is None else self.starts[i]
            rows.append((token, t, at, s))
            token, state = token + t, state + s
        #: rows of q, and of k and v, that the sequences take
        self.tokens, self.total_states = token, max((r[2] + r[3] for r in rows), default=0)
        spans = sorted((r[2], r[2] + r[3]) for r in rows if r[3])
        #: whether no two sequences share states, which gradients need
        self.apart = all(a[1] <= b[0] for a, b in zip(spans, spans[1:]))
        #: whether the sequences' states are all rows up to the last one's
        self.dense = sum(b - a for a, b in spans) == self.total_states if self.apart else False
        self._rows = (C.c_int64 * max(1, 4 * len(rows)))(*[x for r in rows for x in r])
        self._plans: dict = {}
        self._calls: dict = {}

    def __len__(self) -> int:
        return len(self.lengths)

    def _plan(self, d, backward: bool, device: int):
        """(the list of work in host memory, the same on the GPU, the stream that it was allocated on) for calls of this
        kind."""
        key = d.heads, d.kv_heads, d.dim, d.dtype, backward, device
        hit = self._plans.get(key)
        if hit is not None:
            return hit
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("the first call of a kind on PackedSequences cannot be captured: make it once before")
        lib, n = _lib.load(), len(self.lengths)
        nbytes = _bytes(lib.rdv_causal_attention_plan_bytes(C.byref(d), self._rows, n, backward), "causal_attention")
        host = torch.empty(nbytes, dtype=torch.uint8)
        _check(lib.rdv_causal_attention_plan(C.byref(d), self._rows, n, backward, host.data_ptr(), nbytes),
               "causal_attention")
        lists = host.to(f"cuda:{device}")  # a synchronous copy: any stream may read it
        return self._plans.setdefault(key, (host, lists, _stream(device)))  # another thread may have been first

    def _call(self, layout, device: int):
        """What a call on tensors of this layout (_causal_desc's arguments) needs: (descriptor, reference to it, list of
        work in host memory, on the GPU, workspace bytes)."""
        hit = self._calls.get((layout, device))
        if hit is None:
            hit = self._plan_call(layout, device)
        # The list's memory outlives what reads it: the launches of streams other than its own, and a graph's replays.
        if hit[5] != _stream(device):
            hit[3].record_stream(torch.cuda.current_stream())
        if torch.cuda.is_current_stream_capturing():
            with _CAPTURED_LOCK:
                if not any(hit[3] is t for t in _CAPTURED):
                    _CAPTURED.append(hit[3])
        return hit[:5]

    def release(self) -> None:
        """Lets go of the lists that graphs have captured: to be called when every replay of those graphs has run and
        none follows.  Eager calls and new graphs can go on using the sequences."""
        mine = [lists for _, lists, _ in list(self._plans.values())]
        with _CAPTURED_LOCK:
            _CAPTURED[:] = [t for t in _CAPTURED if not any(t is m for m in mine)]

    def _plan_call(self, layout, device: int):
        d = _causal_desc(*layout)
        assert self.tokens <= d.tokens, f"the sequences have {self.tokens} tokens, q {d.tokens} rows"
        assert self.total_states <= d.states, f"the sequences have {self.total_states} states, k and v {d.states} rows"
        backward = layout[6] is not None
        host, lists, stream = self._plan(d, backward, device)
        nbytes = _bytes(_lib.load().rdv_causal_attention_workspace_bytes(C.byref(d), host.data_ptr(), backward),
                        "causal_attention")
        if len(self._calls) >= 256:  # of changing strides or scales: their plans stay
            self._calls.clear()
        hit = self._calls[layout, device] = d, C.byref(d), host, lists, nbytes, stream
        return hit


class AttentionStats(NamedTuple):
    """What causal_attention_backward takes from the forward call beside its result."""
    #: [heads, tokens] float32, the logarithm of each softmax's denominator (-inf where nothing is seen)
    lse: torch.Tensor
    #: like out, what rounding it to a 16-bit type left; None for float32
    rest: Optional[torch.Tensor]


def _counts(values, what: str) -> tuple:
    try:
        values = tuple(values.tolist() if isinstance(values, torch.Tensor) else values)
        if any(not 0 <= v < 1 << 31 or int(v) != v for v in values):  # NaN and infinities too
            raise ValueError(f"{what} must be whole numbers in [0, 2^31)")
        return tuple(int(v) for v in values)
    except TypeError:
        raise TypeError(f"{what} must be whole numbers, one per sequence") from None


def _causal_desc(q_shape, k_shape, v_shape, q_stride, k_stride, v_stride, g_stride, dtype, scale):
    """The descriptor of a call on tensors of this layout; g_stride is None for the forward call."""
    assert len(q_shape) == 3, "q must be [tokens, heads, dim]"
    assert len(k_shape) == 3 and k_shape == v_shape, "k and v must both be [states, kv_heads, dim]"
    tokens, hq, dim = q_shape
    states, hkv, k_dim = k_shape
    assert k_dim == dim, f"q has heads of {dim} dimensions, k and v of {k_dim}"
    assert hkv >= 1 and hq >= 1 and hq % hkv == 0, f"kv_heads ({hkv}) must divide heads ({hq})"
    assert dim >= 1, "dim must be >= 1"
    if dim > _lib.ATTENTION_MAX_DIM:
        raise NotImplementedError(f"dim must be at most {_lib.ATTENTION_MAX_DIM}, got {dim}")
    scale = 1.0 / math.sqrt(dim) if scale is None else scale
    if not math.isfinite(scale):
        raise ValueError(f"scale must be finite, got {scale}")
    d = _lib.CausalAttentionDesc()
    d.tokens, d.states, d.heads, d.kv_heads, d.dim = tokens, states, hq, hkv, dim
    d.dtype, d.scale = _DTYPES[dtype], scale
    d.q_stride[:], d.k_stride[:], d.v_stride[:] = q_stride[:2], k_stride[:2], v_stride[:2]
    if g_stride is not None:
        d.g_stride[:] = g_stride[:2]
    return d


def _causal_inputs(q, k, v, sequences, scale, grad=None):
    """The checked inputs as the library reads them, and what the call needs (PackedSequences._call)."""
    q, k, v = _data(q, "q"), _data(k, "k"), _data(v, "v")
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise TypeError(f"q, k and v must have one type, got {q.dtype}, {k.dtype} and {v.dtype}")
    if not isinstance(sequences, PackedSequences):
        raise TypeError(f"sequences must be PackedSequences, got {type(sequences).__name__}")
    if q.dim() == k.dim() == v.dim() == 3:  # else the descriptor refuses
        q, k, v = _rows_in_place(q), _rows_in_place(k), _rows_in_place(v)
    if grad is not None:
        grad = _rows_in_place(_like(grad, q, "grad"))
    layout = (q.shape, k.shape, v.shape, q.stride(), k.stride(), v.stride(), None if grad is None else grad.stride(),
              q.dtype, None if scale is None else float(scale))
    device = _gpu_index()
    if not q.is_cuda:
        _causal_desc(*layout)  # what is wrong with the call comes before where it is made
    _on_gpu(device, q, "q", k, "k", v, "v", grad, "grad")
    return q, k, v, grad, sequences._call(layout, device), device


def _causal_attention_into(call, q, k, v, out, lse, rest, device: int) -> None:
    """Launches rdv_causal_attention into out, and into lse and rest (or None)."""
    _, d, host, lists, nbytes = call
    ws = _workspace(nbytes, q)
    _check(_lib.load().rdv_causal_attention(d, host.data_ptr(), lists.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(),
                                            out.data_ptr(), _ptr(lse), _ptr(rest), _ptr(ws), nbytes, _stream(device)),
           "causal_attention")


def causal_attention(q, k, v, sequences: PackedSequences, scale: float | None = None, out=None,
                     return_lse: bool = False):
    """softmax(scale q k^T) v within packed sequences, from q [tokens, heads, dim] to
    k and v [states, kv_heads, dim] (views of one projection's output, say): of a
    sequence of T tokens and S states, token i sees the states j <= i + S - T; head
    h reads state head h // (heads // kv_heads); dim at most 128; scale defaults to
    1 / sqrt(dim).  What k and v hold at states that a token does not see has no
    effect on it, and a token that sees none gets 0.

    Returns out [tokens, heads, dim] and with return_lse also AttentionStats (lse,
    rest), which causal_attention_backward takes: lse [heads, tokens] float32, the
    logarithm of each softmax's denominator (-inf where nothing is seen), and rest,
    like out, what rounding out to a 16-bit type left (None for float32).  Rows
    behind the last sequence are left as they are in `out`, and are 0 (-inf) in
    fresh results.  float16 and bfloat16 inputs: the matrix cores take softmax terms
    rounded to that type; float32: float32 throughout."""
    given = q, k, v
    q, k, v, _, call, device = _causal_inputs(q, k, v, sequences, scale)
    d = call[0]
    y = _like_out(out, q)
    if out is not None:
        _apart(y, *zip((_tensor(t, n) for t, n in zip(given, "qkv")), "qkv"))
    elif sequences.tokens < d.tokens:
        y[sequences.tokens:].zero_()
    lse = rest = None
    if return_lse:
        lse = torch.empty((d.heads, d.tokens), dtype=torch.float32, device=q.device)
        rest = None if q.dtype == torch.float32 else _like_out(None, y)
        if sequences.tokens < d.tokens:
            lse[:, sequences.tokens:].fill_(-math.inf)
            if rest is not None:
                rest[sequences.tokens:].zero_()
    with launch_scope():
        _causal_attention_into(call, q, k, v, y, lse, rest, device)
    return (y, AttentionStats(lse, rest)) if return_lse else y


def causal_attention_backward(grad, q, k, v, out, stats, sequences: PackedSequences, scale: float | None = None,
                              grads=None):
    """(dq, dk, dv) of causal_attention for grad = dL/dout, given the out and stats
    that it returned for the same arguments with return_lse (stats may be lse alone:
    each row's sum of grad * out is then of `out` as it was rounded).  dk and dv are summed over the heads that
    share a state head and are 0 at states that no token sees; no two sequences may
    share states.  `grads` supplies the three buffers, whose rows that belong to no
    sequence are left as they are (0 in fresh ones).  float16 and bfloat16 inputs:
    the matrix cores take softmax terms and the scores' gradients rounded to that
    type."""
    if isinstance(sequences, PackedSequences) and not sequences.apart:
        raise NotImplementedError("gradients of sequences that share states")
    q, k, v, grad, call, device = _causal_inputs(q, k, v, sequences, scale, _tensor(grad, "grad"))
    d, desc, host, lists, nbytes = call
    out = _like(out, q, "out").contiguous()
    lse, rest = stats if isinstance(stats, (list, tuple)) and len(stats) == 2 else (stats, None)
    lse = _tensor(lse, "lse")
    if rest is not None:
        rest = _like(rest, q, "rest").contiguous()
    assert tuple(lse.shape) == (d.heads, d.tokens) and lse.is_contiguous(), \
        f"lse must be a contiguous [{d.heads}, {d.tokens}] tensor, as causal_attention returns it"
    if lse.dtype != torch.float32:
        raise TypeError(f"lse must be float32, got {lse.dtype}")
    _on_gpu(device, out, "out", lse, "lse", rest, "rest")
    given = grads is not None
    dq, dk, dv = _grad_tensors(grads, (q, k, v), ("dq", "dk", "dv"))
    if given:
        for t in (dq, dk, dv):
            _apart(t, (grad, "grad"), (q, "q"), (k, "k"), (v, "v"), (out, "out"), (lse, "lse"), (rest, "rest"))
    else:
        if sequences.tokens < d.tokens:
            dq[sequences.tokens:].zero_()
        if not sequences.dense or sequences.total_states < d.states:
            at = sequences.total_states if sequences.dense else 0
            dk[at:].zero_()
            dv[at:].zero_()
    with launch_scope():
        out = out if out.data_ptr() % 16 == 0 else out.clone()
        rest = rest if rest is None or rest.data_ptr() % 16 == 0 else rest.clone()
        ws = _workspace(nbytes, q)
        _check(_lib.load().rdv_causal_attention_backward(desc, host.data_ptr(), lists.data_ptr(), grad.data_ptr(),
                                                         q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
                                                         lse.data_ptr(), _ptr(rest), dq.data_ptr(), dk.data_ptr(),
                                                         dv.data_ptr(), _ptr(ws), nbytes, _stream(device)),
               "causal_attention_backward")
    return dq, dk, dv
