"""What the operators of a prompt's encoder refuse, and how; the lists of work that the library makes (CPU only, no
launches, but for the tests of buffers)."""
import ctypes as C
import itertools

import numpy as np
import pytest
import torch

import rdv_project_amd as rdv
from rdv_project_amd import _lib

T, W, G = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(10, 8), torch.zeros(2, 3, 8)
X, P = torch.zeros(5, 12), torch.ones(12)
Q, K, LSE = torch.zeros(7, 4, 8), torch.zeros(9, 2, 8), torch.zeros(4, 7)
S = rdv.PackedSequences((3, 4), (3, 6))


@pytest.mark.parametrize("call,error,text", [
    (lambda: rdv.embedding(T.float(), W), TypeError, "tokens must be int32"),
    (lambda: rdv.embedding(T, W[0]), AssertionError, "vocab, dim"),
    (lambda: rdv.embedding(T, W[:0]), AssertionError, "vocab, dim"),
    (lambda: rdv.embedding(T, W.int()), TypeError, "weight must be float32"),
    (lambda: rdv.embedding([1], W), TypeError, "torch tensor"),
    (lambda: rdv.embedding_backward(G[0], T, 10), AssertionError, "grad must be"),
    (lambda: rdv.embedding_backward(G, T[:1], 10), AssertionError, "grad must be"),
    (lambda: rdv.embedding_backward(G, T.short(), 10), TypeError, "tokens must be int32"),
    (lambda: rdv.embedding_backward(G, T, 0), AssertionError, "vocab and dim"),
    (lambda: rdv.embedding_backward(G, T, 1 << 26), NotImplementedError, "2\\^25"),
    (lambda: rdv.embedding_backward(G, T, 10, scale=float("inf")), ValueError, "finite"),
    (lambda: rdv.rms_norm(X.int(), P), TypeError, "x must be float32"),
    (lambda: rdv.rms_norm(X, P[:5]), AssertionError, "weight must be"),
    (lambda: rdv.rms_norm(X, P.half()), TypeError, "weight must be float32"),
    (lambda: rdv.rms_norm(X, P, residual=X[:2]), AssertionError, "residual must have"),
    (lambda: rdv.rms_norm(X, P, residual=X.half()), TypeError, "residual must be"),
    (lambda: rdv.rms_norm(X, P, sum_out=X), TypeError, "residual"),
    (lambda: rdv.rms_norm(X, P, eps=-1.0), ValueError, "eps"),
    (lambda: rdv.rms_norm(X, P, eps=float("nan")), ValueError, "eps"),
    (lambda: rdv.rms_norm_backward(X[:2], X, P, X[:, 0]), AssertionError, "grad must have"),
    (lambda: rdv.rms_norm_backward(X, X, P, X[:2, 0]), AssertionError, "stats must be"),
    (lambda: rdv.rms_norm_backward(X, X, P, X[:, 0]), AssertionError, "stats must be"),
    (lambda: rdv.rms_norm_backward(X, X, P, torch.zeros(5).half()), TypeError, "stats must be float32"),
    (lambda: rdv.rms_norm_backward(X, X, P, torch.zeros(5), grad_sum=X.half()), TypeError, "grad_sum"),
    (lambda: rdv.PackedSequences((1, -1)), ValueError, "lengths"),
    (lambda: rdv.PackedSequences((1.5,)), ValueError, "lengths"),
    (lambda: rdv.PackedSequences(4), TypeError, "lengths"),
    (lambda: rdv.PackedSequences((1 << 31,)), ValueError, "lengths"),
    (lambda: rdv.PackedSequences((1, 2), (3,)), ValueError, "states"),
    (lambda: rdv.PackedSequences((1, 2), (3, 4), (0,)), ValueError, "starts"),
    (lambda: rdv.causal_attention(Q[0], K, K, S), AssertionError, "q must be"),
    (lambda: rdv.causal_attention(Q, K, K[:5], S), AssertionError, "k and v"),
    (lambda: rdv.causal_attention(Q[..., :7], K, K, S), AssertionError, "dimensions"),
    (lambda: rdv.causal_attention(Q[:, :3], K, K, S), AssertionError, "kv_heads"),
    (lambda: rdv.causal_attention(Q.half(), K, K, S), TypeError, "one type"),
    (lambda: rdv.causal_attention(Q, K, K, (3, 4)), TypeError, "PackedSequences"),
    (lambda: rdv.causal_attention(Q, K, K, S, scale=float("nan")), ValueError, "finite"),
    (lambda: rdv.causal_attention(*[torch.zeros(7, 1, 129)] * 3, S), NotImplementedError, "at most 128"),
    (lambda: rdv.causal_attention_backward(Q, Q, K, K, Q, LSE, rdv.PackedSequences((3, 4), (5, 5), (0, 4))),
     NotImplementedError, "share states"),
    # no CPU path
    (lambda: rdv.embedding(T, W), TypeError, "GPU tensor"),
    (lambda: rdv.embedding_backward(G, T, 10), TypeError, "GPU tensor"),
    (lambda: rdv.rms_norm(X, P), TypeError, "GPU tensor"),
    (lambda: rdv.rms_norm_backward(X, X, P, torch.zeros(5)), TypeError, "GPU tensor"),
    (lambda: rdv.causal_attention(Q, K, K, S), TypeError, "GPU tensor"),
    (lambda: rdv.causal_attention_backward(Q, Q, K, K, Q, LSE, S), TypeError, "GPU tensor"),
])
def test_refusals(call, error, text):
    with pytest.raises(error, match=text):
        call()


def test_packed_sequences():
    s = rdv.PackedSequences(torch.tensor([3, 0, 2]), [5, 1, 0])
    assert (s.lengths, s.states, s.tokens, s.total_states, len(s)) == ((3, 0, 2), (5, 1, 0), 5, 6, 3)
    assert s.apart and s.dense
    assert rdv.PackedSequences((2, 2)).states == (2, 2)
    assert rdv.PackedSequences(()).tokens == 0
    s = rdv.PackedSequences((1, 1), (10, 10), (20, 0))
    assert s.apart and not s.dense and s.total_states == 30
    assert not rdv.PackedSequences((1, 1), (10, 10), (9, 0)).apart


def _desc(**kw):
    d = _lib.CausalAttentionDesc(tokens=7, states=9, heads=4, kv_heads=2, dim=64, dtype=_lib.DTYPE_F16, scale=1.0)
    for name, value in kw.items():
        setattr(d, name, value)
    return d


def _rows(*rows):
    return (C.c_int64 * max(1, 4 * len(rows)))(*itertools.chain(*rows))


@pytest.mark.parametrize("kw,code,text", [
    (dict(heads=3), -1, "divide"), (dict(kv_heads=0), -1, "divide"), (dict(heads=65536, kv_heads=1), -1, "65535"),
    (dict(dim=0), -1, "dim"), (dict(dim=129), -2, "at most 128"), (dict(tokens=-1), -1, "tokens"),
    (dict(states=1 << 31), -1, "states"), (dict(dtype=5), -1, "dtype"), (dict(scale=float("inf")), -1, "scale"),
    (dict(reserved=1), -1, "reserved"),
])
def test_library_refuses_causal_attention(kw, code, text):
    lib, d = _lib.load(), _desc(**kw)
    assert lib.rdv_causal_attention_plan_bytes(C.byref(d), _rows((0, 7, 0, 9)), 1, 0) == code and text in _lib.last_error()
    assert lib.rdv_causal_attention(C.byref(d), 16, 16, 16, 16, 16, 16, None, None, None, 0, None) == code


@pytest.mark.parametrize("row,code", [
    ((0, 8, 0, 9), -1), ((1, 7, 0, 9), -1), ((0, 7, 0, 10), -1), ((0, 7, 9, 1), -1), ((-1, 7, 0, 9), -1), ((0, -1, 0, 9), -1),
    ((0, 7, -1, 9), -1), ((0, 7, 0, -9), -1), ((1 << 62, 1 << 62, 0, 9), -1), ((0, 7, 0, 9), 0), ((7, 0, 9, 0), 0),
])
def test_library_refuses_sequences_out_of_range(row, code):
    lib, d = _lib.load(), _desc()
    got = lib.rdv_causal_attention_plan_bytes(C.byref(d), _rows(row), 1, 0)
    assert got == code or (code == 0 and got > 0)


def test_library_refuses_rows_past_32_bits():
    lib = _lib.load()
    d = _desc(tokens=1 << 20, states=1 << 20, heads=1 << 15, kv_heads=1)
    assert lib.rdv_causal_attention_plan_bytes(C.byref(d), _rows((0, 1 << 20, 0, 1 << 20)), 1, 0) == _lib.RDV_ERR_UNSUPPORTED
    assert "rows" in _lib.last_error()


def _plan(d, rows, backward):
    lib = _lib.load()
    n = lib.rdv_causal_attention_plan_bytes(C.byref(d), _rows(*rows), len(rows), backward)
    assert n > 0
    buffer = np.zeros(n + 64, np.uint8)
    assert lib.rdv_causal_attention_plan(C.byref(d), _rows(*rows), len(rows), backward, buffer.ctypes.data, n) == 0
    assert not buffer[n:].any()
    assert lib.rdv_causal_attention_plan(C.byref(d), _rows(*rows), len(rows), backward, buffer.ctypes.data, n - 1) == -1
    return buffer[:n]


def test_plans_are_checked():
    """A plan serves calls of its heads, dimensions, type and direction on at least its rows, and no others."""
    lib = _lib.load()
    plan = _plan(_desc(), [(0, 7, 0, 9)], 0)
    ok = lambda d, backward=0: lib.rdv_causal_attention_workspace_bytes(C.byref(d), plan.ctypes.data, backward)
    assert ok(_desc()) >= 0 and ok(_desc(tokens=100, states=100, scale=2.0)) >= 0
    for kw in (dict(heads=2), dict(kv_heads=4), dict(dim=32), dict(dtype=_lib.DTYPE_BF16), dict(tokens=6), dict(states=8)):
        assert ok(_desc(**kw)) == _lib.RDV_ERR_INVALID and "made for other" in _lib.last_error()
    assert ok(_desc(), 1) == _lib.RDV_ERR_INVALID
    plan[0] ^= 1
    assert ok(_desc()) == _lib.RDV_ERR_INVALID and "not a plan" in _lib.last_error()


def _items(plan):
    """(rows, states) lists of (token, tokens, state, states, tile, begin, end, slot) of a plan, and the joins."""
    words = plan[:256].view(np.int32)
    # the descriptor is found by its own size; what follows it are backward, cu, then the counts
    base = (16 + C.sizeof(_lib.CausalAttentionDesc)) // 4
    few, rows, keys, row_joins, key_joins = words[base + 2:base + 7]
    size = 8 * 4
    at = 256 if (base + 15) * 4 + 5 * 8 <= 256 else 512
    out = []
    for count in (few, rows, keys, row_joins, key_joins):
        out.append(plan[at:at + count * size].view(np.int32).reshape(-1, 8).tolist())
        at += -(-count * size // 256) * 256
    assert at == len(plan)
    return out


@pytest.mark.parametrize("dtype", [_lib.DTYPE_F32, _lib.DTYPE_F16])
@pytest.mark.parametrize("lengths,states,heads,kv_heads,dim", [
    ((5,), (5,), 2, 1, 64), ((700, 0, 1, 33), (700, 3, 1, 33), 4, 2, 64), ((4096,), (4096,), 8, 8, 128), ((9000, 5), (9000, 5), 1, 1, 40),
    ((1, 1, 1), (30000, 1, 0), 16, 4, 128), ((3, 100), (2000, 50), 3, 1, 32), ((2000,) * 9, (2500,) * 9, 6, 3, 96), ((1,) * 300, (1,) * 300, 2, 2, 16),
])
def test_lists_cover_the_work_once(dtype, lengths, states, heads, kv_heads, dim):
    """Every row of every tile goes over every state that it sees, and every state over every token that sees it, in
    exactly one part; parts have places of their own, and joins name them."""
    share = heads // kv_heads
    rows, t, s = [], 0, 0
    for a, b in zip(lengths, states):
        rows.append((t, a, s, b))
        t, s = t + a, s + b
    d = _desc(tokens=t, states=s, heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype)
    step = 64 if dtype != _lib.DTYPE_F32 or dim <= 64 else 32
    for backward in (0, 1):
        few, tiles, keys, row_joins, key_joins = _items(_plan(d, rows, backward))
        assert not (backward and few)
        for items, joins, by_state in ((few + tiles, row_joins, False), (keys, key_joins, True)):
            if by_state and not backward:
                assert not items
                continue
            parts = {}
            for i in items:
                parts.setdefault(tuple(i[:5]), []).append(i[5:])
            slots = sorted(i[7] for i in items if i[7] >= 0)
            assert slots == list(range(len(slots)))
            joined = {tuple(j[:5]): (j[5], j[6]) for j in joins}
            size = 64 if by_state or few != items else None
            for row in rows:
                token, a, state, b = row
                mine = {k[4]: v for k, v in parts.items() if k[:4] == (token, a, state, b)}
                total = b if by_state else a * share
                firsts = sorted(mine)
                if total == 0:
                    continue
                assert firsts[0] == 0 and all(x - y in (64, 128) for x, y in zip(firsts[1:], firsts))
                width = firsts[1] if len(firsts) > 1 else 128
                assert firsts[-1] + width >= total > firsts[-1]
                for first, v in mine.items():
                    v = sorted(v)
                    last = min(first + width, total) - 1
                    if by_state:
                        from_ = max(first - (b - a), 0)
                        end = share * (-(-(a - from_) // step)) if a > from_ else 0
                    else:
                        end = max(0, last // share + b - a + 1)
                    assert v[0][0] == 0 and v[-1][1] >= end and all(x[1] == y[0] for x, y in zip(v, v[1:]))
                    assert v[-1][1] == end and (by_state or all(x[1] % 64 == 0 for x in v[:-1]))
                    key = (token, a, state, b, first)
                    if len(v) == 1:
                        assert v[0][2] == -1 and key not in joined
                    else:
                        assert joined[key] == (v[0][2], len(v)) and [x[2] for x in v] == list(range(v[0][2], v[0][2] + len(v)))
            assert size is None or size == 64


@pytest.mark.parametrize("kw,code,text", [
    (dict(tokens=-1), -1, "tokens"), (dict(vocab=0), -1, "vocab"), (dict(dim=0), -1, "dim"), (dict(dtype=3), -1, "dtype"),
    (dict(scale=float("nan")), -1, "scale"), (dict(wide_tokens=2), -1, "wide_tokens"), (dict(reserved=1), -1, "reserved"),
    (dict(w_row_stride=-1, g_row_stride=-1), -1, "strides"), (dict(tokens=(1 << 30) + 1), -2, "2^30"), (dict(vocab=1 << 26), -2, "2^25"),
])
def test_library_refuses_embedding(kw, code, text):
    lib = _lib.load()
    d = _lib.EmbeddingDesc(tokens=5, vocab=7, dim=8, dtype=0, scale=1.0, w_row_stride=8, g_row_stride=8)
    for name, value in kw.items():
        setattr(d, name, value)
    assert lib.rdv_embedding_workspace_bytes(C.byref(d)) == code and text in _lib.last_error()
    assert lib.rdv_embedding(C.byref(d), 16, 16, 16, None) == code
    assert lib.rdv_embedding_backward(C.byref(d), 16, 16, 16, 16, 1 << 40, None) == code


@pytest.mark.parametrize("kw,text", [
    (dict(width=0), "width"), (dict(width=(1 << 20) + 1), "width"), (dict(rows=-1), "rows"), (dict(rows=1 << 38), "rows"),
    (dict(dtype=7), "dtype"), (dict(reserved=1), "reserved"), (dict(x_row_stride=-1), "strides"),
])
def test_library_refuses_rms_norm(kw, text):
    lib = _lib.load()
    d = _lib.RmsNormDesc(rows=3, width=8, dtype=0, eps=1e-6, x_row_stride=8, g_row_stride=8)
    for name, value in kw.items():
        setattr(d, name, value)
    assert lib.rdv_rms_norm_workspace_bytes(C.byref(d)) == _lib.RDV_ERR_INVALID and text in _lib.last_error()
    assert lib.rdv_rms_norm(C.byref(d), 16, None, None, None, 16, None, None, None) == _lib.RDV_ERR_INVALID


def test_library_refuses_null_pointers_and_small_workspaces():
    lib = _lib.load()
    e = _lib.EmbeddingDesc(tokens=5, vocab=7, dim=8, dtype=0, scale=1.0, w_row_stride=8, g_row_stride=8)
    r = _lib.RmsNormDesc(rows=3, width=8, dtype=0, eps=1e-6, x_row_stride=8, g_row_stride=8)
    assert lib.rdv_embedding(None, 16, 16, 16, None) == _lib.RDV_ERR_INVALID
    assert lib.rdv_embedding(C.byref(e), 16, None, 16, None) == _lib.RDV_ERR_INVALID
    assert lib.rdv_embedding_backward(C.byref(e), None, 16, 16, 16, 1 << 30, None) == _lib.RDV_ERR_INVALID
    n = lib.rdv_embedding_workspace_bytes(C.byref(e))
    assert lib.rdv_embedding_backward(C.byref(e), 16, 16, 16, 16, n - 1, None) == _lib.RDV_ERR_WORKSPACE
    assert lib.rdv_embedding_backward(C.byref(e), 16, 16, 16, 8, n, None) == _lib.RDV_ERR_WORKSPACE
    assert lib.rdv_rms_norm(C.byref(r), None, None, None, None, 16, None, None, None) == _lib.RDV_ERR_INVALID
    assert lib.rdv_rms_norm(C.byref(r), 16, 16, None, None, 16, None, None, None) == _lib.RDV_ERR_INVALID
    r.eps = -1.0
    assert lib.rdv_rms_norm(C.byref(r), 16, None, None, None, 16, None, None, None) == _lib.RDV_ERR_INVALID
    n = lib.rdv_rms_norm_workspace_bytes(C.byref(r))
    assert n > 0
    assert lib.rdv_rms_norm_backward(C.byref(r), 16, None, 16, None, 16, 16, 16, 16, n - 1, None) == _lib.RDV_ERR_WORKSPACE
    assert lib.rdv_rms_norm_backward(C.byref(r), 16, None, 16, None, 16, 16, None, 16, n, None) == _lib.RDV_ERR_INVALID
    d, plan = _desc(), _plan(_desc(), [(0, 7, 0, 9)], 0)
    call = lambda *a: lib.rdv_causal_attention(C.byref(d), *a, None)
    assert call(None, 16, 16, 16, 16, 16, None, None, None, 0) == _lib.RDV_ERR_INVALID
    assert call(plan.ctypes.data, 8, 16, 16, 16, 16, None, None, None, 0) == _lib.RDV_ERR_INVALID
    d.k_stride[0] = 3  # rows that have to be copied first
    assert call(plan.ctypes.data, 16, 16, 16, 16, 16, None, None, None, 0) == _lib.RDV_ERR_WORKSPACE
    d.k_stride[0] = 128
    assert call(plan.ctypes.data, 16, None, 16, 16, 16, None, None, None, 0) == _lib.RDV_ERR_INVALID
    assert call(plan.ctypes.data, 16, 16, 16, 16, 24, None, None, None, 0)
    assert call(plan.ctypes.data, 16, 16, 16, 16, 16, None, 24, None, 0) == _lib.RDV_ERR_INVALID


@pytest.mark.gpu
def test_refusals_of_buffers():
    t, w, g, x, p = T.cuda(), W.cuda(), G.cuda(), X.cuda(), P.cuda()
    q, k, lse, st = Q.cuda(), K.cuda(), LSE.cuda(), torch.zeros(5).cuda()
    eight = torch.empty(5, 12, dtype=torch.float8_e4m3fn).cuda()
    flat = torch.zeros(400).cuda()
    dq, dk = torch.empty_like(q), torch.empty_like(k)
    for call, error, text in (
        (lambda: rdv.embedding(T, w), TypeError, "tokens must be a GPU tensor"),
        (lambda: rdv.embedding(t, w, out=g.half()), TypeError, "out must be"),
        (lambda: rdv.embedding(t, w, out=w[:6].reshape(2, 3, 8)), AssertionError, "share memory"),
        (lambda: rdv.embedding_backward(g, t, 6, out=g.reshape(6, 8)), AssertionError, "share memory"),
        (lambda: rdv.embedding_backward(g, t, 6, out=w), AssertionError, "out must have"),
        (lambda: rdv.rms_norm(x, P), TypeError, "weight must be a GPU tensor"),
        (lambda: rdv.rms_norm(x, p, residual=x, out=x), AssertionError, "share memory"),
        (lambda: rdv.rms_norm(flat[1:61].reshape(5, 12), p, out=flat[:60].reshape(5, 12)), AssertionError, "share memory"),
        (lambda: rdv.rms_norm(x, p, residual=flat[:60].reshape(5, 12), sum_out=flat[12:72].reshape(5, 12)), AssertionError,
         "share memory"),
        (lambda: rdv.rms_norm(x, p, residual=x, out=flat[:60].reshape(5, 12), sum_out=flat[:60].reshape(5, 12)),
         AssertionError, "share memory"),
        (lambda: rdv.rms_norm(x, p, eight_bits=True, out=eight), TypeError, "values, scales"),
        (lambda: rdv.rms_norm(x, p, eight_bits=True, out=(x, st)), TypeError, "values must be"),
        (lambda: rdv.rms_norm(x, p, eight_bits=True, out=(eight, st[:4])), AssertionError, "scales must have"),
        (lambda: rdv.rms_norm_backward(x, x, p, st, grads=(x,)), TypeError, "grads must be"),
        (lambda: rdv.rms_norm_backward(x, x, p, st, grads=(x, p)), AssertionError, "share memory"),
        (lambda: rdv.rms_norm_backward(x, x, p, st, grads=(flat[:60].reshape(5, 12), flat[50:62])), AssertionError, "share memory"),
        (lambda: rdv.causal_attention(q, k, k, S, out=q), AssertionError, "share memory"),
        (lambda: rdv.causal_attention(q[:6], k, k, S), AssertionError, "7 tokens, q 6 rows"),
        (lambda: rdv.causal_attention(q, k[:8], k[:8], S), AssertionError, "9 states, k and v 8 rows"),
        (lambda: rdv.causal_attention(q, K, k, S), TypeError, "k must be a GPU tensor"),
        (lambda: rdv.causal_attention_backward(q, q, k, k, q, lse[:2], S), AssertionError, "lse must be"),
        (lambda: rdv.causal_attention_backward(q, q, k, k, q, lse, S, grads=(dq, dk, dk)), AssertionError, "share memory"),
        (lambda: rdv.causal_attention_backward(q, q, k, k, q, lse, S, grads=(q, dk, k)), AssertionError, "share memory"),
    ):
        with pytest.raises(error, match=text):
            call()


@pytest.mark.parametrize("backward", [0, 1])
def test_plans_need_the_rows_of_their_sequences(backward):
    """A plan serves every call whose tensors hold its sequences, whatever rows those that it was made with had."""
    lib, rows = _lib.load(), [(2, 5, 3, 6), (0, 2, 11, 9), (90, 0, 190, 0)]  # 7 tokens, 20 states
    plan = _plan(_desc(tokens=100, states=200), rows, backward)
    ok = lambda **kw: lib.rdv_causal_attention_workspace_bytes(C.byref(_desc(**kw)), plan.ctypes.data, backward)
    assert ok(tokens=100, states=200) >= 0 and ok(tokens=7, states=20) >= 0 and ok(tokens=1000, states=20) >= 0
    for kw in (dict(tokens=6, states=200), dict(tokens=100, states=19)):
        assert ok(**kw) == _lib.RDV_ERR_INVALID and "made for other" in _lib.last_error()
    assert np.array_equal(plan, _plan(_desc(tokens=500, states=200), rows, backward))


def test_lengths_may_be_any_iterable():
    """Numbers that can be read once are checked as a list's are."""
    s = rdv.PackedSequences(map(int, "302"), (x for x in (5, 1, 0)), iter((7, 0, 2)))
    assert (s.lengths, s.states, s.starts) == ((3, 0, 2), (5, 1, 0), (7, 0, 2))
    for values in ((1.5,), (1, 1e10), (float("nan"),), (float("inf"),), (1 << 40,)):
        for make in (list, iter, lambda v: (x for x in v)):
            with pytest.raises(ValueError, match="lengths"):
                rdv.PackedSequences(make(values))
            with pytest.raises(ValueError, match="states"):
                rdv.PackedSequences((1,) * len(values), make(values))


@pytest.mark.parametrize("lengths,kv_heads,pairs", [((64,), 1, True), ((700, 0, 1, 33), 2, True), ((20000,), 8, False),
                                                    ((2000,) * 20, 4, False)])
@pytest.mark.parametrize("backward", [0, 1])
def test_tiles_are_as_the_plan_says(lengths, kv_heads, pairs, backward):
    """A block's rows and states: 64 where pairs of waves share them, because blocks of 128 would leave CUs idle."""
    rows, t = [], 0
    for a in lengths:
        rows.append((t, a, t, a))
        t += a
    plan = _plan(_desc(tokens=t, states=t, heads=2 * kv_heads, kv_heads=kv_heads), rows, backward)
    words = plan[:256].view(np.int32)[(16 + C.sizeof(_lib.CausalAttentionDesc)) // 4:]
    (row_pairs, key_pairs, tile_rows, key_tile), (few, tiles, keys, _, _) = words[9:13].tolist(), _items(plan)
    assert (bool(row_pairs), tile_rows) == (pairs, 64 if pairs else 128)
    assert {i[4] % tile_rows for i in tiles} == {0}
    for token, a, _, _ in rows:
        firsts = {i[4] for i in few + tiles if i[:2] == [token, a]}
        assert firsts == set(range(0, 2 * a, tile_rows))
        if backward:
            assert {i[4] for i in keys if i[:2] == [token, a]} == set(range(0, a, key_tile))
    if backward:
        assert (bool(key_pairs), key_tile) == (pairs, 64 if pairs else 128)


@pytest.mark.parametrize("tokens,vocab,dim,fits", [
    (1000, 1 << 25, 1, True), (1000, 1 << 25, 4096, True), (1 << 20, 1 << 25, 64, True), (1 << 30, 1000, 1024, True),
    (0, 1 << 20, 1 << 20, True), (1 << 20, 256000, 16384, True), (1, 1 << 25, 1 << 20, False), (1 << 30, 5, 1 << 20, False),
])
def test_embedding_gradients_that_fit(tokens, vocab, dim, fits):
    """Every vocabulary that the forward call takes has a gradient, up to what launches can count."""
    lib = _lib.load()
    for dtype in (_lib.DTYPE_F32, _lib.DTYPE_BF16):
        d = _lib.EmbeddingDesc(tokens=tokens, vocab=vocab, dim=dim, dtype=dtype, scale=1.0, g_row_stride=dim)
        got = lib.rdv_embedding_workspace_bytes(C.byref(d))
        assert got >= vocab * 4 if fits else got == _lib.RDV_ERR_UNSUPPORTED and "too large" in _lib.last_error()
