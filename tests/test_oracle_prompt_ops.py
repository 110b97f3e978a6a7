"""The 64-bit forms of oracle/prompt_ops.py against torch's autograd and against differences (CPU)."""
import math

import numpy as np
import pytest
import torch

from oracle import prompt_ops as O


def _draw(*shape, seed=0):
    return np.random.default_rng(seed + sum(shape)).standard_normal(shape)


def test_embedding():
    weight, grad = _draw(7, 3), _draw(6, 3, seed=1)
    tokens = np.array([2, 6, 2, -1, 7, 0])
    w = torch.tensor(weight, requires_grad=True)
    inside = torch.tensor([True, True, True, False, False, True])[:, None]
    y = torch.where(inside, w[torch.tensor(np.clip(tokens, 0, 6))], 0.0) * 1.5
    y.backward(torch.tensor(grad))
    np.testing.assert_allclose(O.embedding(tokens, weight, 1.5), y.detach().numpy(), rtol=1e-12)
    dw, err = O.embedding_grad(grad, tokens, 7, 1.5, "f32")
    np.testing.assert_allclose(dw, w.grad.numpy(), rtol=1e-12)
    assert not dw[[1, 3, 4, 5]].any() and (err >= 0).all()


@pytest.mark.parametrize("weighted,summed", [(True, True), (False, False), (True, False)])
def test_rms_norm(weighted, summed):
    h, g, gs = _draw(5, 8), _draw(5, 8, seed=1), _draw(5, 8, seed=2) if summed else None
    weight = _draw(8, seed=3) if weighted else None
    x = torch.tensor(h, requires_grad=True)
    w = torch.tensor(weight if weighted else np.ones(8), requires_grad=True)
    y = w * x / torch.sqrt((x * x).mean(1, keepdim=True) + 1e-3)
    loss = (y * torch.tensor(g)).sum() + (0 if gs is None else (x * torch.tensor(gs)).sum())
    loss.backward()
    r = O.rms_norm(h, weight, 1e-3, "f32", g, gs)
    np.testing.assert_allclose(r["y"], y.detach().numpy(), rtol=1e-12)
    np.testing.assert_allclose(r["dx"], x.grad.numpy(), rtol=1e-10, atol=1e-13)
    np.testing.assert_allclose(r["dweight"], w.grad.numpy(), rtol=1e-12)


@pytest.mark.parametrize("t,n", [(1, 1), (5, 5), (3, 7), (6, 2), (4, 0)])
def test_causal_attention(t, n):
    d, scale = 4, 0.6
    q, k, v, g = _draw(t, d), _draw(n, d, seed=1), _draw(n, d, seed=2), _draw(t, d, seed=3)
    r = O.causal_attention(q, k, v, scale, grad=g)
    tq, tk, tv = (torch.tensor(x, requires_grad=True) for x in (q, k, v))
    loss = torch.zeros((), dtype=torch.float64)
    for i in range(t):
        seen = i + n - t + 1
        if seen <= 0:
            assert not r["out"][i].any() and r["lse"][i] == -math.inf and not r["dq"][i].any()
            continue
        s = tk[:seen] @ tq[i] * scale
        o = torch.softmax(s, 0) @ tv[:seen]
        np.testing.assert_allclose(r["out"][i], o.detach().numpy(), rtol=1e-10, atol=1e-13)
        np.testing.assert_allclose(r["lse"][i], torch.logsumexp(s, 0).item(), rtol=1e-12)
        loss = loss + (o * torch.tensor(g[i])).sum()
    if loss.requires_grad:
        loss.backward()
    for name, x in (("dq", tq), ("dk", tk), ("dv", tv)):
        want = np.zeros(x.shape) if x.grad is None else x.grad.numpy()
        np.testing.assert_allclose(r[name], want, rtol=1e-9, atol=1e-12)


def test_causal_attention_gradient_by_differences():
    """dL/dk of one element, from the forward form alone."""
    q, k, v, g = (_draw(5, 3, seed=s) for s in range(4))
    step = 1e-6
    ends = []
    for sign in (1, -1):
        moved = k.copy()
        moved[1, 2] += sign * step
        ends.append((O.causal_attention(q, moved, v, 0.7)["out"] * g).sum())
    want = (ends[0] - ends[1]) / (2 * step)
    assert abs(O.causal_attention(q, k, v, 0.7, grad=g)["dk"][1, 2] - want) < 1e-8
