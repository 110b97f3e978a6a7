"""The plain 64-bit forms of the image-network operators against other formulations: gradients against central
differences, statistics against their definitions, the generator against its authors' published known answers."""
import numpy as np
import pytest

from oracle import image_ops as O


def _rng(seed):
    return np.random.default_rng(seed)


def _difference(f, x, direction, h=1e-5):
    return (f(x + h * direction) - f(x - h * direction)) / (2 * h)


@pytest.mark.parametrize("activation", ["none", "relu", "silu"])
@pytest.mark.parametrize("shape,groups", [((2, 7, 6), 3), ((1, 5, 4), 1), ((3, 1, 8), 2), ((1, 9, 3), 3)])
def test_group_norm_gradients_against_differences(activation, shape, groups):
    r = _rng(1)
    x, g = r.normal(size=shape) * 2 + 1, r.normal(size=shape)
    w, b = r.uniform(0.5, 1.5, shape[2]), r.normal(size=shape[2])
    ref = O.group_norm(x, w, b, groups, activation=activation, grad=g)

    def loss(x, w, b):
        return (O.group_norm(x, w, b, groups, activation=activation)["y"] * g).sum()

    for arg, grad, at in (("x", ref["dx"], x), ("w", ref["dweight"], w), ("b", ref["dbias"], b)):
        d = r.normal(size=at.shape)
        num = _difference(lambda t: loss(**{**dict(x=x, w=w, b=b), arg: t}), at, d)
        assert abs(num - (grad * d).sum()) <= 1e-6 * (np.abs(grad * d).sum() + 1), arg


def test_group_norm_statistics():
    x = _rng(2).normal(size=(2, 11, 12)) * 3 - 5
    y = O.group_norm(x, None, None, 4, eps=0.0)["y"].reshape(2, 11, 4, 3)
    assert np.abs(y.mean(axis=(1, 3))).max() < 1e-12 and np.abs(y.var(axis=(1, 3)) - 1).max() < 1e-12


@pytest.mark.parametrize("lq,lk,d,counted", [(3, 5, 4, 5), (4, 1, 3, 1), (1, 6, 2, 4), (2, 4, 5, 0)])
def test_attention_gradients_against_differences(lq, lk, d, counted):
    r = _rng(3)
    q, k, v, g = r.normal(size=(lq, d)), r.normal(size=(lk, d)), r.normal(size=(lk, d)), r.normal(size=(lq, d))
    valid = np.zeros(lk, bool)
    valid[r.permutation(lk)[:counted]] = True
    ref = O.attention(q, k, v, valid, 0.7, grad=g)

    def loss(q, k, v):
        return (O.attention(q, k, v, valid, 0.7)["out"] * g).sum()

    for arg, at in (("q", q), ("k", k), ("v", v)):
        grad, dirn = ref["d" + arg], r.normal(size=at.shape)
        num = _difference(lambda t: loss(**{**dict(q=q, k=k, v=v), arg: t}), at, dirn)
        assert abs(num - (grad * dirn).sum()) <= 1e-6 * (np.abs(grad * dirn).sum() + 1), arg
    assert not ref["dk"][~valid].any() and not ref["dv"][~valid].any()


def test_attention_against_the_definition():
    r = _rng(4)
    q, k, v = r.normal(size=(3, 4)), r.normal(size=(5, 4)), r.normal(size=(5, 4))
    valid = np.array([1, 0, 1, 1, 0], bool)
    ref = O.attention(q, k, v, valid, 0.5)
    for i in range(3):
        e = [np.exp(0.5 * (q[i] @ k[j])) if valid[j] else 0.0 for j in range(5)]
        assert np.allclose(ref["out"][i], sum(e[j] * v[j] for j in range(5)) / sum(e), atol=1e-14)
        assert np.isclose(ref["lse"][i], np.log(sum(e)))


@pytest.mark.parametrize("counter,key,words", [
    ([0] * 4, [0] * 2, [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]),
    ([0xFFFFFFFF] * 4, [0xFFFFFFFF] * 2, [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]),
    ([0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344], [0xA4093822, 0x299F31D0],
     [0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1]),
])
def test_generator_known_answers(counter, key, words):
    assert O.philox4x32(counter, key) == words


def test_dropout_keeps_its_share():
    n, p = 20000, 0.3
    kept = (O.dropout(np.ones(n), p, 12345, 7) != 0).mean()
    assert abs(kept - (1 - p)) < 5 * np.sqrt(p * (1 - p) / n)
