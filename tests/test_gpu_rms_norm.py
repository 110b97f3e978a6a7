"""GPU parity of rms_norm and rms_norm_backward against oracle/prompt_ops.py, whose bounds are the tolerances."""
import numpy as np
import pytest
import torch

import rdv_project_amd as rdv
from oracle import prompt_ops as O

pytestmark = pytest.mark.gpu

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def _np(t):
    return t.detach().double().cpu().numpy()


def _close(got, ref, err, what):
    got = _np(got)
    assert got.shape == ref.shape and np.isfinite(got).all(), what
    d = np.abs(got - ref) - err
    if d.size:
        at = np.unravel_index(np.argmax(d), d.shape)
        assert d[at] <= 0, f"{what}: |err| {np.abs(got - ref)[at]:.3g} > bound {err[at]:.3g} at {at}"


def _inputs(rows, width, dtype, seed=0):
    g = torch.Generator().manual_seed(seed + rows + 3 * width)
    make = lambda: torch.randn(rows, width, generator=g).to(TYPES[dtype]).cuda()
    return make(), make() * 3, make(), make(), (torch.rand(width, generator=g) + 0.5).cuda()


def _sum(x, r):
    """The sum as it is stored."""
    return (x.float() + r.float()).to(x.dtype)


def _check(rows, width, dtype, eps=1e-6, what=""):
    x, r, g, gs, w = _inputs(rows, width, dtype)
    for residual, weight, grad_sum in ((None, w, None), (r, w, gs), (r, None, None)):
        h = x if residual is None else _sum(x, residual)
        ref = O.rms_norm(_np(h), None if weight is None else _np(weight), eps, dtype, _np(g),
                         None if grad_sum is None else _np(grad_sum))
        got = rdv.rms_norm(x, weight, residual=residual, eps=eps, return_stats=True)
        y, stats = got[0], got[-1]
        assert y.dtype == x.dtype and y.is_contiguous()
        if residual is not None:
            assert torch.equal(got[1], h), what
        _close(y, ref["y"], ref["y_err"], what + " y")
        _close(stats, ref["stats"], ref["stats_err"], what + " stats")
        dx, dw = rdv.rms_norm_backward(g, h, weight, stats, grad_sum=grad_sum)
        _close(dx, ref["dx"], ref["dx_err"], what + " dx")
        _close(dw, ref["dweight"], ref["dweight_err"], what + " dweight")
        got = rdv.rms_norm(x, weight, residual=residual, eps=eps, eight_bits=True)
        values, scales = got if residual is None else got[0]
        assert values.dtype == torch.float8_e4m3fn and values.shape == x.shape
        _close(scales, ref["scale"], ref["scale_err"], what + " scales")
        ratio = ref["y"] / np.where(ref["scale"] == 0, 1.0, ref["scale"])[:, None]
        _close(values.float(), ratio, O.e4m3_bound(ratio), what + " values")
        if residual is not None:
            assert torch.equal(got[1], h)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,width", [
    (1, 1), (3, 7), (5, 8), (64, 32), (33, 33), (9, 64), (17, 100), (130, 128), (4, 255), (21, 256), (7, 512), (11, 513),
    (5, 777), (3, 1024), (2, 1025), (6, 2048), (3, 2049), (2, 4096), (3, 5001), (2, 8192), (2, 9000), (1, 16384),
])
def test_matches_oracle(dtype, rows, width):
    _check(rows, width, dtype, what=f"{rows} x {width} {dtype}")


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,width", [(5000, 24), (3001, 300), (1500, 1000), (1200, 1024), (1100, 2048)])
def test_many_rows(dtype, rows, width):
    """More rows than blocks: groups go from row to row."""
    _check(rows, width, dtype, what=f"{rows} x {width} {dtype}")


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("width", [16385, 32768, 40000, 70001])
def test_wide_rows(dtype, width):
    """Up to four pieces of a thread of 1,024 in registers, and past them."""
    _check(3, width, dtype, what=f"3 x {width} {dtype}")


def test_no_rows():
    x, w = torch.zeros(0, 40).cuda(), torch.ones(40).cuda()
    y, h, stats = rdv.rms_norm(x, w, residual=x, return_stats=True)
    assert y.shape == h.shape == (0, 40) and stats.shape == (0,)
    dx, dw = rdv.rms_norm_backward(x, h, w, stats)
    assert dx.shape == (0, 40) and not dw.any() and dw.shape == (40,)
    (values, scales) = rdv.rms_norm(x, w, eight_bits=True)
    assert values.shape == (0, 40) and scales.shape == (0,)


def test_zeros_and_extremes():
    """A row of zeros is zeros (scale 0), large and tiny rows keep their size, NaN and infinity stay in their row."""
    x = torch.randn(6, 96).cuda()
    x[0] = 0
    x[1] *= 1e18
    x[2] *= 1e-30
    x[3, 5] = float("nan")
    x[4, 7] = float("inf")
    w = torch.ones(96).cuda()
    y = rdv.rms_norm(x, w)
    assert not y[0].any() and torch.isnan(y[3]).all() and torch.isfinite(y[[0, 1, 2, 5]]).all()
    want = x[1].double() / x[1].double().square().mean().sqrt()
    assert (y[1].double() - want).abs().max() < 1e-5
    (values, scales) = rdv.rms_norm(x, w, eight_bits=True)
    assert scales[0] == 0 and not values[0].float().any()
    assert torch.isfinite(values[[0, 1, 2, 5]].float()).all() and torch.isnan(values[3].float()).all()
    assert (values.float()[5].abs().max() == 448.0)


def test_eight_bits_of_tiny_rows():
    """Where max |y| / 448 is below fp32's normal numbers the scale is the smallest of them."""
    x = torch.full((2, 64), 1e-37).cuda()
    x[1] = 1e-39
    values, scales = rdv.rms_norm(x, None, eps=1.0, eight_bits=True)
    assert (scales == torch.finfo(torch.float32).tiny).all()
    back = values.double() * scales.double()[:, None]
    assert ((back - x.double()).abs() <= 2.0 ** -4 * x.double() + 2.0 ** -10 * scales.double()[:, None]).all()


def test_layouts_and_buffers():
    """Views of wider rows, transposed rows, more dimensions, and results in the inputs' own memory."""
    base, other = torch.randn(30, 100).cuda(), torch.randn(30, 60).cuda()
    w = torch.rand(60).cuda() + 0.5
    x, r = base[:, 20:80], other
    want, h = rdv.rms_norm(x.contiguous(), w, residual=r)
    got, h2 = rdv.rms_norm(x, w, residual=r)
    assert torch.equal(got, want) and torch.equal(h, h2)
    got, h2 = rdv.rms_norm(x.reshape(5, 6, 60), w, residual=r.reshape(5, 6, 60))
    assert got.shape == (5, 6, 60) and torch.equal(got.reshape(30, 60), want)
    turned = x.t().contiguous().t()
    assert torch.equal(rdv.rms_norm(turned, w, residual=r)[0], want)
    stream = r.clone()  # the residual stream in place
    got, h2 = rdv.rms_norm(x, w, residual=stream, sum_out=stream)
    assert h2 is stream and torch.equal(stream, h) and torch.equal(got, want)
    xc = x.contiguous()
    got, h2 = rdv.rms_norm(xc, w, residual=r, sum_out=xc)
    assert h2 is xc and torch.equal(xc, h) and torch.equal(got, want)
    plain = rdv.rms_norm(r, w)
    own = r.clone()
    assert rdv.rms_norm(own, w, out=own) is own and torch.equal(own, plain)
    wide = torch.randn(2, 40000).cuda()
    plain = rdv.rms_norm(wide, None)
    assert torch.equal(rdv.rms_norm(wide, None, out=wide), plain)
    buffer = torch.empty(30 * 60 + 1).cuda()[1:].reshape(30, 60)
    assert rdv.rms_norm(x, w, residual=r, out=buffer)[0] is buffer and torch.equal(buffer, want)
    g = torch.randn(30, 200).cuda()[:, 70:130]
    y, h, stats = rdv.rms_norm(x, w, residual=r, return_stats=True)
    dx, dw = rdv.rms_norm_backward(g.contiguous(), h, w, stats)
    dx2, dw2 = rdv.rms_norm_backward(g, h, w, stats)
    assert torch.equal(dx, dx2) and torch.equal(dw, dw2)
    into = torch.empty(30, 60).cuda(), torch.empty(60).cuda()
    assert rdv.rms_norm_backward(g, h, w, stats, grads=into)[0] is into[0]
    assert torch.equal(into[0], dx) and torch.equal(into[1], dw)


def test_gradients_by_differences():
    x, _, g, _, w = _inputs(3, 20, "f32")
    y, stats = rdv.rms_norm(x, w, return_stats=True)
    dx, dw = rdv.rms_norm_backward(g, x, w, stats)

    def loss(a, b):
        a, b = a.double(), b.double()
        return (b * a / torch.sqrt((a * a).mean(1, keepdim=True) + 1e-6) * g.double()).sum()

    step = 1e-5
    for t, grad, at in ((x, dx, (1, 4)), (x, dx, (2, 19)), (w, dw, (7,))):
        ends = []
        for sign in (1, -1):
            moved = t.double().clone()
            moved[at] += sign * step
            ends.append(loss(moved, w) if t is x else loss(x, moved))
        assert abs((ends[0] - ends[1]) / (2 * step) - grad[at]) < 1e-5 * (1 + abs(grad[at]))


def test_offsets_past_32_bits():
    """The last rows of more than 2^31 elements, the others zeros, which add nothing to dweight."""
    rows = (1 << 21) + 5
    x = torch.zeros(rows, 1024, dtype=torch.bfloat16, device="cuda")
    x[-5:] = torch.randn(5, 1024)
    w = torch.rand(1024).cuda()
    y, stats = rdv.rms_norm(x, w, return_stats=True)
    dx, dw = rdv.rms_norm_backward(y, x, w, stats)
    assert not y[:-5].any() and not dx[:-5].any()
    ref = O.rms_norm(_np(x[-5:]), _np(w), 1e-6, "bf16", _np(y[-5:]))
    for got, name in ((y[-5:], "y"), (stats[-5:], "stats"), (dx[-5:], "dx"), (dw, "dweight")):
        _close(got, ref[name], ref[name + "_err"], name)


@pytest.mark.parametrize("width", [64, 777, 4096, 33000])
def test_eight_bits_with_statistics(width):
    """What a call returns beside 8 bits is what it returns beside y, and its values are y's."""
    x, r = torch.randn(5, width).half().cuda(), torch.randn(5, width).half().cuda()
    w = (1 + 0.1 * torch.randn(width)).cuda()
    y, h, stats = rdv.rms_norm(x, w, residual=r, return_stats=True)
    buffers = torch.empty(5, width, dtype=torch.float8_e4m3fn, device="cuda"), torch.empty(5, device="cuda")
    (values, scales), h8, stats8 = rdv.rms_norm(x, w, residual=r, return_stats=True, eight_bits=True, out=buffers)
    assert values is buffers[0] and scales is buffers[1]
    assert torch.equal(h8, h) and torch.equal(stats8, stats)
    # y is rounded by 2^-11 and the value by 2^-4, or by half of e4m3's smallest step (2^-10) times the scale
    back, y = values.double() * scales.double()[:, None], y.double()
    assert ((back - y).abs() <= y.abs() * (2.0 ** -4 + 2.0 ** -10) + scales.double()[:, None] * 2.0 ** -10 + 2.0 ** -25).all()
    (values, scales), stats8 = rdv.rms_norm(x, w, return_stats=True, eight_bits=True)
    assert torch.equal(stats8, rdv.rms_norm(x, w, return_stats=True)[1])


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("width", [40, 1100, 9000, 40000])
def test_eight_bits_of_a_weight_that_is_nan(dtype, width):
    """max |y| of a row with a NaN in y is NaN, and so are its scale and what it stands for; an infinite y gives an infinite
    scale, NaN there and zeros elsewhere."""
    x = torch.randn(4, width).to(TYPES[dtype]).cuda()
    x[3] = 0
    w = (torch.rand(width) + 0.5).cuda()
    for at in (0, width // 2, width - 1):
        bad = w.clone()
        bad[at] = float("nan")
        values, scales = rdv.rms_norm(x, bad, eight_bits=True)
        assert torch.isnan(scales).all() and torch.isnan(values.float()).all()
        bad[at] = float("inf")
        values, scales = rdv.rms_norm(x[:3], bad, eight_bits=True)
        assert torch.isinf(scales).all()
        nan = torch.isnan(values.float())
        assert nan[:, at].all() and nan.sum() == 3 and not values.float().nan_to_num().any()


@pytest.mark.parametrize("dtype,rows,width", [("f32", 1 << 26, 8), ("f32", 1 << 22, 136), ("f32", 1 << 20, 1100),
                                              ("f16", 1 << 18, 8200), ("f16", 1 << 18, 33000), ("f16", 32767, 4100),
                                              ("f16", 32768, 4100), ("f16", 32769, 4100), ("f32", 65537, 5000),
                                              ("f32", 98304, 1100), ("f32", 98305, 1100), ("f16", 32769, 33000)])
def test_dweight_of_very_many_rows(dtype, rows, width):
    """Equal rows, whose terms' roundings do not cancel.  A thread adds at most 128 terms one after the other, 127 U32 of
    their sum, then at most 22 of those sums (the 2,731 rows of a group of 2^26 rows in 24,576 of them), 21 U32; the groups
    of a block add up to 32, 31 U32; then it is 64 bits, rounded once.  A term is two products, 2 U32."""
    r = torch.Generator().manual_seed(width)
    x = torch.tensor([1.0, 2.0]).repeat(width // 2).to(TYPES[dtype]).cuda()
    grad = (1 + torch.rand(width, generator=r)).to(TYPES[dtype]).cuda()
    stats = torch.full((rows,), 0.4 ** 0.5).cuda()
    _, dw = rdv.rms_norm_backward(grad.expand(rows, -1), x.expand(rows, -1), None, stats)
    want = rows * grad.double() * x.double() * stats[0].double()
    assert ((dw.double() - want).abs() <= (127 + 21 + 31 + 1 + 2) * 2.0 ** -24 * want).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows,width", [(600, 9000), (600, 40000), (2000, 4096), (600, 16385)])
def test_many_wide_rows(dtype, rows, width):
    """More rows than blocks of those that share a row among 256 or 1,024 threads, in registers and past them."""
    _check(rows, width, dtype, what=f"{rows} x {width} {dtype}")
