"""Layer norm on the GPU, forward and backward, against the formulas in float64.

Bounds, elementwise, from the arithmetic alone.  u is half a step of the
compute type (2^-24, 2^-53 in float64) and D bounds how many additions one
element of a row's sum goes through (at most h / 64 in its lane, then the tree
over lanes and waves): a sum is off by at most D u sum|terms|.  A result
stored in a narrower type is off by half a step of it more.
"""

from __future__ import annotations

import pytest
import torch

from _helpers import DEV, say, seeded
from resihp_megatron_amd import kernels as K
from resihp_megatron_amd import layer, moe

pytestmark = pytest.mark.gpu

HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24, torch.float64: 2.0 ** -53}
TYPES = [(torch.bfloat16, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.float32, torch.float32),
         (torch.float64, torch.float64)]
# One element to rows longer than any register holds; odd sizes, sizes around the vectors' and the waves' ends.
HIDDEN = [1, 2, 3, 7, 8, 9, 63, 64, 65, 127, 255, 256, 257, 511, 512, 700, 1000, 1023, 1365, 1400, 1801, 2048, 2049,
          2560, 4096, 4099, 5001, 5120, 6001, 8192, 8200, 10007, 16384, 16392, 20001]


def _unit(dtype):
    return 2.0 ** -53 if dtype == torch.float64 else 2.0 ** -24


def _depth(h):
    return h // 64 + 24


def _inputs(T, h, dt, wdt, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, h, generator=g, dtype=torch.float64) + 0.3
    x[:, :: max(1, h // 3)] *= 20
    w = 1 + 0.1 * torch.randn(h, generator=g, dtype=torch.float64)
    b = 0.1 * torch.randn(h, generator=g, dtype=torch.float64)
    dy = torch.randn(T, h, generator=g, dtype=torch.float64)
    dres = torch.randn(T, h, generator=g, dtype=torch.float64)
    return x.to(dt), w.to(wdt), b.to(wdt), dy.to(dt), dres.to(dt)


def _close(got, want, tol, what):
    got = got.detach().cpu().double()
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), (what, int(bad.sum()), float((got - want).abs()[bad].max()), float(tol[bad].min()))


def _check_forward(x, w, b, eps, y, mean, rstd):
    dt, h = x.dtype, x.shape[1]
    u, D = _unit(dt), _depth(h)
    xd = x.double()
    one = torch.ones(h, dtype=torch.float64)
    wd, bd = one if w is None else w.double(), 0 * one if b is None else b.double()
    m = xd.mean(1, keepdim=True)
    c = xd - m
    var = (c * c).mean(1, keepdim=True)
    r = (var + eps).rsqrt()
    em = (D + 2) * u * xd.abs().mean(1, keepdim=True)                       # of the mean
    # Of the variance: the sum's own, c's rounding and the mean's error (which enters squared).
    ev = (D + 4) * u * var + em * em + 2 * u * (c.abs() * xd.abs()).mean(1, keepdim=True)
    er = r * (0.5 * ev / (var + eps) + 4 * u) + 0 * r                        # of rstd
    _close(mean, m[:, 0], em[:, 0], "mean")
    _close(rstd, r[:, 0], er[:, 0], "rstd")
    y64 = c * r * wd + bd
    tol = wd.abs() * (r * (em + u * c.abs()) + c.abs() * er + 2 * u * c.abs() * r) + 2 * u * (y64.abs() + bd.abs())
    _close(y, y64, tol * 1.01 + (y64.abs() + tol) * HALF[dt], "y")


def _check_backward(dy, x, w, mean, rstd, dres, dx, dw, db, wdt):
    dt, (T, h) = x.dtype, x.shape
    u, D = _unit(dt), _depth(h)
    dyd, xd = dy.double(), x.double()
    wd = torch.ones(h, dtype=torch.float64) if w is None else w.double()
    m, r = mean.double().cpu()[:, None], rstd.double().cpu()[:, None]
    g, xh = dyd * wd, (xd - m) * r
    c1, c2 = (g * xh).mean(1, keepdim=True), g.mean(1, keepdim=True)
    a1, a2 = (g * xh).abs().mean(1, keepdim=True), g.abs().mean(1, keepdim=True)
    if dx is not None:
        want = r * (g - c2 - xh * c1)
        tol = r * u * (3 * g.abs() + (D + 4) * a2 + xh.abs() * ((D + 8) * a1 + 6 * c1.abs()) + 4 * c2.abs())
        if dres is not None:
            want = want + dres.double()
            tol = tol + u * want.abs()
        _close(dx, want, tol * 1.01 + (want.abs() + tol) * HALF[dt], "dx")
    # A column's sum goes through at most T additions, and from 64 rows on there are at least 16 partial sums.
    rows = T + 8 if T < 64 else T // 16 + 600
    for got, terms, name in ((dw, dyd * xh, "dw"), (db, dyd, "db")):
        if got is not None:
            want = terms.sum(0)
            tol = (rows + 4) * u * terms.abs().sum(0)
            _close(got, want, tol + (want.abs() + tol) * HALF[wdt], name)


@pytest.mark.parametrize("h", HIDDEN)
@pytest.mark.parametrize("dt,wdt", TYPES, ids=["bf16-f32", "bf16", "f32", "f64"])
def test_rows_of_every_length(h, dt, wdt):
    for T in (1, 5) if h > 300 else (1, 2, 67):
        say(f"norm T={T} h={h} {dt} {wdt}")
        x, w, b, dy, dres = _inputs(T, h, dt, wdt, seed=h)
        eps = 1e-5
        dev = [t.to(DEV) for t in (x, w, b, dy, dres)]
        y, mean, rstd = K.layer_norm(*dev[:3], eps)
        assert y.dtype == dt and mean.dtype == rstd.dtype == (torch.float64 if dt == torch.float64 else torch.float32)
        _check_forward(x, w, b, eps, y, mean, rstd)
        dx, dw, db = K.layer_norm_bwd(dev[3], dev[0], dev[1], mean, rstd, dres=dev[4])
        _check_backward(dy, x, w, mean, rstd, dres, dx, dw, db, wdt)
        dx, dw, db = K.layer_norm_bwd(dev[3], dev[0], dev[1], mean, rstd)
        _check_backward(dy, x, w, mean, rstd, None, dx, dw, db, wdt)


@pytest.mark.parametrize("T", [1, 2, 3, 15, 16, 17, 63, 64, 65, 255, 257, 1000, 2047, 4101])
@pytest.mark.parametrize("h,dt,wdt", [(256, torch.bfloat16, torch.float32), (333, torch.bfloat16, torch.bfloat16),
                                      (1536, torch.float32, torch.float32), (96, torch.float64, torch.float64)])
def test_row_counts(T, h, dt, wdt):
    say(f"norm T={T} h={h} {dt}")
    x, w, b, dy, dres = _inputs(T, h, dt, wdt, seed=T)
    dev = [t.to(DEV) for t in (x, w, b, dy, dres)]
    y, mean, rstd = K.layer_norm(*dev[:3], 1e-5)
    _check_forward(x, w, b, 1e-5, y, mean, rstd)
    got = K.layer_norm_bwd(dev[3], dev[0], dev[1], mean, rstd, dres=dev[4])
    _check_backward(dy, x, w, mean, rstd, dres, *got, wdt)
    again = K.layer_norm_bwd(dev[3], dev[0], dev[1], mean, rstd, dres=dev[4])
    assert all(torch.equal(a, c) for a, c in zip(got, again)), "the same call twice"


@pytest.mark.parametrize("h", [8, 64, 333, 1024, 1400, 2048, 2301, 4096, 9000])
def test_a_row_keeps_its_bits_in_any_batch(h):
    x, w, b, dy, dres = (t.to(DEV) for t in _inputs(600, h, torch.bfloat16, torch.float32, seed=3))
    say(f"norm batch independence h={h}")
    y, mean, rstd = K.layer_norm(x, w, b, 1e-5)
    dx, _, _ = K.layer_norm_bwd(dy, x, w, mean, rstd, dres=dres)
    for t0, t1 in ((0, 1), (599, 600), (17, 40), (100, 500)):
        s = slice(t0, t1)
        y1, m1, r1 = K.layer_norm(x[s].clone(), w, b, 1e-5)
        assert torch.equal(y1, y[s]) and torch.equal(m1, mean[s]) and torch.equal(r1, rstd[s])
        d1, _, _ = K.layer_norm_bwd(dy[s].clone(), x[s].clone(), w, mean[s].clone(), rstd[s].clone(), dres=dres[s].clone())
        assert torch.equal(d1, dx[s])


def _at_offset(t, k):
    """A contiguous copy of t that starts k elements into its allocation."""
    flat = torch.empty(t.numel() + k, dtype=t.dtype, device=DEV)
    out = flat[k:].view(t.shape)
    out.copy_(t)
    return out


@pytest.mark.parametrize("k", [1, 3, 4])
def test_tensors_at_any_element(k):
    for dt, wdt, h in ((torch.bfloat16, torch.bfloat16, 264), (torch.bfloat16, torch.float32, 4096), (torch.float32,
                       torch.float32, 1000), (torch.float64, torch.float64, 66)):
        say(f"norm at element {k} {dt} h={h}")
        x, w, b, dy, dres = _inputs(70, h, dt, wdt, seed=k)
        dev = [_at_offset(t, k) for t in (x, w, b, dy, dres)]
        y, mean, rstd = K.layer_norm(*dev[:3], 1e-5)
        y0, mean0, rstd0 = K.layer_norm(*(t.to(DEV) for t in (x, w, b)), 1e-5)
        assert torch.equal(y, y0) and torch.equal(mean, mean0) and torch.equal(rstd, rstd0)
        got = K.layer_norm_bwd(dev[3], dev[0], dev[1], mean, rstd, dres=dev[4])
        want = K.layer_norm_bwd(dy.to(DEV), x.to(DEV), w.to(DEV), mean, rstd, dres=dres.to(DEV))
        assert all(torch.equal(a, c) for a, c in zip(got, want))


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,h", [(40, 512), (300, 777), (9, 9001)])
def test_without_weight_bias_or_some_gradients(dt, T, h):
    say(f"norm options {dt} T={T} h={h}")
    x, w, b, dy, _ = _inputs(T, h, dt, torch.float32, seed=5)
    xg, wg, bg, dyg = (t.to(DEV) for t in (x, w, b, dy))
    for ww, bb, wd, bd in ((wg, None, w, None), (None, bg, None, b), (None, None, None, None)):
        y, mean, rstd = K.layer_norm(xg, ww, bb, 1e-6)
        _check_forward(x, wd, bd, 1e-6, y, mean, rstd)
    full = K.layer_norm_bwd(dyg, xg, wg, mean, rstd)
    for need in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 1, 0), (0, 1, 1), (0, 0, 0)):
        got = K.layer_norm_bwd(dyg, xg, wg, mean, rstd, None, *map(bool, need))
        for a, c, n in zip(got, full, need):
            assert (a is None) == (not n)
            if n:   # dx has one formula; the sums may take another order where dx is not wanted
                torch.testing.assert_close(a, c, rtol=1e-4, atol=1e-4 * T ** 0.5)
        _check_backward(dy, x, w, mean, rstd, None, *got, torch.float32)
    dx, dw, db = K.layer_norm_bwd(dyg, xg, None, mean, rstd, dtype=torch.float32)
    _check_backward(dy, x, None, mean, rstd, None, dx, dw, db, torch.float32)


def test_no_rows():
    say("norm T=0")
    x = torch.empty(0, 96, device=DEV)
    w = torch.ones(96, device=DEV)
    y, mean, rstd = K.layer_norm(x, w, w)
    assert y.shape == (0, 96) and mean.shape == rstd.shape == (0,)
    dx, dw, db = K.layer_norm_bwd(y, x, w, mean, rstd)
    assert dx.shape == (0, 96) and torch.all(dw == 0) and torch.all(db == 0)
    z = torch.zeros(3, 0, 96, device=DEV, requires_grad=True)
    assert layer.layer_norm(z, w, w).shape == (3, 0, 96)


@pytest.mark.parametrize("h", [64, 1000, 9000])
def test_rows_that_are_constant_huge_or_not_finite(h):
    """A constant row gives the bias (its centred values are exact zeros where the mean is exact); a row with an
    infinity or a NaN is NaN and leaves its neighbours alone; a large mean does not swamp the variance."""
    g = torch.Generator().manual_seed(11)
    x = torch.randn(8, h, generator=g)
    x[1] = 2.0
    x[2, h // 2] = float("inf")
    x[3, 0] = float("nan")
    x[4] = 4096.0 + torch.randint(0, 8, (h,), generator=g).float()
    x[5] *= 1e15
    x[6] *= 1e-15
    w, b = torch.ones(h), torch.full((h,), 0.25)
    say(f"norm odd rows h={h}")
    y, mean, rstd = K.layer_norm(x.to(DEV), w.to(DEV), b.to(DEV), 1e-5)
    rows = [0, 1, 4, 5, 6, 7]
    _check_forward(x[rows], w, b, 1e-5, y[rows], mean[rows], rstd[rows])
    assert torch.all(y[1].cpu() == 0.25) and torch.isnan(y[2:4]).all()
    dy = torch.randn(8, h, generator=g)
    dx, dw, db = K.layer_norm_bwd(dy.to(DEV), x.to(DEV), w.to(DEV), mean, rstd)
    _check_backward(dy[rows], x[rows], w, mean[rows], rstd[rows], None, dx[rows], None, None, torch.float32)
    assert torch.isnan(dx[2:4]).all() and torch.isnan(dw).any() and torch.isfinite(db).all()


@pytest.mark.parametrize("dt,h", [(torch.bfloat16, 8), (torch.bfloat16, 24), (torch.bfloat16, 100), (torch.float32, 4),
                                  (torch.float32, 36), (torch.float32, 50)])
def test_a_mean_whose_product_with_rstd_overflows(dt, h):
    """Rows of 2^120 (their sums are exact): mean * rstd is past float32, the gradient is not."""
    say(f"norm huge mean h={h} {dt}")
    _, w, b, dy, dres = _inputs(5, h, dt, torch.float32, seed=h)
    x = torch.full((5, h), 2.0 ** 120, dtype=dt)
    dev = [t.to(DEV) for t in (x, w, b, dy, dres)]
    y, mean, rstd = K.layer_norm(*dev[:3], 1e-5)
    assert torch.equal(mean.cpu(), torch.full((5,), 2.0 ** 120)) and torch.equal(y.cpu(), b.to(dt).expand(5, h))
    for res in (None, 4):
        dx, dw, db = K.layer_norm_bwd(dev[3], dev[0], dev[1], mean, rstd, dres=None if res is None else dev[4])
        _check_backward(dy, x, w, mean, rstd, None if res is None else dres, dx, dw, db, torch.float32)


def test_offsets_past_two_gigabytes():
    """More than 2^31 elements: the last rows are what they are in a batch of their own."""
    T, h = (1 << 31) // 4096 + 40, 4096
    say(f"norm T={T} h={h}")
    x = torch.empty(T, h, dtype=torch.bfloat16, device=DEV)
    x.view(torch.int16).random_(0, 0x4000, generator=torch.Generator(device=DEV).manual_seed(1))   # finite, [0, 2)
    w, b = (t.to(DEV) for t in _inputs(1, h, torch.bfloat16, torch.float32)[1:3])
    y, mean, rstd = K.layer_norm(x, w, b)
    tail = K.layer_norm(x[-37:].clone(), w, b)
    assert torch.equal(y[-37:], tail[0]) and torch.equal(mean[-37:], tail[1]) and torch.equal(rstd[-37:], tail[2])
    dx, dw, db = K.layer_norm_bwd(y, x, w, mean, rstd)
    t2 = K.layer_norm_bwd(y[-37:].clone(), x[-37:].clone(), w, mean[-37:].clone(), rstd[-37:].clone())
    assert torch.equal(dx[-37:], t2[0])
    want = torch.zeros(h, dtype=torch.float64, device=DEV)
    for part in y.split(1 << 16):
        want += part.sum(0, dtype=torch.float64)
    assert ((db.double() - want).abs() <= (T // 16 + 600) * 2.0 ** -24 * T * 20).all()


def test_the_longest_rows():
    h = (1 << 26) - 3
    say(f"norm h={h}")
    x, w, b, dy, _ = _inputs(1, h, torch.bfloat16, torch.float32)
    dev = [t.to(DEV) for t in (x, w, b, dy)]
    y, mean, rstd = K.layer_norm(*dev[:3], 1e-5)
    _check_forward(x, w, b, 1e-5, y, mean, rstd)
    dx, dw, db = K.layer_norm_bwd(dev[3], dev[0], dev[1], mean, rstd)
    _check_backward(dy, x, w, mean, rstd, None, dx, dw, db, torch.float32)


def test_refusals():
    x = torch.zeros(4, 64, device=DEV, dtype=torch.bfloat16)
    w = torch.ones(64, device=DEV)
    _, mean, rstd = K.layer_norm(x, w, w)
    bad = [lambda: K.layer_norm(x, w[:32].contiguous(), None), lambda: K.layer_norm(x, w.double(), None),
           lambda: K.layer_norm(x, w, w.bfloat16()), lambda: K.layer_norm(x.float(), w.bfloat16(), None),
           lambda: K.layer_norm(x.half(), None, None), lambda: K.layer_norm(x[0], None, None),
           lambda: K.layer_norm(x.t(), None, None), lambda: K.layer_norm(x, w.cpu(), None),
           lambda: K.layer_norm(x, w, w, -1.0), lambda: K.layer_norm(torch.empty(4, 0, device=DEV)),
           lambda: K.layer_norm_bwd(x[:3], x, w, mean, rstd), lambda: K.layer_norm_bwd(x.float(), x, w, mean, rstd),
           lambda: K.layer_norm_bwd(x, x, w, mean[:3], rstd), lambda: K.layer_norm_bwd(x, x, w, mean.double(), rstd),
           lambda: K.layer_norm_bwd(x, x, w, mean, rstd, dres=x[:2]),
           lambda: layer.layer_norm(torch.empty(4, 0, device=DEV))]
    for i, f in enumerate(bad):
        with pytest.raises(RuntimeError):
            f()
            pytest.fail(f"call {i} was taken")


# ----------------------------------------------------------------------------- autograd, graphs, streams


def test_autograd_against_the_formula_and_against_differences():
    say("norm autograd")
    g = torch.Generator().manual_seed(2)
    x = torch.randn(2, 3, 24, generator=g, dtype=torch.float64).to(DEV).requires_grad_(True)
    w = torch.randn(24, generator=g, dtype=torch.float64).to(DEV).requires_grad_(True)
    b = torch.randn(24, generator=g, dtype=torch.float64).to(DEV).requires_grad_(True)
    assert torch.autograd.gradcheck(lambda *a: layer.layer_norm(*a, 1e-3), (x, w, b))
    assert torch.autograd.gradcheck(lambda *a: layer.layer_norm(*a), (x, None, b))
    with pytest.raises(RuntimeError, match="once_differentiable"):   # no second derivative, and it says so
        dx, = torch.autograd.grad(layer.layer_norm(x, w, b).square().sum(), x, create_graph=True)
        dx.sum().backward()
    # A transposed view goes in and a strided gradient comes back.
    xt = torch.randn(24, 10, generator=g, dtype=torch.float64).to(DEV).requires_grad_(True)
    y = layer.layer_norm(xt.t(), w, b)
    dy = torch.randn(24, 10, generator=g, dtype=torch.float64).to(DEV).t()
    got = torch.autograd.grad(y, (xt, w, b), dy)
    x64 = xt.detach().cpu().t().contiguous().requires_grad_(True)
    w64, b64 = w.detach().cpu().requires_grad_(True), b.detach().cpu().requires_grad_(True)
    c = x64 - x64.mean(1, keepdim=True)
    want = torch.autograd.grad(c / (c.pow(2).mean(1, keepdim=True) + 1e-5).sqrt() * w64 + b64, (x64, w64, b64), dy.cpu())
    for a, e in zip((got[0].t(), got[1], got[2]), want):
        torch.testing.assert_close(a.cpu(), e, rtol=1e-12, atol=1e-12)


@pytest.mark.parametrize("T,h", [(5, 4096), (700, 1000)])
def test_captured_and_replayed(T, h):
    """Two captured graphs that share nothing but their inputs, replayed between eager calls."""
    x, w, b, dy, dres = (t.to(DEV) for t in _inputs(T, h, torch.bfloat16, torch.float32, seed=9))
    say(f"norm graph T={T} h={h}")
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        K.layer_norm_bwd(dy, x, w, *K.layer_norm(x, w, b)[1:], dres=dres)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=side):
            y, mean, rstd = K.layer_norm(x, w, b)
            out = (y, *K.layer_norm_bwd(dy, x, w, mean, rstd, dres=dres))
        graphs.append((gr, out))
    for i in range(4):
        x.copy_(_inputs(T, h, torch.bfloat16, torch.float32, seed=20 + i)[0])
        y, mean, rstd = K.layer_norm(x, w, b)
        want = (y, *K.layer_norm_bwd(dy, x, w, mean, rstd, dres=dres))
        for gr, out in graphs if i % 2 else graphs[::-1]:
            gr.replay()
        torch.cuda.synchronize()
        for gr, out in graphs:
            assert all(torch.equal(a, c) for a, c in zip(out, want)), i


def test_captured_autograd():
    """Forward and backward of the autograd function in one graph, on inputs that no eager graph holds."""
    x, w, b, dy, _ = (t.to(DEV) for t in _inputs(300, 520, torch.bfloat16, torch.float32, seed=4))
    say("norm autograd graph")

    def step():
        leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
        y = layer.layer_norm(*leaves)
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr, stream=side):
        out = step()
    for i in range(3):
        x.copy_(_inputs(300, 520, torch.bfloat16, torch.float32, seed=30 + i)[0])
        want = step()
        gr.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(out, want)), i


def test_two_streams_at_once():
    say("norm on two streams")
    sets = [[t.to(DEV) for t in _inputs(2000, h, torch.bfloat16, torch.float32, seed=h)] for h in (2048, 2056)]
    want = []
    for x, w, b, dy, dres in sets:
        y, m, r = K.layer_norm(x, w, b)
        want.append((y, *K.layer_norm_bwd(dy, x, w, m, r, dres=dres)))
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in sets], [[], []]
    for _ in range(5):
        for i, (x, w, b, dy, dres) in enumerate(sets):
            with torch.cuda.stream(streams[i]):
                y, m, r = K.layer_norm(x, w, b)
                got[i].append((y, *K.layer_norm_bwd(dy, x, w, m, r, dres=dres)))
    torch.cuda.synchronize()
    for i in range(2):
        for out in got[i]:
            assert all(torch.equal(a, c) for a, c in zip(out, want[i]))


# ----------------------------------------------------------------------------- in front of the layer


def _block64(x, p, cfg, topi):
    """The pre-norm block in float64 with given expert choices."""
    c = x - x.mean(1, keepdim=True)
    n = c / (c.pow(2).mean(1, keepdim=True) + cfg.norm_eps).sqrt() * p["norm.weight"] + p["norm.bias"]
    gates = torch.softmax((n @ p["router.weight"].t()).gather(1, topi), 1)
    out = x
    for e in range(cfg.num_experts):
        z = n @ p[f"experts.{e}.fc1.weight"].t()
        gate, up = z.chunk(2, 1)
        y = (torch.nn.functional.silu(gate) * up) @ p[f"experts.{e}.fc2.weight"].t()
        out = out + ((topi == e) * gates).sum(1, keepdim=True) * y
    for s in range(cfg.num_shared):
        gate, up = (n @ p[f"shared_experts.{s}.fc1.weight"].t()).chunk(2, 1)
        out = out + (torch.nn.functional.silu(gate) * up) @ p[f"shared_experts.{s}.fc2.weight"].t()
    return out


# bfloat16: the layer's own bar against float64 (its products read bfloat16 rows), which the norm's half step
# of 2^-8 on those rows is part of.
@pytest.mark.parametrize("dt,shared,tol", [(torch.float64, 0, 1e-10), (torch.float32, 1, 2e-5), (torch.bfloat16, 0, 2e-2),
                                           (torch.bfloat16, 2, 2e-2)])
def test_pre_norm_block_against_float64(dt, shared, tol):
    cfg = moe.MoEConfig(hidden=128, ffn=96, num_experts=6, top_k=2, tokens=200, dtype=dt, act="swiglu", norm="layer",
                        num_shared=shared, device=DEV)
    say(f"pre-norm block {dt} shared={shared}")
    params = {k: torch.nn.Parameter(moe.init_param(cfg, s)) for k, s in moe.moe_specs(cfg).items() if s.trainable}
    with torch.no_grad():
        params["norm.weight"].add_(seeded((128,), 1, 0.1).to(DEV))
        params["norm.bias"].add_(seeded((128,), 2, 0.1).to(DEV))
    x = (seeded((200, 128), 3, 2.0) + 0.5).to(DEV, dt).requires_grad_(True)
    dout = seeded((200, 128), 4).to(DEV, dt)
    out = moe.reference_forward(cfg, params, x)
    out.backward(dout)
    n = K.layer_norm(x.detach(), params["norm.weight"].detach(), params["norm.bias"].detach(), cfg.norm_eps)[0]
    topi, _ = moe.route(cfg, n, params["router.weight"])
    p64 = {k: v.detach().cpu().double().requires_grad_(True) for k, v in params.items()}
    x64 = x.detach().cpu().double().requires_grad_(True)
    ref = _block64(x64, p64, cfg, topi.cpu())
    ref.backward(dout.cpu().double())
    pairs = {"out": (out, ref), "dx": (x.grad, x64.grad)} | {k: (params[k].grad, p64[k].grad) for k in params}
    for k, (a, e) in pairs.items():
        e = e.detach()
        err = float((a.detach().cpu().double() - e).abs().max() / e.abs().max())
        assert err <= tol, (k, err)
    with torch.no_grad():
        again = moe.reference_forward(cfg, params, x)
    assert torch.equal(again, out)


def test_pre_norm_block_with_frozen_parts():
    """Any of x, the norm and the experts may go without gradients; the others' stay the same bits."""
    cfg = moe.MoEConfig(hidden=64, ffn=64, num_experts=4, top_k=2, tokens=50, dtype=torch.bfloat16, act="swiglu",
                        norm="layer", device=DEV)
    say("pre-norm block, frozen parts")
    names = [k for k, s in moe.moe_specs(cfg).items() if s.trainable]
    x0, dout = seeded((50, 64), 1).to(DEV, torch.bfloat16), seeded((50, 64), 2).to(DEV, torch.bfloat16)

    def grads(frozen):
        params = {k: moe.init_param(cfg, moe.moe_specs(cfg)[k]).requires_grad_(k not in frozen) for k in names}
        x = x0.clone().requires_grad_("x" not in frozen)
        moe.reference_forward(cfg, params, x).backward(dout)
        return {**{k: p.grad for k, p in params.items()}, "x": x.grad}

    full = grads(())
    for frozen in (("x",), ("norm.weight", "norm.bias"), ("x", "norm.bias"), ("x", "norm.weight", "norm.bias")):
        got = grads(frozen)
        for k, g in got.items():
            if k in frozen:
                assert g is None, k
            elif k.startswith("norm."):   # sums may take another order where dx is not wanted
                torch.testing.assert_close(g, full[k], rtol=1e-4, atol=1e-4)
            else:
                assert torch.equal(g, full[k]), (frozen, k)


def test_norm_none_keeps_the_layer_as_it_was():
    cfg = moe.MoEConfig(hidden=64, ffn=64, num_experts=4, top_k=2, tokens=50, dtype=torch.bfloat16, act="swiglu", device=DEV)
    params = {k: moe.init_param(cfg, s) for k, s in moe.moe_specs(cfg).items()}
    assert not any(k.startswith("norm.") for k in params)


def test_send_side_routes_and_sends_normalised_rows():
    from resihp_megatron_amd.placement import ExpertPlacement

    cfg = moe.MoEConfig(hidden=64, ffn=32, num_experts=4, top_k=2, tokens=40, dtype=torch.float32, norm="layer", device=DEV)
    params = {k: torch.nn.Parameter(moe.init_param(cfg, s)) for k, s in moe.moe_specs(cfg).items()}
    place = ExpertPlacement(4, (("a", "b"),), {"a": (0, 1), "b": (2, 3)})
    rt = moe.EPRuntime(cfg, place, "a", ["a", "b"], None, None, params)
    x = (seeded((40, 64), 6) * 3 + 1).to(DEV)
    say("pre-norm send")
    rows, counts, splits, plan, gates = rt.send(x)
    n = K.layer_norm(x, params["norm.weight"].detach(), params["norm.bias"].detach(), cfg.norm_eps)[0]
    topi, g2 = moe.route(cfg, n, params["router.weight"])
    assert torch.equal(gates, g2) and int(counts.sum()) == 80
    assert torch.equal(rows[plan.row.long()], n.repeat_interleave(2, 0))


def test_fp8_block_behind_a_norm():
    from resihp_megatron_amd.fp8 import Fp8State

    cfg = moe.MoEConfig(hidden=256, ffn=128, num_experts=4, top_k=2, dtype=torch.bfloat16, act="swiglu", norm="layer", device=DEV)
    specs = moe.moe_specs(cfg)
    params = {k: torch.nn.Parameter(moe.init_param(cfg, s)) for k, s in specs.items()}
    fc1, fc2 = ([params[f"experts.{e}.{w}.weight"] for e in range(4)] for w in ("fc1", "fc2"))
    meta = layer.LayerMeta(num_experts=4, top_k=2, ffn=128, act="swiglu")
    x = seeded((96, 256), 1, 3.0).to(DEV, torch.bfloat16).requires_grad_(True)
    dout = seeded((96, 256), 2).to(DEV, torch.bfloat16)
    say("fp8 pre-norm block")
    norm = layer.Norm(params["norm.weight"], params["norm.bias"])
    got = []
    for split in (False, True):
        st = Fp8State(4, 16, device=DEV)
        if split:   # the same layer over rows normalised outside, minus its residual
            n = layer.layer_norm(x, *norm)
            out = layer.moe_layer(meta, n, params["router.weight"], None, fc1, fc2, fp8=st)[0]
        else:
            out = layer.moe_layer(meta, x, params["router.weight"], None, fc1, fc2, fp8=st, norm=norm)[0]
        got.append(torch.autograd.grad(out, [params["router.weight"], *fc1, *fc2], dout))
    for a, c in zip(*got):   # the weights' gradients do not see the residual
        assert torch.equal(a, c)
