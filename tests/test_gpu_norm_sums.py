"""Layer norm's sums on the GPU where they are long: over the columns of rows past the registers, over many rows."""

from __future__ import annotations

import pytest
import torch

from _helpers import DEV, say
from resihp_megatron_amd import kernels as K

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
LONG = [(torch.bfloat16, h) for h in (16392, 20001, (1 << 20) + 3, 1 << 24, (1 << 26) - 3, 1 << 26)] + \
       [(torch.float32, h) for h in (8196, 20001, (1 << 20) + 3, (1 << 24) + 1, 1 << 26)]


def _close(got, want, tol, what):
    bad = ~((got.double() - want).abs() <= tol)
    assert not bad.any(), (what, int(bad.sum()), float((got.double() - want).abs()[bad].max()))


@pytest.mark.parametrize("dt,h", LONG)
def test_a_long_constant_row_gives_the_bias(dt, h):
    say(f"norm constant h={h} {dt}")
    x = torch.full((2, h), 0.1, device=DEV).to(dt)
    x[1] = -7.3
    b = torch.full((h,), 0.25, device=DEV)
    y, mean, rstd = K.layer_norm(x, None, b, 1e-5)
    assert torch.equal(mean, x[:, 0].float())
    assert torch.equal(y, torch.full_like(y, 0.25))
    assert ((rstd.double() - 1e-5 ** -0.5).abs() <= 4 * U * 1e-5 ** -0.5).all()


@pytest.mark.parametrize("dt,h", LONG)
def test_long_rows_against_float64(dt, h):
    """Sums that no length dims: D additions in float (a chunk of at most eight values in pairs), the rest in double.
    Every element's part is seen: the rows are zeros but for a few large ones, in the last chunk and behind it."""
    D = 4
    g = torch.Generator(device=DEV).manual_seed(h)
    for at in (None, h - 1, h // 8 * 8 - 1, 0, 5000):
        say(f"norm h={h} {dt} at={at}")
        if at is None:
            x = (torch.rand(1, h, generator=g, device=DEV) + 0.5).to(dt)      # one sign: no errors cancel
        else:
            x = torch.zeros(1, h, device=DEV, dtype=dt)
            x[0, at] = 1024.0
        y, mean, rstd = K.layer_norm(x, None, None, 1e-5)
        xd = x.double()
        m = xd.mean(1, keepdim=True)
        c = xd - m
        var = (c * c).mean(1, keepdim=True)
        r = (var + 1e-5).rsqrt()
        em = (D + 2) * U * xd.abs().mean(1, keepdim=True)
        ev = (D + 4) * U * var + em * em + 2 * U * (c.abs() * xd.abs()).mean(1, keepdim=True)
        er = r * (0.5 * ev / (var + 1e-5) + 4 * U)
        _close(mean, m[:, 0], em[:, 0], "mean")
        _close(rstd, r[:, 0], er[:, 0], "rstd")
        want = c * r
        tol = r * (em + U * c.abs()) + c.abs() * er + 2 * U * c.abs() * r
        _close(y, want, tol * 1.01 + (want.abs() + tol) * torch.finfo(dt).eps / 2, "y")
        del y, c, want, tol
        # Backward: the same for the sums of g and of g xh, whose terms have roundings of their own.
        dy = (torch.rand(1, h, generator=g, device=DEV) + 0.5).to(dt)
        dx, dw, db = K.layer_norm_bwd(dy, x, None, mean, rstd)
        md, rd, dyd = mean.double()[:, None], rstd.double()[:, None], dy.double()
        xh = (xd - md) * rd
        c1, a1 = (dyd * xh).mean(1, keepdim=True), (dyd * xh).abs().mean(1, keepdim=True)
        c2 = dyd.mean(1, keepdim=True)
        want = rd * (dyd - c2 - xh * c1)
        tol = rd * U * (3 * dyd + (D + 4) * c2 + xh.abs() * ((D + 8) * a1 + 6 * c1.abs()) + 4 * c2)
        _close(dx, want, tol * 1.01 + (want.abs() + tol) * torch.finfo(dt).eps / 2, "dx")
        wt = (dyd * xh)[0]
        _close(dw, wt, 4 * U * wt.abs() * 1.01 + wt.abs() * torch.finfo(dt).eps / 2, "dw")
        assert torch.equal(db, dy[0])


@pytest.mark.parametrize("dt,h,T,lane", [(torch.bfloat16, 5, (1 << 24) + 77, 64), (torch.float32, 3, (1 << 24) + 77, 64),
                                         (torch.bfloat16, 20001, 3000, 58), (torch.bfloat16, 16392, 40000, 500)])
def test_column_sums_of_many_rows_outside_the_registers(dt, h, T, lane):
    """A lane's rows are summed in double, 64 in float at a time (rows under a chunk), or few are (at most 512): that
    makes ``lane`` additions.  Beside them
    there are the rounding of the lane's sum to float, three additions over the block's waves, and of at most 256
    slices on 16 waves 15 + 15 additions, and the result's rounding."""
    say(f"norm columns T={T} h={h} {dt}")
    x = torch.full((T, h), 1.0, dtype=dt, device=DEV)
    x[:, 1] = 3.0
    dy = torch.full((T, h), 0.1, device=DEV).to(dt)
    w = torch.ones(h, device=DEV, dtype=torch.float32)
    mean, rstd = torch.full((T,), 0.5, device=DEV), torch.full((T,), 0.3, device=DEV)
    _, dw, db = K.layer_norm_bwd(dy, x, w, mean, rstd, need_x=False)
    want_b = T * dy[0].double()
    want_w = (dy[0].double() * (x[0].double() - 0.5) * rstd[0].double()) * T
    _close(db, want_b, (36 + lane) * U * want_b.abs(), "db")
    _close(dw, want_w, (39 + lane) * U * want_w.abs(), "dw")      # each term: the centred value, xh and the product


@pytest.mark.parametrize("T,h", [(1 << 28, 4), (300_000, 8188)])
def test_column_sums_of_very_many_rows(T, h):
    """A group of lanes adds at most 512 rows in float; then there are 3 additions between groups of a wave, at most 4
    between a block's parts, the partial rows on 16 waves (T / 64 / 512 / 16 for the short rows) and 15 more, and the
    roundings of a term (3) and of the result."""
    say(f"norm columns T={T} h={h}")
    x, dy = torch.full((T, h), 1.0, device=DEV), torch.full((T, h), 0.1, device=DEV)
    mean, rstd = torch.full((T,), 0.5, device=DEV), torch.full((T,), 0.3, device=DEV)
    _, dw, db = K.layer_norm_bwd(dy, x, None, mean, rstd, need_x=False)
    tol = (512 + 3 + 4 + max(37, -(-T // (64 * 512 * 16))) + 15 + 4) * U
    want_b = T * dy[0].double()
    want_w = (dy[0].double() * 0.5 * rstd[0].double()) * T
    _close(db, want_b, tol * want_b.abs(), "db")
    _close(dw, want_w, tol * want_w.abs(), "dw")


def _rows(dt, h, res):
    """Rows that the register kernels' 256 blocks hold at a time in the backward: each of its groups has one.  (How
    many threads have a row is the kernels' choice; what counts here is that groups walk several rows.)"""
    chunks = -(-h * torch.finfo(dt).bits // 128)
    for tpr, nv in ((8, 2), (16, 2), (32, 2), (64, 2), (64, 3), (64, 4), (128, 2), (192, 2), (256, 2), (384, 2), (512, 2)):
        if chunks <= tpr * nv and (nv < 4 or not res and h * torch.finfo(dt).bits % 128 == 0):
            threads = 576 if tpr == 192 else 512 if tpr < 384 else 768 if tpr == 384 else tpr
            return 256 * (threads // tpr)
    return 256


# Rows on 8, 16 and 32 lanes, on a wave with two, three and four chunks, on 128 to 1024 threads; whole and cut chunks.
@pytest.mark.parametrize("dt,h", [(torch.bfloat16, h) for h in (64, 100, 250, 500, 1000, 1100, 1536, 1800, 2048, 2500,
                                                                2816, 4000, 4099, 6000, 6144, 8000, 12001, 16384)] +
                         [(torch.float32, h) for h in (60, 250, 700, 768, 1000, 1400, 3000, 4000, 8192)])
@pytest.mark.parametrize("res", [False, True])
def test_groups_that_walk_several_rows(dt, h, res):
    """Two or three rows a group, against float64: the row after the first has its loads ahead, or none, and its terms
    in the same column sums.  A column's sum: three additions in a lane, three between a wave's groups, four
    between a block's parts, 16 + 15 over the partial rows, the term's own three roundings and the result's."""
    T = 2 * _rows(dt, h, res) + 37
    say(f"norm several rows T={T} h={h} {dt} res={res}")
    g = torch.Generator(device=DEV).manual_seed(h)
    rand = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    x, dy = (rand(T, h) * 2 + 0.3).to(dt), rand(T, h).to(dt)
    w, b, dres = 1 + 0.1 * rand(h), 0.1 * rand(h), rand(T, h).to(dt) if res else None
    y, mean, rstd = K.layer_norm(x, w, b, 1e-5)
    dx, dw, db = K.layer_norm_bwd(dy, x, w, mean, rstd, dres=dres)
    half, D = torch.finfo(dt).eps / 2, 32 + 10 + 16     # additions: in a lane, over its lanes, over the waves
    xd, dyd, wd = x.double(), dy.double(), w.double()
    m = xd.mean(1, keepdim=True)
    c = xd - m
    var = (c * c).mean(1, keepdim=True)
    r = (var + 1e-5).rsqrt()
    em = (D + 2) * U * xd.abs().mean(1, keepdim=True)
    ev = (D + 4) * U * var + em * em + 2 * U * (c.abs() * xd.abs()).mean(1, keepdim=True)
    er = r * (0.5 * ev / (var + 1e-5) + 4 * U)
    _close(mean, m[:, 0], em[:, 0], "mean")
    _close(rstd, r[:, 0], er[:, 0], "rstd")
    want = c * r * wd + b.double()
    tol = wd.abs() * (r * (em + U * c.abs()) + c.abs() * er + 2 * U * c.abs() * r) + 2 * U * (want.abs() + b.double().abs())
    _close(y, want, tol * 1.01 + (want.abs() + tol) * half, "y")
    m, r = mean.double()[:, None], rstd.double()[:, None]
    gd, xh = dyd * wd, (xd - m) * r
    c1, c2 = (gd * xh).mean(1, keepdim=True), gd.mean(1, keepdim=True)
    a1, a2 = (gd * xh).abs().mean(1, keepdim=True), gd.abs().mean(1, keepdim=True)
    want = r * (gd - c2 - xh * c1)
    tol = r * U * (3 * gd.abs() + (D + 4) * a2 + xh.abs() * ((D + 8) * a1 + 6 * c1.abs()) + 4 * c2.abs())
    if res:
        want = want + dres.double()
        tol = tol + U * want.abs()
    _close(dx, want, tol * 1.01 + (want.abs() + tol) * half, "dx")
    for got, terms, name in ((dw, dyd * xh, "dw"), (db, dyd, "db")):
        _close(got, terms.sum(0), (3 + 3 + 4 + 16 + 15 + 4) * U * terms.abs().sum(0), name)
