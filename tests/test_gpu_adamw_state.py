"""What an AdamW optimizer holds beside its moments: which tensors its plan steps, which of its settings a step
reads, which states it takes."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from _helpers import DEV, say, seeded
from oracle import adamw_ref as R
from resihp_megatron_amd import kernels as K
from resihp_megatron_amd import moe

pytestmark = pytest.mark.gpu

HYPER = dict(lr=2e-3, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.1)


def _param(n, seed, dtype=torch.float32):
    return torch.nn.Parameter(seeded((n,), seed, 0.05).to(dtype).to(DEV))


@pytest.mark.parametrize("bits", [32, 8])
def test_a_parameter_retyped_at_its_address_is_stepped_as_its_new_type(bits):
    """float32 to bfloat16 over one buffer: the bytes behind the smaller tensor stay as they were."""
    n = 3000
    buf = torch.full((2 * n,), 7.0, device=DEV)
    buf[:n] = seeded((n,), 1, 0.05).to(DEV)
    p = torch.nn.Parameter(buf[:n])
    opt = moe.AdamW({"p": p}, **HYPER, state_bits=bits)
    p.grad = seeded((n,), 2).to(DEV)
    say(f"adamw retyped parameter {bits}")
    opt.step()
    p.grad = None
    p.data = buf.view(torch.bfloat16)[:n]
    p.data.copy_(seeded((n,), 3, 0.05))
    p.grad = seeded((n,), 4).to(torch.bfloat16).to(DEV)
    behind, before = buf[n // 2:].clone(), p.detach().float().cpu().numpy().copy()
    opt.step()
    assert torch.equal(buf[n // 2:].view(torch.int32), behind.view(torch.int32))
    m, v = (t.float().cpu().numpy()[:n] for t in opt.moments())
    if bits == 32:      # (codes of 8 bits are what m and v became, not what the weight was stepped with)
        want = R.weight(before, m, v, np.float64, *HYPER.values(), 2)
        tol = 2.0 ** -24 * (4 * np.abs(before) + 16 * np.abs(want - before))
        assert (np.abs(p.detach().double().cpu().numpy() - want) <= tol + 2.0 ** -8 * (np.abs(want) + tol)).all()
    assert not torch.equal(p.detach().float().cpu(), torch.from_numpy(before))
    p.grad = None
    p.data = torch.zeros(n, dtype=torch.float64, device=DEV)
    with pytest.raises(RuntimeError):
        opt.step()
    assert opt.step_count == 2


def test_a_parameter_put_in_anothers_place_is_stepped():
    """As Adam steps it: the optimizer's dict says whom the moments belong to, the plan follows."""
    say("adamw replaced parameter")
    a, b, other = _param(300, 1), _param(20, 2), _param(300, 1)
    opt = moe.AdamW({"a": a, "b": b}, **HYPER)
    for p in (a, b, other):
        p.grad = torch.ones_like(p)
    opt.step()
    kept = a.detach().clone()
    other.data.copy_(a.data)
    opt.params["a"] = other
    opt.step()
    assert torch.equal(a, kept) and not torch.equal(other, kept) and opt.step_count == 2
    opt.params["new"] = _param(8, 3)
    with pytest.raises(KeyError, match="new"):
        opt.step()
    assert opt.step_count == 2


def test_no_decay_is_read_at_every_step():
    say("adamw no_decay")
    opt = moe.AdamW({"a": _param(300, 1), "b": _param(20, 2)}, lr=0.5, weight_decay=1.0)
    for want in ((), ("a",), ("a", "b"), ("b",)):
        opt.no_decay = set(want)
        before = {n: p.detach().clone() for n, p in opt.params.items()}
        opt.step()      # no gradients: only the decay moves a weight
        for n, p in opt.params.items():
            assert torch.equal(p, before[n] if n in want else before[n] * 0.5), (want, n)
    opt.no_decay.add("c")
    with pytest.raises(ValueError, match="no_decay"):
        opt.step()


@pytest.mark.parametrize("bits", [32, 8])
def test_a_graph_outlives_a_moved_parameter(bits):
    """A captured step reads its plan's image at every replay: the optimizer keeps that plan when it makes another,
    and the graph goes on stepping the storage that it was captured with."""
    say(f"adamw graph after a move {bits}")
    n = 3000
    opt = moe.AdamW({"p": _param(n, 1), "q": _param(40, 2)}, **HYPER, state_bits=bits)
    p = opt.params["p"]
    for t in opt.params.values():
        t.grad = torch.ones_like(t)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        opt.step()
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr, stream=side):
        opt.step()
    old, size = p.data, opt._plan.dev_image.numel()
    p.data = old.clone()
    opt.step()
    torch.cuda.synchronize()
    junk = [torch.full((size,), 0xAB, dtype=torch.uint8, device=DEV) for _ in range(64)]   # takes what was given back
    held = [old, opt.params["q"].data, *(t for b in opt.state.values() for t in b.values())]
    for _ in range(3):
        saved, moved = [t.clone() for t in held], p.detach().clone()
        gr.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in held]
        assert torch.equal(p.detach(), moved) and not torch.equal(got[0], saved[0])
        for t, s in zip(held, saved):
            t.copy_(s)
        new, p.data, opt.step_count = p.data, old, 1
        opt.step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, held))
        p.data = new
    assert len(junk) == 64


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("b2", [0.999, 0.999999])
def test_small_second_moments_under_a_large_bias_correction(bits, b2):
    """At the first steps the root is multiplied by up to 1 / sqrt(1 - b2) before eps is added: a subnormal second
    moment shows beside an eps that hides it without that factor.  The weights are zeros, so that the update's 16 u
    are all of the bound."""
    n = 4096
    for eps in (2.1e-12, 1e-10, 1e-8):
        hyper = dict(lr=1.0, betas=(0.9, b2), eps=eps, weight_decay=0.0)
        g32 = (seeded((n,), 2) * 10.0 ** torch.linspace(-21, -12, n))
        p = torch.zeros(n, device=DEV)
        sdt = torch.uint8 if bits == 8 else torch.float32
        m, v = torch.zeros(n, dtype=sdt, device=DEV), torch.zeros(n, dtype=sdt, device=DEV)
        sc = [torch.zeros(n // 128, 2, dtype=torch.uint8, device=DEV)] if bits == 8 else None
        plan = K.AdamWPlan([p], [m], [v], sc, keys=[1])
        say(f"adamw eps={eps} b2={b2} {bits}")
        K.adamw_step(plan, [g32.to(DEV)], *hyper.values(), 1)
        _, m32, v32 = R.update(np.zeros(n), g32.numpy(), np.zeros(n), np.zeros(n), np.float32, *hyper.values(), 1)
        want = R.weight(np.zeros(n), m32, v32, np.float64, *hyper.values(), 1)
        # m / d and a * it may be subnormal themselves: half of the smallest step each, times a at most.
        tol = 2.0 ** -24 * 16 * np.abs(want) + 2.0 ** -149 * 16
        bad = ~(np.abs(p.cpu().double().numpy() - want) <= tol)
        assert not bad.any(), (int(bad.sum()), float((np.abs(p.cpu().double().numpy() - want) / np.abs(want))[bad].max()))


def test_negative_and_negative_zero_second_moments():
    """-0 is a zero and leaves its block alone; a negative second moment has no root: its block reads as NaN."""
    say("moments encode signs")
    g = np.random.default_rng(5)
    n = 128 * 5 + 40
    m = g.standard_normal(n).astype(np.float32)
    v = (g.standard_normal(n) ** 2).astype(np.float32)
    v[[3, 128 * 2 + 5, n - 1]] = 0.0
    plain = v.copy()
    v[[3, 128 * 2 + 5, n - 1]] = -0.0
    v[128 + 7] = -1e-6
    v[128 * 3 + 100] = -np.inf
    out = [torch.zeros(n, dtype=torch.uint8, device=DEV), torch.zeros(n, dtype=torch.uint8, device=DEV),
           torch.zeros(6, 2, dtype=torch.uint8, device=DEV)]
    K.moments_encode(torch.from_numpy(m).to(DEV), torch.from_numpy(v).to(DEV), *out)
    want = R.encode(m, plain, R.nearest(n))
    for b in (1, 3):
        want[1][128 * b:128 * (b + 1)] = 0
        want[2][b, 1] = 255
    for t, e in zip(out, want):
        assert np.array_equal(t.cpu().numpy(), e)
    got = K.moments_decode(*out)[1].float().cpu().numpy().reshape(-1)
    bad = np.zeros(n, bool)
    bad[128:256] = bad[384:512] = True
    assert np.array_equal(np.isnan(got), bad)


def _state(bits):
    opt = moe.AdamW({"a": _param(300, 1, torch.bfloat16), "b": _param(20, 2, torch.bfloat16)}, **HYPER, state_bits=bits,
                    master_weights=True)
    for p in opt.params.values():
        p.grad = torch.ones_like(p)
    opt.step()
    return opt


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("change", [
    lambda t: t.pop("param/b"),
    lambda t: t.pop("exp_avg_sq/b"),
    lambda t: t.update({"exp_avg/b": t["exp_avg/b"].to(torch.uint8 if t["exp_avg/b"].is_floating_point() else torch.float32)}),
    lambda t: t.update({"exp_avg/b": t["exp_avg/b"][:1]}),
    lambda t: t.update({"exp_avg_sq/b": t["exp_avg_sq/b"].view(2, 10)}),
    lambda t: t.update({"param/b": t["param/b"][:1]}),
    lambda t: t.update({"master/b": t["master/b"][:1]}),
    lambda t: t.update({"param/b": t["param/b"].to(torch.uint8)}),
    lambda t: t.update({"master/b": t["master/b"].to(torch.int32)}),
    lambda t: t.update({"exp_avg/b": t["exp_avg/b"].to(torch.int32), "exp_avg_sq/b": t["exp_avg_sq/b"].to(torch.int32)}),
], ids=["no-param", "no-moment", "mixed-widths", "short-moment", "reshaped-moment", "short-param", "short-master",
        "int-param", "int-master", "int-moments"])
def test_a_state_that_does_not_fit_changes_nothing(bits, change):
    saved = {k: t.clone() for k, t in _state(bits).state_tensors().items()}
    opt = _state(bits)
    opt.step()
    before = {k: t.clone() for k, t in opt.state_tensors().items()}
    change(saved)
    say(f"adamw state that does not fit {bits}")
    with pytest.raises((KeyError, ValueError)):
        opt.load_state_tensors(saved, 1)
    assert opt.step_count == 2
    for k, t in opt.state_tensors().items():
        assert torch.equal(t, before[k]), k


@pytest.mark.parametrize("bits", [32, 8])
def test_scales_that_do_not_fit_change_nothing(bits):
    """Of one row (which a copy would spread over all blocks), or of another type."""
    saved = {k: t.clone() for k, t in _state(8).state_tensors().items()}
    opt = _state(bits)
    before = {k: t.clone() for k, t in opt.state_tensors().items()}
    for sc in (saved["scales/a"][:1], saved["scales/a"].float(), saved["scales/a"].view(-1)):
        with pytest.raises(ValueError):
            opt.load_state_tensors({**saved, "scales/a": sc}, 1)
        for k, t in opt.state_tensors().items():
            assert torch.equal(t, before[k]), k
    opt.load_state_tensors(saved, 7)
    assert opt.step_count == 7 and torch.equal(opt.params["a"].detach(), saved["param/a"])


@pytest.mark.parametrize("scale", [1.0, 1e60])
def test_clipped_step_of_float64_weights(scale):
    """The coefficient that clips float64 gradients is float64: neither its rounding to float32 nor float32's range
    comes into the step.  The norm's sum of 5000 squares and the coefficient are off by at most 40 u, m by 4 u more
    and v by twice that; the update's own 16 u."""
    n = 5000
    opt = moe.AdamW({"p": torch.nn.Parameter(seeded((n,), 1, 0.05).double().to(DEV))}, **HYPER, max_grad_norm=0.5)
    p = opt.params["p"]
    p.grad = seeded((n,), 2).double().to(DEV) * scale
    w, g = p.detach().cpu().numpy().copy(), p.grad.cpu().numpy()
    say(f"adamw f64 clip {scale}")
    opt.step()
    norm = float(np.sqrt((g ** 2).sum()))
    coef = min(1.0, 0.5 / (norm + 1e-6))
    u = 2.0 ** -53
    got = opt.grad_norm.tolist()
    assert opt.grad_norm.dtype == torch.float64
    assert abs(got[0] - norm) <= 40 * u * norm and abs(got[1] - coef) <= 44 * u * coef
    m, v = (1 - 0.9) * coef * g, (1 - 0.95) * (coef * g) ** 2
    assert (np.abs(opt.state["p"]["exp_avg"].cpu().numpy() - m) <= 52 * u * np.abs(m)).all()
    assert (np.abs(opt.state["p"]["exp_avg_sq"].cpu().numpy() - v) <= 104 * u * v).all()
    want = R.weight(w, m, v, np.float64, *HYPER.values(), 1)
    tol = u * (4 * np.abs(w) + 130 * np.abs(want - w * (1 - HYPER["lr"] * HYPER["weight_decay"])))
    assert (np.abs(p.detach().cpu().numpy() - want) <= tol).all()


def test_a_float64_coefficient_is_for_float64_weights():
    say("adamw float64 coefficient")
    z = lambda n, dt=torch.float32: torch.zeros(n, dtype=dt, device=DEV)  # noqa: E731
    one = torch.ones(1, dtype=torch.float64, device=DEV)
    step = lambda plan, dt, c: K.adamw_step(plan, [z(10, dt)], 1e-3, (0.9, 0.999), 1e-8, 0.0, 1, c)  # noqa: E731
    plans = {dt: K.AdamWPlan([z(10, dt)], [z(10, dt)], [z(10, dt)]) for dt in (torch.float32, torch.float64)}
    step(plans[torch.float64], torch.float64, one)
    step(plans[torch.float64], torch.float64, one.float())
    with pytest.raises(RuntimeError):
        step(plans[torch.float32], torch.float32, one)
    g = [seeded((777,), 1).to(DEV), seeded((5,), 2).to(torch.bfloat16).to(DEV)]
    assert torch.equal(K.grad_norm(g, 0.5, torch.float64).float(), K.grad_norm(g, 0.5))
    with pytest.raises(RuntimeError):
        K.grad_norm(g, 0.5, torch.bfloat16)
