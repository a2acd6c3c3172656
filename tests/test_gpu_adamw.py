"""AdamW and the gradient norm on the GPU against the numpy restatement (oracle/adamw_ref.py): moments and 8-bit
codes bit for bit, weights against float64 within what the update's roundings allow.

u = 2^-24 (2^-53 for float64 weights).  The weight p keep - a (m / d): d = sqrt(v) ibc2s + eps goes through four
roundings (a square root or reciprocal of one step instead of half a step counts as two), the quotient, the
product with a and the scalars a few more: the update is off by at most 16 u of itself beside m's and v's
own errors, which come from the same float32 values here; p keep is off by 2 u, the difference by u.
"""

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
# None, a few, around the ends of vectors, blocks of 128, waves and thread blocks (1024 and 4096 elements).
SIZES = [0, 1, 3, 4, 5, 7, 8, 9, 127, 128, 129, 511, 513, 1000, 1023, 1025, 2048, 2049, 4095, 4096, 4097, 6143, 40961]


def _params(sizes, dtypes, seed):
    return {f"p{i}": torch.nn.Parameter(seeded((n,), seed + i, 0.05).to(dtypes[i % len(dtypes)]).to(DEV))
            for i, n in enumerate(sizes)}


def _f32(t):
    return t.detach().float().cpu().numpy().copy()


def _weights_ok(got, want64, before64, dtype):
    """got: the stored weight; want64 the exact one, before64 the one before the step."""
    u = 2.0 ** -53 if dtype == torch.float64 else 2.0 ** -24
    tol = u * (4 * np.abs(before64) + 16 * np.abs(want64 - before64))
    if dtype == torch.bfloat16:
        tol = tol + 2.0 ** -8 * (np.abs(want64) + tol)
    got = got.detach().double().cpu().numpy()
    bad = ~(np.abs(got - want64) <= tol)
    assert not bad.any(), (int(bad.sum()), np.abs(got - want64)[bad].max())


def _exact(p, g, m, v, hyper, step, scale=1.0, decay=True):
    """The weight in float64 from the moments as their own type holds them, and those."""
    st = np.float64 if p.dtype == np.float64 else np.float32
    h = (hyper["lr"], hyper["betas"], hyper["eps"], hyper["weight_decay"])
    _, m, v = R.update(p, g, m, v, st, *h, step, scale, decay)
    return R.weight(p, m, v, np.float64, *h, step, decay), m, v


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtypes", [(torch.float32,), (torch.bfloat16,), (torch.bfloat16, torch.float32)], ids=str)
@pytest.mark.parametrize("master", [False, True])
def test_steps_match_the_oracle(bits, dtypes, master):
    params = _params(SIZES, dtypes, 100)
    opt = moe.AdamW(params, **HYPER, state_bits=bits, master_weights=master, no_decay=("p5", "p11"), seed=(7 << 32) + 5)
    keys = {n: __import__("zlib").crc32(n.encode()) for n in params}
    say(f"adamw {bits} {dtypes} master={master}")
    for step in range(1, 5):
        hosts = {}
        for i, (n, p) in enumerate(params.items()):
            p.grad = None if (i == 9 and step == 2) else \
                (seeded(p.shape, 1000 * step + i) * 10.0 ** seeded(p.shape, 2000 * step + i)).to(p.dtype).to(DEV)
            st = opt.state[n]
            w = _f32(st["master"] if "master" in st else p)
            g = np.zeros(p.numel(), np.float32) if p.grad is None else _f32(p.grad)
            mv = R.decode(*(st[k].cpu().numpy() for k in ("exp_avg", "exp_avg_sq", "scales"))) if bits == 8 else \
                (_f32(st["exp_avg"]), _f32(st["exp_avg_sq"]))
            hosts[n] = (w, g, *mv)
        opt.step()
        torch.cuda.synchronize()
        for n, p in params.items():
            w, g, m, v = hosts[n]
            decay = n not in opt.no_decay
            st = opt.state[n]
            _, m32, v32 = R.update(w, g, m, v, np.float32, *HYPER.values(), step, 1.0, decay)
            if bits == 32:
                assert np.array_equal(_f32(st["exp_avg"]), m32) and np.array_equal(_f32(st["exp_avg_sq"]), v32), n
            else:
                want = R.encode(m32, v32, R.random_bits(p.numel(), opt.seed, step, keys[n]))
                for key, e in zip(("exp_avg", "exp_avg_sq", "scales"), want):
                    assert np.array_equal(st[key].cpu().numpy(), e), (n, key, step)
            p64, _, _ = _exact(w, g, m, v, HYPER, step, 1.0, decay)
            if "master" in st:
                _weights_ok(st["master"], p64, w.astype(np.float64), torch.float32)
                assert torch.equal(p.detach(), st["master"].to(p.dtype)), n
            else:
                _weights_ok(p, p64, w.astype(np.float64), p.dtype)


def test_float64_weights():
    params = _params(SIZES, (torch.float64,), 7)
    opt = moe.AdamW(params, **HYPER)
    say("adamw f64")
    for step in (1, 2, 3):
        before = {}
        for i, (n, p) in enumerate(params.items()):
            p.grad = seeded(p.shape, 50 * step + i).double().to(DEV)
            before[n] = [t.detach().cpu().numpy().copy() for t in (p, p.grad, opt.state[n]["exp_avg"], opt.state[n]["exp_avg_sq"])]
        opt.step()
        for n, p in params.items():
            p64, m64, v64 = _exact(*before[n], HYPER, step)
            assert np.array_equal(opt.state[n]["exp_avg"].cpu().numpy(), m64)
            assert np.array_equal(opt.state[n]["exp_avg_sq"].cpu().numpy(), v64)
            _weights_ok(p, p64, before[n][0], torch.float64)
    with pytest.raises(ValueError, match="AdamW of their own"):
        moe.AdamW({**_params([3], (torch.float64,), 1), "x": torch.nn.Parameter(torch.zeros(3, device=DEV))})
    with pytest.raises(ValueError, match="AdamW of their own"):
        moe.AdamW(_params([3], (torch.float64,), 1), state_bits=8)


@pytest.mark.parametrize("bits", [32, 8])
def test_gradients_of_another_type(bits):
    """float32 gradients (accumulated buckets) of bfloat16 weights and the reverse, through the kernels' own entry."""
    say(f"adamw grad types {bits}")
    for pdt, gdt in ((torch.bfloat16, torch.float32), (torch.float32, torch.bfloat16)):
        n = 3001
        p, g = seeded((n,), 1, 0.05).to(pdt).to(DEV), seeded((n,), 2).to(gdt).to(DEV)
        mine = [torch.zeros(n, dtype=torch.uint8 if bits == 8 else torch.float32, device=DEV) for _ in range(2)]
        sc = [torch.zeros(-(-n // 128), 2, dtype=torch.uint8, device=DEV)] if bits == 8 else None
        plan = K.AdamWPlan([p], [mine[0]], [mine[1]], sc, keys=[3])
        before = _f32(p)
        K.adamw_step(plan, [g], 1e-3, (0.9, 0.999), 1e-8, 0.0, 1, seed=4)
        p64, _, _ = _exact(before, _f32(g), 0 * before, 0 * before, dict(lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0), 1)
        _weights_ok(p, p64, before.astype(np.float64), pdt)


@pytest.mark.parametrize("k", [1, 3])
def test_tensors_at_any_element(k):
    """Weights, gradients and moments that start anywhere in their allocation."""
    def at(t):
        flat = torch.zeros(t.numel() + k + 9, dtype=t.dtype, device=DEV)
        flat[k:k + t.numel()] = t.to(DEV)
        return flat, flat[k:k + t.numel()]

    for bits in (32, 8):
        for dt in (torch.bfloat16, torch.float32):
            n = 5000 + k
            sdt = torch.uint8 if bits == 8 else torch.float32
            say(f"adamw at element {k} {bits} {dt}")
            out = []
            for make in (at, lambda t: (None, t.to(DEV))):
                (fp, p), (fg, g) = make(seeded((n,), 1, 0.05).to(dt)), make(seeded((n,), 2).to(dt))
                (fm, m), (fv, v) = make(torch.zeros(n, dtype=sdt)), make(torch.zeros(n, dtype=sdt))
                sc = [torch.zeros(-(-n // 128), 2, dtype=torch.uint8, device=DEV)] if bits == 8 else None
                plan = K.AdamWPlan([p], [m], [v], sc, keys=[3])
                for step in (1, 2):
                    K.adamw_step(plan, [g], *list(HYPER.values()), step)
                out.append([p.clone(), m.clone(), v.clone()])
                if fp is not None:   # what lies around the tensors stays as it was
                    for f in (fp, fm, fv):
                        assert torch.all(f[:k] == 0) and torch.all(f[k + n:] == 0)
            assert all(torch.equal(a, c) for a, c in zip(*out))


@pytest.mark.parametrize("bits", [32, 8])
def test_more_tensors_than_a_launch_takes(bits):
    params = _params([5 + i % 200 for i in range(1000)], (torch.float32, torch.bfloat16), 3)
    opt = moe.AdamW(params, **HYPER, state_bits=bits, seed=1)
    for i, p in enumerate(params.values()):
        p.grad = seeded(p.shape, 9000 + i).to(p.dtype).to(DEV)
    before = {n: _f32(p) for n, p in params.items()}
    say(f"adamw 1000 tensors {bits}")
    opt.step()
    for n, p in params.items():
        z = np.zeros_like(before[n])
        p64, _, _ = _exact(before[n], _f32(p.grad), z, z, HYPER, 1)
        _weights_ok(p, p64, before[n].astype(np.float64), p.dtype)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_gradients_that_are_not_finite(bits, bad):
    """They spoil their own element; with 8 bits the block of 128 that shares its exponent, and nothing else.
    Clipped, the norm says so."""
    params = _params([1000], (torch.float32,), 5)
    opt = moe.AdamW(params, **HYPER, state_bits=bits, max_grad_norm=None)
    p = params["p0"]
    p.grad = torch.ones_like(p)
    p.grad[300] = bad
    say(f"adamw not finite {bits} {bad}")
    opt.step()
    opt.step()
    m, v = (t[:1000].float() for t in opt.moments())
    hit = torch.zeros(1000, dtype=torch.bool, device=DEV)
    hit[256:384 if bits == 8 else 256] = True
    hit[300] = True
    assert torch.equal(~torch.isfinite(v), hit) and torch.all(torch.isfinite(m[~hit]))
    assert torch.equal(torch.isnan(p.detach()), hit)
    clipped = moe.AdamW(params, max_grad_norm=1.0)
    clipped.step()
    norm, coef = clipped.grad_norm.tolist()
    assert (norm == bad and coef == 0.0) if bad == float("inf") else (norm != norm and coef != coef)


def test_eight_bits_reproducible_and_bound_to_the_name():
    """The same seed gives the same bits; a parameter keeps its random bits when others come and go."""
    say("adamw8 names")
    def run(names, seed):
        params = {n: torch.nn.Parameter(seeded((3000,), 1 + i, 0.05).to(DEV)) for i, n in enumerate("abc") if n in names}
        opt = moe.AdamW(params, **HYPER, state_bits=8, seed=seed)
        for step in range(3):
            for i, n in enumerate("abc"):
                if n in names:
                    params[n].grad = seeded((3000,), 10 * step + i).to(DEV)
            opt.step()
        return {k: v.clone() for k, v in opt.state_tensors().items()}
    full, again, alone, other = run("abc", 1), run("abc", 1), run("b", 1), run("abc", 2)
    assert all(torch.equal(full[k], again[k]) for k in full)
    assert all(torch.equal(full[k], alone[k]) for k in alone)
    assert not torch.equal(full["exp_avg/b"], other["exp_avg/b"])


@pytest.mark.parametrize("bits", [32, 8])
def test_state_moves_by_name(bits):
    """State tensors loaded into a new optimizer continue the run bit for bit; 8-bit and 32-bit states convert."""
    say(f"adamw state {bits}")
    sizes, dts = [300, 129, 2050], (torch.bfloat16, torch.float32)
    def grads(params, step):
        for i, p in enumerate(params.values()):
            p.grad = seeded(p.shape, 70 * step + i).to(p.dtype).to(DEV)
    make = lambda: moe.AdamW(_params(sizes, dts, 1), **HYPER, state_bits=bits, master_weights=True, seed=3)  # noqa: E731
    a = make()
    for step in range(3):
        grads(a.params, step)
        a.step()
    saved = {k: t.detach().cpu().clone() for k, t in a.state_tensors().items()}
    assert sorted(k.split("/")[0] for k in saved if k.endswith("/p0")) == sorted(
        ["param", "exp_avg", "exp_avg_sq", "master"] + (["scales"] if bits == 8 else []))
    b = make()
    b.load_state_tensors(saved, a.step_count)
    for opt in (a, b):
        for step in (3, 4):
            grads(opt.params, step)
            opt.step()
    for k, t in a.state_tensors().items():
        assert torch.equal(t, b.state_tensors()[k]), k
    # Into the other width: values become nearest codes, codes their values.
    c = moe.AdamW(_params(sizes, dts, 9), **HYPER, state_bits=40 - bits)
    c.load_state_tensors(saved, 3)
    for n in a.params:
        if bits == 8:
            m, v = R.decode(*(saved[f"{k}/{n}"].numpy() for k in ("exp_avg", "exp_avg_sq", "scales")))
            assert np.array_equal(_f32(c.state[n]["exp_avg"]), m) and np.array_equal(_f32(c.state[n]["exp_avg_sq"]), v)
        else:
            m, v = saved[f"exp_avg/{n}"].numpy(), saved[f"exp_avg_sq/{n}"].numpy()
            want = R.encode(m, v, R.nearest(m.size))
            for key, e in zip(("exp_avg", "exp_avg_sq", "scales"), want):
                assert np.array_equal(c.state[n][key].cpu().numpy(), e), (n, key)
    with pytest.raises(TypeError):
        a.state["p0"]["exp_avg"] = None


def test_parameters_that_move_are_followed():
    """Storage put in a parameter's place (a re-placement) is stepped, not the old one."""
    say("adamw moved parameter")
    params = _params([500, 20], (torch.float32,), 1)
    opt = moe.AdamW(params, **HYPER)
    for step in range(2):
        for p in params.values():
            p.grad = torch.ones_like(p)
        old = params["p0"].detach()
        opt.step()
        if step == 0:
            params["p0"].data = params["p0"].detach().clone()
            kept = old.clone()
    assert torch.equal(old, params["p0"].detach()) and not torch.equal(old, kept)
    plan = opt._plan
    params["p0"].data = params["p0"].detach().clone()
    with pytest.raises(K.KernelArgumentError, match="moved"):
        K.adamw_step(plan, [None, None], 1e-3, (0.9, 0.999), 1e-8, 0.0, 1)


@pytest.mark.parametrize("anew", [lambda t: t.t(), lambda t: t[:32], lambda t: t.reshape(32, 128)],
                         ids=["transposed", "fewer-rows", "reshaped"])
def test_parameters_laid_out_anew_in_place_are_refused(anew):
    """At the same address with another shape or other strides: the moments no longer belong to the elements."""
    say("adamw parameter laid out anew")
    p = torch.nn.Parameter(seeded((64, 64), 1).to(DEV))
    opt = moe.AdamW({"p": p})
    opt.step()
    old = p.data
    p.data = anew(old)
    before = old.clone()
    with pytest.raises(RuntimeError):
        opt.step()
    assert opt.step_count == 1 and torch.equal(old, before)
    p.data = old
    opt.step()
    assert opt.step_count == 2 and not torch.equal(old, before)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("eps", [0.0, 1e-20, 1.9e-12, 2.1e-12, 1e-3])
def test_eps_down_to_zero(bits, eps):
    """Second moments from subnormals up: with an eps that does not hide them the root is the exact one."""
    n = 4096
    p, g = seeded((n,), 1, 0.05).to(DEV), (seeded((n,), 2) * 10.0 ** torch.linspace(-21, 3, n)).to(DEV)
    sdt = torch.uint8 if bits == 8 else torch.float32
    m, v = torch.zeros(n, dtype=sdt, device=DEV), torch.zeros(n, dtype=sdt, device=DEV)
    sc = [torch.zeros(n // 128, 2, dtype=torch.uint8, device=DEV)] if bits == 8 else None
    plan = K.AdamWPlan([p], [m], [v], sc, keys=[1])
    hyper = dict(lr=1e-3, betas=(0.9, 0.95), eps=eps, weight_decay=0.0)
    say(f"adamw eps={eps} {bits}")
    for step in (1, 2):
        before, hv = _f32(p), (R.decode(*(t.cpu().numpy() for t in (m, v, sc[0]))) if bits == 8 else (_f32(m), _f32(v)))
        K.adamw_step(plan, [g], *hyper.values(), step)
        p64, _, v32 = _exact(before, _f32(g), *hv, hyper, step)
        some = v32 > 0          # where a square underflows and eps is 0, m / 0 is infinite
        assert some.mean() > 0.9
        _weights_ok(p[torch.from_numpy(some).to(DEV)], p64[some], before[some].astype(np.float64), torch.float32)
        assert torch.isfinite(p).all().item() == (eps > 0.0 or bool(some.all()))
        p.copy_(torch.from_numpy(before))


@pytest.mark.parametrize("bits", [32, 8])
def test_a_tensor_of_more_than_two_giga_elements(bits):
    n, tail = (1 << 31) + 5000, 5000 + 128
    say(f"adamw n={n} {bits}")
    p = torch.zeros(n, dtype=torch.bfloat16, device=DEV)
    g = torch.zeros(n, dtype=torch.bfloat16, device=DEV)
    sdt = torch.uint8 if bits == 8 else torch.float32
    m, v = torch.zeros(n, dtype=sdt, device=DEV), torch.zeros(n, dtype=sdt, device=DEV)
    sc = torch.zeros(-(-n // 128), 2, dtype=torch.uint8, device=DEV) if bits == 8 else None
    p[-tail:], g[-tail:] = seeded((tail,), 1, 0.05).to(DEV), seeded((tail,), 2).to(DEV)
    before, hg = _f32(p[-tail:]), _f32(g[-tail:])
    plan = K.AdamWPlan([p], [m], [v], None if sc is None else [sc], keys=[77])
    K.adamw_step(plan, [g], *HYPER.values(), 1, seed=6)
    z = np.zeros(tail, np.float32)
    p64, m32, v32 = _exact(before, hg, z, z, HYPER, 1)
    _weights_ok(p[-tail:], p64, before.astype(np.float64), torch.bfloat16)
    if bits == 32:
        assert np.array_equal(_f32(m[-tail:]), m32) and np.array_equal(_f32(v[-tail:]), v32)
    else:
        want = R.encode(m32, v32, R.random_bits(tail, 6, 1, 77, n - tail))
        for t, e in zip((m[-tail:], v[-tail:], sc[-want[2].shape[0]:]), want):
            assert np.array_equal(t.cpu().numpy(), e)
    head = slice(0, n - tail)
    for t in (p, m, v):
        assert not torch.any(t[head].view(torch.uint8 if t.dtype == torch.uint8 else torch.int16 if t.dtype == torch.bfloat16
                                          else torch.int32))
    assert abs(K.grad_norm([g])[0].item() - np.sqrt((hg.astype(np.float64) ** 2).sum())) < 1e-4


def test_every_element_is_stepped_where_a_step_takes_several_launches():
    n = (2 << 30) + 3001
    say(f"adamw n={n} without a gradient")
    p = torch.ones(n, dtype=torch.bfloat16, device=DEV)
    m, v = torch.zeros(n, device=DEV), torch.zeros(n, device=DEV)
    K.adamw_step(K.AdamWPlan([p], [m], [v]), [None], 0.5, (0.9, 0.999), 1e-8, 1.0, 1)
    assert all(bool((t == 0.5).all()) for t in p.split(1 << 28))


def test_gradients_with_strides_and_parameters_twice():
    say("adamw strided gradient")
    a, b = (moe.AdamW({"w": torch.nn.Parameter(seeded((40, 70), 1, 0.05).to(DEV))}, **HYPER) for _ in range(2))
    g = seeded((70, 40), 2).to(DEV).t()
    a.params["w"].grad, b.params["w"].grad = g, g.contiguous()
    a.step()
    b.step()
    assert torch.equal(a.params["w"], b.params["w"])
    p = torch.nn.Parameter(torch.zeros(10, device=DEV))
    twice = moe.AdamW({"a": p, "b": p})
    p.grad = torch.ones(10, device=DEV)
    with pytest.raises(RuntimeError, match="share memory"):
        twice.step()
    assert twice.step_count == 0 and torch.all(p == 0)


def test_a_graph_that_holds_the_parameters_notices_the_step():
    p = torch.nn.Parameter(torch.ones(10, device=DEV))
    opt = moe.AdamW({"p": p})
    y = (p * p).sum()
    p.grad = torch.ones(10, device=DEV)
    opt.step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_what_a_state_lacks_is_named():
    opt = moe.AdamW({"p": torch.nn.Parameter(torch.ones(10, device=DEV))}, state_bits=8)
    st = dict(opt.state_tensors())
    for key in ("exp_avg/p", "scales/p"):
        with pytest.raises(KeyError):
            opt.load_state_tensors({k: v for k, v in st.items() if k != key}, 1)
    with pytest.raises(RuntimeError, match="unsupported dtype"):
        moe.AdamW({"p": torch.nn.Parameter(torch.ones(10, device=DEV, dtype=torch.float16))})


def test_no_parameters():
    opt = moe.AdamW({})
    opt.step()
    assert opt.step_count == 1 and opt.state_tensors() == {} and opt.buffers() == {}


def test_refusals():
    p, g = torch.zeros(10, device=DEV), torch.zeros(10, device=DEV)
    z = lambda n, dt=torch.float32: torch.zeros(n, dtype=dt, device=DEV)  # noqa: E731
    plan = K.AdamWPlan([p], [z(10)], [z(10)])
    step = lambda grads, **kw: K.adamw_step(plan, grads, 1e-3, (0.9, 0.999), 1e-8, 0.0, **({"step": 1} | kw))  # noqa: E731
    u8 = torch.uint8
    bad = [lambda: step([]), lambda: step([g.half()]), lambda: step([g.double()]), lambda: step([g[:5]]),
           lambda: step([z(20)[::2]]), lambda: step([g.cpu()]), lambda: step([g], step=0),
           lambda: step([g], grad_scale=z(2)), lambda: step([g], grad_scale=z(1).double()),
           lambda: step([g], grad_scale=z(1).cpu()),
           lambda: K.AdamWPlan([], [], []), lambda: K.AdamWPlan([p.half()], [z(10)], [z(10)]),
           lambda: K.AdamWPlan([p], [z(9)], [z(10)]), lambda: K.AdamWPlan([p], [z(10, torch.bfloat16)], [z(10)]),
           lambda: K.AdamWPlan([p], [z(10, u8)], [z(10, u8)], [torch.zeros(2, 2, dtype=u8, device=DEV)]),
           lambda: K.AdamWPlan([p], [z(10)], [z(10)], masters=[z(10)]),
           lambda: K.AdamWPlan([p.double(), p], [z(10).double(), z(10)], [z(10).double(), z(10)]),
           lambda: K.moments_decode(z(10, u8), z(10, u8), torch.zeros(2, 2, dtype=u8, device=DEV)),
           lambda: K.moments_decode(z(10), z(10), torch.zeros(1, 2, dtype=u8, device=DEV)),
           lambda: K.moments_encode(z(10), z(9), z(10, u8), z(10, u8), torch.zeros(1, 2, dtype=u8, device=DEV)),
           lambda: K.grad_norm([g], 0.0), lambda: K.grad_norm([g.half()]), lambda: K.grad_norm([g, g.cpu()])]
    for i, f in enumerate(bad):
        with pytest.raises(RuntimeError):
            f()
            pytest.fail(f"call {i} was taken")
    assert torch.all(p == 0)


@pytest.mark.parametrize("n", [1, 2, 8, 127, 128, 129, 4096, 100003])
def test_decode_and_encode(n):
    say(f"moments n={n}")
    g = np.random.default_rng(n)
    qm, qv = (g.integers(0, 256, n).astype(np.uint8) for _ in range(2))
    sc = g.integers(0, 256, (-(-n // 128), 2)).astype(np.uint8)
    m, v = K.moments_decode(*(torch.from_numpy(t).to(DEV) for t in (qm, qv, sc)))
    hm, hv = R.decode(qm, qv, sc)
    assert np.array_equal(_f32(m), hm, equal_nan=True) and np.array_equal(_f32(v), hv, equal_nan=True)
    a = (g.standard_normal(n) * 10.0 ** g.uniform(-40, 38, n)).astype(np.float32)
    b = np.abs((g.standard_normal(n) * 10.0 ** g.uniform(-40, 38, n)).astype(np.float32))
    out = [torch.from_numpy(t).to(DEV) for t in (qm, qv, sc)]
    K.moments_encode(torch.from_numpy(a).to(DEV), torch.from_numpy(b).to(DEV), *out)
    for t, e in zip(out, R.encode(a, b, R.nearest(n))):
        assert np.array_equal(t.cpu().numpy(), e)


# ----------------------------------------------------------------------------- the gradients' norm


def _norm64(gs):
    return float(np.sqrt(sum(float((g.detach().cpu().double() ** 2).sum()) for g in gs)))


@pytest.mark.parametrize("sizes", [[1], [3, 0, 5], [4095, 4096, 4097], [100003, 1, 8192], [17] * 500, [3_000_001]],
                         ids=lambda s: f"{len(s)}x{max(s)}")
def test_grad_norm(sizes):
    """A double sum of at most 2^22 squares is off by far less than float's half step; the float results by that
    half step (and the coefficient's float by another)."""
    for dts in ((torch.bfloat16,), (torch.float32,), (torch.float64,), (torch.float32, torch.bfloat16, torch.float64)):
        gs = [seeded((n,), i).to(dts[i % len(dts)]).to(DEV) for i, n in enumerate(sizes)]
        say(f"grad norm {len(sizes)} tensors {dts}")
        for top in (1.0, 1e6, float("inf")):
            got = K.grad_norm(gs, top).double().cpu()
            norm = _norm64(gs)
            assert abs(float(got[0]) - norm) <= norm * 2.0 ** -23
            coef = min(1.0, top / (norm + 1e-6))
            assert abs(float(got[1]) - coef) <= coef * 2.0 ** -23
        assert torch.equal(K.grad_norm(gs, 1.0), K.grad_norm([None, *gs, None], 1.0))


def test_grad_norm_at_the_ends_of_the_range():
    say("grad norm ranges")
    for value, n in ((3e38, 1), (1e30, 1000), (1e-30, 1000), (1e-44, 3), (0.0, 100)):
        g = torch.full((n,), value, device=DEV)
        want = _norm64([g])
        got = K.grad_norm([g], 1.0).tolist()
        assert got[0] == np.float32(want) or abs(got[0] - want) <= want * 2.0 ** -23 + 1e-45
        assert got[1] == (1.0 if want < 0.5 else np.float32(1.0 / (want + 1e-6)))
    odd = torch.zeros(1 << 16 | 5, device=DEV, dtype=torch.bfloat16)[5:]     # starts 10 bytes into its allocation
    odd[-1] = 3.0
    assert K.grad_norm([odd]).tolist() == [3.0, 1.0]
    out = K.grad_norm([torch.tensor([1.0, float("nan")], device=DEV)], 1.0)
    assert torch.isnan(out).all()
    assert K.grad_norm([torch.tensor([1.0, -float("inf")], device=DEV)], 1.0).tolist() == [float("inf"), 0.0]
    assert K.grad_norm([torch.zeros(0, device=DEV)], 1.0).tolist() == [0.0, 1.0]


@pytest.mark.parametrize("bits", [32, 8])
def test_clipped_step(bits):
    """The step of clipped gradients is the step of gradients times the coefficient, which stays on the device."""
    params = _params([3000, 77], (torch.float32, torch.bfloat16), 1)
    opt = moe.AdamW(params, **HYPER, state_bits=bits, max_grad_norm=0.5)
    gs = []
    for i, p in enumerate(params.values()):
        p.grad = seeded(p.shape, i + 40).to(p.dtype).to(DEV)
        gs.append(p.grad)
    before = {n: _f32(p) for n, p in params.items()}
    say(f"adamw clip {bits}")
    opt.step()
    norm = _norm64(gs)
    coef = np.float32(opt.grad_norm[1].item())
    assert abs(float(coef) - 0.5 / (norm + 1e-6)) <= 2.0 ** -23 * float(coef) and opt.grad_norm.shape == (2,)
    for n, p in params.items():
        z = np.zeros_like(before[n])
        p64, _, _ = _exact(before[n], _f32(p.grad), z, z, HYPER, 1, float(coef))
        _weights_ok(p, p64, before[n].astype(np.float64), p.dtype)
    for p in params.values():
        p.grad = None
    opt.step()
    assert opt.grad_norm is None


# ----------------------------------------------------------------------------- graphs, streams, a run


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_step(bits):
    """A captured clip and step, replayed, does what the eager call does to the same tensors (the scalars, step
    number and seed are those of the capture)."""
    sizes, dts = [5000, 129], (torch.bfloat16, torch.float32)
    params = _params(sizes, dts, 1)
    opt = moe.AdamW(params, **HYPER, state_bits=bits, max_grad_norm=0.5)
    for i, p in enumerate(params.values()):
        p.grad = seeded(p.shape, i).to(p.dtype).to(DEV)
    grads = [p.grad for p in params.values()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        opt.step()
    torch.cuda.synchronize()
    say(f"adamw graph {bits}")
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr, stream=side):
        norm = K.grad_norm(grads, 0.5)
        K.adamw_step(opt._plan, grads, *HYPER.values(), 2, norm[1:], 11)
    state = lambda: [t.clone() for t in (*opt.state_tensors().values(),)]  # noqa: E731
    for i in range(4):
        for k, g in enumerate(grads):
            g.copy_(seeded(g.shape, 100 * i + k))
        saved = state()
        gr.replay()
        torch.cuda.synchronize()
        got = state()
        for t, s in zip(opt.state_tensors().values(), saved):
            t.copy_(s)
        K.adamw_step(opt._plan, grads, *HYPER.values(), 2, K.grad_norm(grads, 0.5)[1:], 11)
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(got, state())), i
    # The optimizer's own step, captured: each replay is one more step with the number it was captured with.
    opt.step_count = 1
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr, stream=side):
        opt.step()
    for i in range(3):
        saved = state()
        gr.replay()
        torch.cuda.synchronize()
        got = state()
        for t, s in zip(opt.state_tensors().values(), saved):
            t.copy_(s)
        opt.step_count = 1
        opt.step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(got, state())), i
    fresh = moe.AdamW(_params([10], (torch.float32,), 1))
    fresh.params["p0"].grad = torch.ones(10, device=DEV)
    with pytest.raises(K.KernelArgumentError, match="captured"):
        with torch.cuda.graph(torch.cuda.CUDAGraph(), stream=side):
            fresh.step()
    torch.cuda.synchronize()


def test_two_optimizers_on_two_streams():
    say("adamw on two streams")
    def run(streams):
        opts = [moe.AdamW(_params([200_000, 3], (torch.bfloat16,), s), **HYPER, state_bits=8, max_grad_norm=1.0) for s in (1, 2)]
        for o in opts:
            for i, p in enumerate(o.params.values()):
                p.grad = seeded(p.shape, i).to(p.dtype).to(DEV)
        torch.cuda.synchronize()
        for _ in range(5):
            for o, s in zip(opts, streams):
                with torch.cuda.stream(s):
                    o.step()
        torch.cuda.synchronize()
        return [t.clone() for o in opts for t in o.state_tensors().values()]
    one = torch.cuda.current_stream()
    for a, c in zip(run([one, one]), run([torch.cuda.Stream(), torch.cuda.Stream()])):
        assert torch.equal(a, c)


def _loss(out, y):
    return ((out - y) ** 2).mean(dim=-1).sum()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("master", [False, True])
def test_a_training_run_of_the_block(master, bits):
    """Norm, layer, backward, clip and step together: each iteration's update is the one that AdamW makes of the
    gradients that iteration had, from the moments that the state stands for."""
    cfg = moe.MoEConfig(hidden=128, ffn=96, num_experts=4, top_k=2, tokens=100, dtype=torch.bfloat16, act="swiglu",
                        norm="layer", init_std=0.05, device=DEV)
    params = {k: torch.nn.Parameter(moe.init_param(cfg, s)) for k, s in moe.moe_specs(cfg).items()}
    opt = moe.AdamW(params, **HYPER, max_grad_norm=0.1, master_weights=master, no_decay=("norm.weight", "norm.bias"),
                    state_bits=bits)
    say(f"training run master={master} {bits}")
    for it in range(3):
        opt.zero_grad()
        x, y = moe.batch(cfg, it)
        (_loss(moe.reference_forward(cfg, params, x), y) / cfg.tokens).backward()
        hosts = {}
        for n, p in params.items():
            st = opt.state[n]
            mv = R.decode(*(st[k].cpu().numpy().reshape(-1, 2) if k == "scales" else st[k].cpu().numpy().reshape(-1)
                            for k in ("exp_avg", "exp_avg_sq", "scales"))) if bits == 8 else \
                (_f32(st["exp_avg"]).reshape(-1), _f32(st["exp_avg_sq"]).reshape(-1))
            hosts[n] = (_f32(st.get("master", p)).reshape(-1), _f32(p.grad).reshape(-1), *mv)
        opt.step()
        norm = np.sqrt(sum((h[1].astype(np.float64) ** 2).sum() for h in hosts.values()))
        assert abs(opt.grad_norm[0].item() - norm) <= 2.0 ** -23 * norm
        scale = opt.grad_norm[1].item()
        assert abs(scale - min(1.0, 0.1 / (norm + 1e-6))) <= 2.0 ** -23
        for n, p in params.items():
            w, g, m, v = hosts[n]
            p64, _, _ = _exact(w, g, m, v, HYPER, it + 1, scale, not n.startswith("norm."))
            mast = opt.state[n].get("master")
            _weights_ok((p if mast is None else mast).reshape(-1), p64, w.astype(np.float64),
                        p.dtype if mast is None else torch.float32)
