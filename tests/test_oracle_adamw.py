"""The 8-bit moments' codes on the CPU: what the numpy restatement of the step's rounding does and why it is
stochastic; and the C entry points' refusals, which come before any kernel."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from oracle import adamw_ref as R
from resihp_megatron_amd import _capi as C
from resihp_megatron_amd import kernels as K
from resihp_megatron_amd import moe


def _wide(n, seed, spread=3.0):
    g = np.random.default_rng(seed)
    return (g.standard_normal(n) * 10.0 ** (spread * g.standard_normal(n))).astype(np.float32)


def test_codes_keep_four_significant_bits():
    """A code's value is within a step (1/8 of the binade, at most 1/8 of the value) of the moment, above where
    the block ends; a value decodes to itself whatever the random bits, and bfloat16 holds it."""
    n = 128 * 40 + 3
    m, v = _wide(n, 1, 0.5), np.abs(_wide(n, 2, 1.0))
    qm, qv, sc = R.encode(m, v, R.random_bits(n, 5, 9, 77))
    dm, dv = R.decode(qm, qv, sc)
    blk = np.arange(n) // 128
    low_m = np.exp2(sc[blk, 0].astype(np.float64) - 127 - 15)
    low_v = np.exp2(sc[blk, 1].astype(np.float64) - 127 - 31)
    big_m, big_v = np.abs(m) >= 1.25 * low_m, v >= 1.25 * low_v
    assert big_m.mean() > 0.95 and big_v.mean() > 0.95
    assert np.all(np.abs(dm - m)[big_m] <= np.abs(m)[big_m] / 8) and np.all(np.abs(dv - v)[big_v] <= v[big_v] / 8)
    assert np.all(np.abs(dm)[~big_m] <= 1.375 * low_m[~big_m])
    assert np.all(np.sign(dm)[big_m] == np.sign(m)[big_m])
    for t in (dm, dv):
        assert np.array_equal(torch.from_numpy(t).bfloat16().float().numpy(), t)
    qm2, qv2, sc2 = R.encode(dm, dv, R.random_bits(n, 6, 10, 78))
    dm2, dv2 = R.decode(qm2, qv2, sc2)
    keep = np.abs(dm) >= 2 * low_m   # a block whose largest value was rounded down a binade keeps one more below
    assert np.array_equal(dm2[keep], dm[keep]) and np.array_equal(dv2[dv >= 2 * low_v], dv[dv >= 2 * low_v])


def test_second_moment_never_becomes_zero():
    v = np.array([1.0, 1e-30, 1e-38, 1e-45, 0.0] + [1e-12] * 5, np.float32)
    for r in (np.zeros(10, np.int64), np.full(10, 0xFFFFFFFF, np.int64)):
        _, qv, sc = R.encode(np.zeros_like(v), v, r)
        _, dv = R.decode(np.zeros(10, np.uint8), qv, sc)
        assert np.all((dv > 0) == (v > 0))
        assert np.all(dv[1:4] <= 1.125 * 2.0 ** -31)


@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan, 3.3e38])
def test_block_that_is_not_finite_reads_as_nan(bad):
    m = np.ones(300, np.float32)
    m[130] = bad
    v = np.ones(300, np.float32)
    qm, qv, sc = R.encode(m, v, R.nearest(300))
    assert list(sc[:, 0]) == [127, 255, 127] and list(sc[:, 1]) == [127] * 3
    dm, dv = R.decode(qm, qv, sc)
    assert np.isnan(dm[128:256]).all() and np.all(dm[:128] == 1) and np.all(dm[256:] == 1) and np.all(dv == 1)


def test_random_bits_are_uniform_and_differ():
    n = 1 << 18
    r = R.random_bits(n, 3, 4, 5)
    for part in (r & 0xFFFF, r >> 16):
        u = part / 65536.0
        assert abs(u.mean() - 0.5) < 6 * np.sqrt(1 / 12 / n)      # six standard deviations of a mean of n
        assert abs((u * u).mean() - 1 / 3) < 6 * np.sqrt(4 / 45 / n)
        for lag in (1, 2, 7, 8, 64, 128):
            c = np.mean((u[:-lag] - 0.5) * (u[lag:] - 0.5)) * 12
            assert abs(c) < 6 / np.sqrt(n), lag
    assert abs(np.mean(((r & 0xFFFF) / 65536 - 0.5) * ((r >> 16) / 65536 - 0.5)) * 12) < 6 / np.sqrt(n)
    for other in (R.random_bits(n, 4, 4, 5), R.random_bits(n, 3, 5, 5), R.random_bits(n, 3, 4, 6)):
        assert abs(np.mean((r & 0xFFFF) == (other & 0xFFFF)) - 2.0 ** -16) < 6 * np.sqrt(2.0 ** -16 / n)


def test_stochastic_rounding_follows_a_steady_gradient_where_nearest_stops():
    """m -> g and v -> g^2 under a constant gradient: the mean over many elements arrives under stochastic
    rounding (the noise of 4096 of them: a code's step is at most 1/8, and a step of v forgets 1/1000 of it, so
    the deviation of one is at most 1/8 and of the mean 1/512), and stays far off under nearest rounding."""
    n, b1, b2 = 4096, np.float32(0.9), np.float32(0.999)
    g = np.full(n, 0.01, np.float32)
    got = {}
    for kind in ("random", "nearest"):
        m, v = np.zeros(n, np.float32), np.full(n, 4e-4, np.float32)
        for t in range(1, 6000):
            m = m * b1 + g * (1 - b1)
            v = v * b2 + g * (1 - b2) * g
            m, v = R.decode(*R.encode(m, v, R.random_bits(n, 1, t, 2) if kind == "random" else R.nearest(n)))
        got[kind] = (m.mean() / 0.01, v.mean() / 1e-4)
    # v has decayed for 6000 steps from 4: 1 + 3 exp(-6) = 1.0075.
    assert abs(got["random"][0] - 1) < 0.02 and abs(got["random"][1] - 1.0075) < 0.02, got
    assert abs(got["nearest"][1] - 1) > 1, got


# ----------------------------------------------------------------------------- refusals (no GPU)

FAKE = 4096   # 16-byte aligned, never dereferenced: the checks come first


def _plan(numel=(10,), dtypes=(C.BF16,), params=(FAKE,), m=(2 * FAKE,), v=(3 * FAKE,), scales=None, masters=None, keys=None,
          bits=32, short=0):
    n = len(numel)
    num = (ctypes.c_int64 * n)(*numel)
    size = C.lib().rhp_adamw_plan_bytes(n, num, bits)
    buf = ctypes.create_string_buffer(max(1, size))
    C.call("rhp_adamw_plan", n, C.ptr_array(params), (ctypes.c_int * n)(*dtypes), C.ptr_array(masters) if masters else None,
           C.ptr_array(m), C.ptr_array(v), C.ptr_array(scales) if scales else None, num,
           (ctypes.c_uint32 * n)(*keys) if keys else None, None, bits, buf, size - short)
    return buf, size


@pytest.mark.parametrize("kw,msg", [
    (dict(bits=16), "32 or 8 bits"),
    (dict(bits=8), "null array"),
    (dict(bits=8, scales=(0,), keys=(1,)), "null tensor"),
    (dict(dtypes=(C.E4M3,)), "unsupported dtype"),
    (dict(dtypes=(C.F32,), masters=(FAKE,)), "masters are for bfloat16"),
    (dict(params=(0,)), "null tensor"),
    (dict(params=(FAKE + 1,)), "not aligned"),
    (dict(m=(FAKE + 2,)), "not aligned"),
    (dict(masters=(FAKE + 2,)), "not aligned"),
    (dict(m=(FAKE + 16,)), "share memory"),
    (dict(m=(3 * FAKE,)), "share memory"),
    (dict(masters=(3 * FAKE + 36,)), "share memory"),
    (dict(bits=8, scales=(3 * FAKE + 9,), keys=(1,)), "share memory"),
    (dict(numel=(10, 10), dtypes=(C.F32,) * 2, params=(FAKE, FAKE), m=(5 * FAKE, 6 * FAKE), v=(7 * FAKE, 8 * FAKE)), "share memory"),
    (dict(short=1), "image smaller"),
    (dict(dtypes=(C.F64,), bits=8, scales=(4 * FAKE,), keys=(1,)), "float64 moments"),
    (dict(numel=(10, 10), dtypes=(C.F64, C.F32), params=(FAKE, 2 * FAKE), m=(3 * FAKE, 4 * FAKE), v=(5 * FAKE, 6 * FAKE)),
     "plan of their own"),
])
def test_plan_refusals(kw, msg):
    with pytest.raises(RuntimeError, match=msg):
        _plan(**kw)


def test_plan_refuses_bad_counts():
    num = (ctypes.c_int64 * 1)(-1)
    assert C.lib().rhp_adamw_plan_bytes(1, num, 32) == 0 and C.lib().rhp_adamw_plan_bytes(-1, None, 32) == 0
    assert C.lib().rhp_adamw_plan_bytes(0, None, 16) == 0 and C.lib().rhp_adamw_plan_bytes(0, None, 8) > 0
    buf = ctypes.create_string_buffer(4096)
    for n in (-1, (1 << 34) + 1):
        with pytest.raises(RuntimeError, match="out of range"):
            C.call("rhp_adamw_plan", 1, C.ptr_array([FAKE]), (ctypes.c_int * 1)(1), None, C.ptr_array([FAKE]),
                   C.ptr_array([FAKE]), None, (ctypes.c_int64 * 1)(n), None, None, 32, buf, 4096)


def test_plan_bytes_of_counts_out_of_range():
    for n in ((1 << 34) + 1, (1 << 63) - 1):
        assert C.lib().rhp_adamw_plan_bytes(1, (ctypes.c_int64 * 1)(n), 32) == 0
    assert C.lib().rhp_adamw_plan_bytes(1, (ctypes.c_int64 * 1)(1 << 34), 8) > 0


def _step(image, size, grads=None, codes=None, step=1, dev=FAKE, hyper=(1e-3, 0.9, 0.999, 1e-8, 0.0)):
    C.call("rhp_adamw_step", image, dev, size, C.ptr_array(grads) if grads else None,
           (ctypes.c_int * 1)(*codes) if codes else None, *hyper, step, None, 0, None)


@pytest.mark.parametrize("kw,msg", [
    (dict(step=0), "counts from 1"),
    (dict(hyper=(1e-3, 1.0, 0.999, 1e-8, 0.0)), "betas"),
    (dict(hyper=(1e-3, 0.9, 1.0, 1e-8, 0.0)), "betas"),
    (dict(hyper=(1e-3, -0.1, 0.9, 1e-8, 0.0)), "betas"),
    (dict(hyper=(float("nan"), 0.9, 0.9, 1e-8, 0.0)), "must not be negative"),
    (dict(hyper=(1e-3, 0.9, 0.9, -1e-8, 0.0)), "must not be negative"),
    (dict(hyper=(1e-3, 0.9, 0.9, 1e-8, -0.1)), "must not be negative"),
    (dict(dev=0), "device image"),
    (dict(dev=FAKE + 8), "device image"),
    (dict(grads=(FAKE,)), "without their dtypes"),
    (dict(grads=(FAKE,), codes=(C.F64,)), "unsupported gradient dtype"),
    (dict(grads=(FAKE + 1,), codes=(C.BF16,)), "not aligned"),
])
def test_step_refusals(kw, msg):
    image, size = _plan()
    with pytest.raises(RuntimeError, match=msg):
        _step(image, size, **kw)


def test_step_refuses_what_is_no_plan():
    with pytest.raises(RuntimeError, match="not an image"):
        _step(ctypes.create_string_buffer(256), 256)
    image, size = _plan()
    with pytest.raises(RuntimeError, match="not an image"):
        _step(image, size - 1)
    with pytest.raises(RuntimeError, match="short image"):
        _step(image, 8)


def test_step_over_empty_tensors_launches_nothing():
    image, size = _plan(numel=(0,), params=(0,), m=(0,), v=(0,))
    _step(image, size, dev=0)


@pytest.mark.parametrize("kw,msg", [
    (dict(max_norm=0.0), "max_norm must be positive"), (dict(max_norm=float("nan")), "max_norm must be positive"),
    (dict(out=0), "output"), (dict(ws=0), "workspace"), (dict(size=8), "workspace"),
    (dict(dtype=C.E5M2), "unsupported dtype"), (dict(g=FAKE + 1), "not aligned"),
    (dict(n=-1), "out of range"),
])
def test_grad_norm_refusals(kw, msg):
    a = dict(max_norm=1.0, out=FAKE, ws=FAKE, size=1 << 20, dtype=C.BF16, g=FAKE, n=10) | kw
    with pytest.raises(RuntimeError, match=msg):
        C.call("rhp_grad_norm", 1, C.ptr_array([a["g"]]), (ctypes.c_int * 1)(a["dtype"]), (ctypes.c_int64 * 1)(a["n"]),
               a["max_norm"], a["out"], a["ws"], a["size"], None)


def _norm_fwd(dtype=C.BF16, wd=C.F32, T=4, h=64, eps=1e-5, x=FAKE, y=2 * FAKE):
    C.call("rhp_layer_norm_fwd", x, dtype, FAKE, FAKE, wd, T, h, eps, y, FAKE, FAKE, None)


@pytest.mark.parametrize("kw,msg", [
    (dict(dtype=C.E4M3), "unsupported dtype"), (dict(dtype=C.F32, wd=C.BF16), "rows' dtype"),
    (dict(dtype=C.F64, wd=C.F32), "rows' dtype"), (dict(T=-1), "negative row count"), (dict(h=0), "h must be"),
    (dict(h=(1 << 28) + 1), "h must be"), (dict(eps=-1e-9), "eps"), (dict(eps=float("nan")), "eps"), (dict(x=0), "null"), (dict(y=0), "null"),
    (dict(x=FAKE + 1), "not aligned"), (dict(y=FAKE), "must not be x"),
])
def test_layer_norm_refusals(kw, msg):
    with pytest.raises(RuntimeError, match=msg):
        _norm_fwd(**kw)


@pytest.mark.parametrize("kw,msg", [
    (dict(dy=0), "null"), (dict(ws=0), "workspace"), (dict(ws=FAKE + 8), "workspace"), (dict(size=16), "workspace"),
    (dict(wd=C.BF16), "rows' dtype"), (dict(dres=FAKE, dx=0), "residual's gradient"), (dict(dy=FAKE + 2), "not aligned"),
    (dict(dx=FAKE), "must not be an input"), (dict(dres=2 * FAKE), "must not be an input"),
])
def test_layer_norm_bwd_refusals(kw, msg):
    a = dict(dy=FAKE, wd=C.F32, dres=0, dx=2 * FAKE, ws=FAKE, size=1 << 24) | kw
    with pytest.raises(RuntimeError, match=msg):
        C.call("rhp_layer_norm_bwd", a["dy"], FAKE, C.F32, FAKE, a["wd"], FAKE, FAKE, a["dres"] or None, 4, 64,
               a["dx"] or None, FAKE, FAKE, a["ws"], a["size"], None)


def test_layer_norm_refuses_rows_past_its_launches():
    """The partial rows are summed by 1024 threads for every 64 of their 2 h columns: at h = 2^27 that would be
    2^32 threads, which no launch has."""
    _norm_fwd(T=0, h=1 << 26)
    for h in ((1 << 26) + 1, 1 << 27, 1 << 28):
        with pytest.raises(RuntimeError, match="h must be"):
            _norm_fwd(T=0, h=h)
        with pytest.raises(RuntimeError, match="h must be"):
            C.call("rhp_layer_norm_bwd", FAKE, FAKE, C.F32, FAKE, C.F32, FAKE, FAKE, None, 0, h, 2 * FAKE, None, None,
                   None, 0, None)


def test_workspace_queries():
    L = C.lib()
    assert L.rhp_layer_norm_bwd_workspace_bytes(-1, 64, C.F32) == 0 and L.rhp_layer_norm_bwd_workspace_bytes(4, 0, C.F32) == 0
    assert L.rhp_layer_norm_bwd_workspace_bytes(0, 64, C.F32) > 0
    assert L.rhp_grad_norm_workspace_bytes(-1) == 0 and L.rhp_grad_norm_workspace_bytes(1) > 0


def test_python_refuses_host_tensors_and_bad_options():
    x = torch.zeros(2, 8)
    with pytest.raises(RuntimeError, match="HIP device"):
        K.layer_norm(x)
    with pytest.raises(RuntimeError, match="HIP device"):
        K.grad_norm([x])
    with pytest.raises(RuntimeError, match="HIP device"):
        moe.AdamW({"a": torch.nn.Parameter(x)})
    with pytest.raises(ValueError, match="32 or 8 bits"):
        moe.AdamW({}, state_bits=16)
    with pytest.raises(ValueError, match="max_grad_norm"):
        moe.AdamW({}, max_grad_norm=0.0)
    with pytest.raises(ValueError, match="no_decay"):
        moe.AdamW({}, no_decay=("b",))
    with pytest.raises(K.KernelArgumentError, match="needs a gradient"):
        K.grad_norm([None])
    with pytest.raises(ValueError, match="norm must be"):
        moe.moe_specs(moe.MoEConfig(norm="rms"))


def test_norm_parameters_in_the_state_contract():
    cfg = moe.MoEConfig(norm="layer", dtype=torch.bfloat16, device="cpu")
    specs = moe.moe_specs(cfg)
    assert specs["norm.weight"].global_shape == (8,) and specs["norm.bias"].trainable
    w, b = (moe.init_param(cfg, specs[k]) for k in ("norm.weight", "norm.bias"))
    assert w.dtype == b.dtype == torch.float32 and torch.all(w == 1) and torch.all(b == 0)
    assert "norm.weight" not in moe.moe_specs(moe.MoEConfig())
