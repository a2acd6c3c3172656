"""The work that training has the operators around the MoE layer do, as measurable cases: the layer norm in
front of the layer (forward and backward), the AdamW step over many tensors with its moments in 32 or in 8
bits, and the norm of all gradients that clips them.

``listed()`` names the cases, ``draw(rng)`` gives more of the same ranges, ``prepare`` builds what a program
holds before the call, ``run`` is one pass: in plain torch, or (``own``) through the package's public entry
points.  ``exact`` is the same pass from the definitions in float64.  Sizes are those of the benchmark
workloads and the tests (the Mixtral-8x7B layer shape, the fine-grained layer with shared experts, the tiny
float32 model) or generic ones.
"""

from __future__ import annotations

import importlib
import importlib.util
import math
import pathlib
import sys
import zlib

import torch

own = False

DEV = "cuda:0"
_PKG_DIR = pathlib.Path(__file__).resolve().parents[1] / "resihp-megatron_amd"


def _module(name: str):
    pkg = "resihp_megatron_amd"
    if pkg not in sys.modules:
        spec = importlib.util.spec_from_file_location(pkg, _PKG_DIR / "__init__.py",
                                                      submodule_search_locations=[str(_PKG_DIR)])
        mod = importlib.util.module_from_spec(spec)
        sys.modules[pkg] = mod
        spec.loader.exec_module(mod)
    return importlib.import_module(f"{pkg}.{name}")


# ----------------------------------------------------------------------------- the cases

MIXTRAL = dict(hidden=4096, ffn=14336, experts=8, shared=0)
FINE = dict(hidden=2048, ffn=1408, experts=64, shared=2)
TINY = dict(hidden=64, ffn=128, experts=8, shared=0)


def _norm(kind: str, tokens: int, hidden: int, dtype: str = "bfloat16", residual: bool = False) -> dict:
    return {"kind": kind, "tokens": tokens, "hidden": hidden, "dtype": dtype, "residual": residual}


def _optim(kind: str, shape: dict, dtype: str = "bfloat16", bits: int = 32, master: bool = False,
           clip: bool = False) -> dict:
    return {"kind": kind, **shape, "dtype": dtype, "bits": bits, "master": master, "clip": clip}


def listed() -> list[dict]:
    return [
        # A decoding step of a few sequences: one row per sequence, nothing but latency.
        {"name": "norm_decode", **_norm("norm", 8, 4096)},
        # A float32 model with a hidden size that no vector divides: the full-precision check of a bf16 run.
        {"name": "norm_odd_f32", **_norm("norm", 1500, 1365, "float32")},
        # Training, the token batch of the Mixtral-shape layer.
        {"name": "norm_train", **_norm("norm", 16384, 4096)},
        # A short micro-batch of the fine-grained layer, backward, with the residual's gradient.
        {"name": "norm_bwd_small", **_norm("norm_bwd", 250, 2048, "bfloat16", True)},
        # The float32 model's backward: odd rows, no residual.
        {"name": "norm_bwd_odd_f32", **_norm("norm_bwd", 1500, 1365, "float32")},
        # Training, backward of the Mixtral-shape batch with the residual's gradient.
        {"name": "norm_bwd_train", **_norm("norm_bwd", 16384, 4096, "bfloat16", True)},
        # The optimizer step of the tiny float32 model (19 tensors): launches and the host are all of it.
        {"name": "adamw_tiny_f32", **_optim("adamw", TINY, "float32", clip=True)},
        # The fine-grained layer's step (135 tensors, 0.57 G parameters): bf16 weights, float32 masters and moments.
        {"name": "adamw_fine", **_optim("adamw", FINE, master=True)},
        # A small bf16 model with moments in 8 bits, clipped.
        {"name": "adamw8_small", **_optim("adamw", dict(hidden=1024, ffn=2736, experts=8, shared=0), bits=8,
                                          clip=True)},
        # The Mixtral-shape layer's step (1.41 G parameters) with moments in 8 bits.
        {"name": "adamw8_mixtral", **_optim("adamw", MIXTRAL, bits=8)},
        # The norm of the tiny model's gradients.
        {"name": "grad_norm_tiny_f32", **_optim("grad_norm", TINY, "float32")},
        # The norm of the Mixtral-shape layer's gradients.
        {"name": "grad_norm_mixtral", **_optim("grad_norm", MIXTRAL)},
    ]


def _log(rng, lo: int, hi: int) -> int:
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng) -> dict:
    kind = rng.choice(["norm", "norm", "norm_bwd", "norm_bwd", "adamw", "adamw", "adamw", "grad_norm"])
    if kind in ("norm", "norm_bwd"):
        # Any hidden size, half of them multiples of 64 as models have them; one token to a training batch.
        h = rng.choice([64 * _log(rng, 1, 128), _log(rng, 33, 8191)])
        dtype = rng.choice(["bfloat16", "bfloat16", "float32"])
        top = min(65536, (1 << 26) // h // (2 if dtype == "float32" else 1))
        return _norm(kind, _log(rng, 1, top), h, dtype, kind == "norm_bwd" and rng.random() < 0.5)
    shape = dict(hidden=64 * _log(rng, 1, 64), ffn=8 * _log(rng, 6, 1792), experts=rng.choice([4, 6, 8]),
                 shared=rng.choice([0, 0, 1, 2]))
    if rng.random() < 0.3:   # many small experts
        shape.update(hidden=64 * _log(rng, 1, 16), ffn=8 * _log(rng, 6, 176), experts=rng.choice([32, 64]))
    while (shape["experts"] + shape["shared"]) * shape["hidden"] * shape["ffn"] > 8 * 4096 * 14336 // 4:
        shape["ffn"] = shape["ffn"] // 16 * 8
    dtype = rng.choice(["bfloat16", "bfloat16", "float32"])
    if kind == "grad_norm":
        return _optim(kind, shape, dtype)
    return _optim(kind, shape, dtype, rng.choice([8, 32]), dtype == "bfloat16" and rng.random() < 0.4,
                  rng.random() < 0.5)


# ----------------------------------------------------------------------------- inputs

EPS = 1e-5
ADAMW = dict(lr=1e-3, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.1)
MAX_NORM = 1.0
SEED = 20
STEPS_DONE = 10
NO_DECAY = ("norm.weight", "norm.bias")
BLOCK = 128          # elements that share an exponent; every tensor of a flat buffer starts at a multiple of it
M32 = 0xFFFFFFFF


def _gen(seed: int) -> torch.Generator:
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(g, *shape, std: float = 1.0, dtype=torch.float32) -> torch.Tensor:
    return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32).mul_(std).to(dtype)


def _norm_inputs(case: dict, seed: int) -> dict:
    """Residual-stream rows (a few channels some twenty times the others, a mean that is not zero)."""
    g, dt = _gen(seed), getattr(torch, case["dtype"])
    T, h = case["tokens"], case["hidden"]
    gain = torch.where(torch.rand(h, generator=g, device=DEV) < 0.004, 20.0, 1.0)
    x = ((_randn(g, T, h) + 0.3) * gain).to(dt)
    s = {"x": x, "w": 1 + _randn(g, h, std=0.1), "b": _randn(g, h, std=0.1)}
    if case["kind"] == "norm_bwd":
        s["dy"] = _randn(g, T, h, dtype=dt)
        s["dres"] = _randn(g, T, h, dtype=dt) if case["residual"] else None
        # The statistics that the forward pass kept.
        xd = x.double()
        s["mean"] = xd.mean(1).float()
        s["rstd"] = (xd.var(1, unbiased=False) + EPS).rsqrt().float()
    return s


def _shapes(case: dict) -> dict[str, tuple[tuple[int, ...], torch.dtype]]:
    """Names, shapes and types of the parameters, the float32 ones first."""
    h, f, dt = case["hidden"], case["ffn"], getattr(torch, case["dtype"])
    out = {"norm.weight": ((h,), torch.float32), "norm.bias": ((h,), torch.float32),
           "router.weight": ((case["experts"], h), torch.float32)}
    for e in range(case["experts"]):
        out[f"experts.{e}.fc1.weight"] = ((2 * f, h), dt)
        out[f"experts.{e}.fc2.weight"] = ((h, f), dt)
    for s in range(case["shared"]):
        out[f"shared_experts.{s}.fc1.weight"] = ((2 * f, h), dt)
        out[f"shared_experts.{s}.fc2.weight"] = ((h, f), dt)
    return out


def _blocks(shape: tuple[int, ...]) -> int:
    return -(-math.prod(shape) // BLOCK)


def _optim_inputs(case: dict, seed: int) -> dict:
    """Flat buffers of the float32 tensors ("a") and of the experts ("b"), each tensor from a multiple of
    BLOCK on with zeros behind its end, and views of them by name."""
    g, dt = _gen(seed), getattr(torch, case["dtype"])
    shapes = _shapes(case)
    names = list(shapes)
    nblk = [_blocks(shapes[n][0]) for n in names]
    na = sum(nblk[:3]) * BLOCK
    n = sum(nblk) * BLOCK
    valid = torch.ones(n // BLOCK, BLOCK, dtype=torch.bool, device=DEV)
    at = 0
    for name, k in zip(names, nblk):
        size = math.prod(shapes[name][0])
        valid[at:at + k].view(-1)[size:] = False
        at += k
    valid = valid.view(-1)

    def flat(count, std, dtype, first):
        return _randn(g, count, std=std, dtype=dtype).mul_(valid[first:first + count])

    s = {"names": names, "shapes": shapes, "nblk": nblk, "na": na, "n": n,
         "ga": flat(na, 1e-3, torch.float32, 0), "gb": flat(n - na, 1e-3, dt, na)}
    if case["kind"] == "grad_norm":
        return s
    s["pa"], s["pb"] = flat(na, 0.02, torch.float32, 0), flat(n - na, 0.02, dt, na)
    s["master"] = None
    if case["master"]:   # the masters hold what the bf16 weights round
        s["master"] = s["pb"].float() * (1 + _randn(g, n - na, std=1e-3))
        s["pb"] = s["master"].to(dt)
    m = flat(n, 3e-4, torch.float32, 0)
    v = flat(n, 1e-3, torch.float32, 0).square_()
    s["keys"] = torch.tensor([zlib.crc32(k.encode()) for k in names], dtype=torch.int64, device=DEV)
    s["count"] = torch.tensor(nblk, dtype=torch.int64, device=DEV)
    decay = torch.tensor([0.0 if k in NO_DECAY else 1.0 for k in names[:3]], device=DEV)
    s["decay_a"] = torch.repeat_interleave(decay, s["count"][:3] * BLOCK)
    s["step"] = STEPS_DONE
    if case["bits"] == 8:
        half = torch.full((1,), 0x8000, dtype=torch.int64, device=DEV)
        s["m"], s["v"], s["scales"] = _encode(m, v, half, half)
    else:
        s["m"], s["v"], s["scales"] = m, v, None
    return s


def _view(s: dict, a: torch.Tensor, b: torch.Tensor) -> dict[str, torch.Tensor]:
    out, at = {}, 0
    for name, k in zip(s["names"], s["nblk"]):
        src, first = (a, at) if at < s["na"] else (b, at - s["na"])
        shape = s["shapes"][name][0]
        out[name] = src[first:first + math.prod(shape)].view(shape)
        at += k * BLOCK
    return out


def prepare(case: dict, seed: int):
    if case["kind"] in ("norm", "norm_bwd"):
        return {"case": case, **_norm_inputs(case, seed)}
    s = {"case": case, **_optim_inputs(case, seed)}
    s["grads"] = _view(s, s["ga"], s["gb"])
    if own and case["kind"] == "adamw":
        params = {k: torch.nn.Parameter(t) for k, t in _view(s, s["pa"], s["pb"]).items()}
        opt = _module("moe").AdamW(params, **ADAMW, state_bits=case["bits"], master_weights=case["master"],
                                   max_grad_norm=MAX_NORM if case["clip"] else None, no_decay=NO_DECAY, seed=SEED)
        opt.step_count = s["step"]
        buffers = opt.buffers()
        for k in ("m", "v", "scales", "master"):
            if s[k] is not None:
                buffers[{"m": "exp_avg", "v": "exp_avg_sq"}.get(k, k)].copy_(s[k])
            del s[k]
        for k, p in params.items():
            p.grad = s["grads"][k]
        s["opt"], s["buffers"] = opt, buffers
    return s


# ----------------------------------------------------------------------------- one pass, plain


def _plain_norm(s: dict):
    x = s["x"].float()
    mean = x.mean(1)
    c = x - mean[:, None]
    rstd = 1.0 / torch.sqrt((c * c).mean(1) + EPS)
    y = c * rstd[:, None] * s["w"] + s["b"]
    return {"y": y.to(s["x"].dtype), "mean": mean, "rstd": rstd}


def _plain_norm_bwd(s: dict):
    dy = s["dy"].float()
    xh = (s["x"].float() - s["mean"][:, None]) * s["rstd"][:, None]
    g = dy * s["w"]
    dx = s["rstd"][:, None] * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
    if s["dres"] is not None:
        dx = dx + s["dres"].float()
    return {"dx": dx.to(s["x"].dtype), "dw": (dy * xh).sum(0, dtype=torch.float64).float(),
            "db": dy.sum(0, dtype=torch.float64).float()}


def _plain_grad_norm(s: dict) -> torch.Tensor:
    """[norm of all gradients, what they are multiplied with]; the sums in float64."""
    norm = (s["ga"].double().square().sum() + s["gb"].double().square().sum()).sqrt()
    return torch.stack([norm, (MAX_NORM / (norm + 1e-6)).clamp(max=1.0)]).float()


def _mix(x):
    """A 32-bit hash (of an int, or of values in int64)."""
    x = ((x ^ (x >> 16)) * 0x7FEB352D) & M32
    x = ((x ^ (x >> 15)) * 0x846CA68B) & M32
    return x ^ (x >> 16)


def _random(s: dict) -> torch.Tensor:
    """32 random bits an element, from (seed, step, name, index): one strong hash a group of eight elements,
    one multiplication an element."""
    salt = _mix(_mix(_mix(s["step"]) ^ (SEED >> 32)) ^ (SEED & M32))
    key = torch.repeat_interleave(_mix(s["keys"] ^ salt), s["count"], output_size=s["n"] // BLOCK)
    first = torch.cumsum(s["count"], 0) - s["count"]
    block = torch.arange(s["n"] // BLOCK, device=DEV)
    block = block - torch.repeat_interleave(first, s["count"], output_size=s["n"] // BLOCK)
    group = block[:, None] * (BLOCK // 8) + torch.arange(BLOCK // 8, device=DEV)
    x = _mix((key[:, None] + group) & M32)
    x = (x[:, :, None] + torch.arange(8, device=DEV) * 0x9E3779B9) & M32
    x = ((x ^ (x >> 16)) * 0x7FEB352D) & M32
    return (x ^ (x >> 15)).view(-1)


def _bits(x: torch.Tensor) -> torch.Tensor:
    return x.view(torch.int32).long()


def _base(top: torch.Tensor, binades: int) -> tuple[torch.Tensor, torch.Tensor]:
    """The exponent of a block whose largest float has the bits ``top``, and its lowest exponent times 8."""
    e = (top + 0xFFFFF) >> 23
    return e, (e - (binades - 1)).clamp(min=0) * 8


def _encode(m: torch.Tensor, v: torch.Tensor, r_m: torch.Tensor, r_v: torch.Tensor):
    """Codes of the first moments (sign and 7 bits) and of the second (8 bits): exponent and 3 mantissa bits
    of the float above the block's lowest exponent, rounded up where the dropped part plus the random bits
    carries; and the exponents [blocks, 2]."""
    bm, bv = _bits(m).view(-1, BLOCK) & 0x7FFFFFFF, _bits(v).view(-1, BLOCK)
    em, base_m = _base(bm.amax(1, keepdim=True), 16)
    ev, base_v = _base(bv.amax(1, keepdim=True), 32)
    r_m = r_m.view(-1, BLOCK) if r_m.numel() > 1 else r_m
    r_v = r_v.view(-1, BLOCK) if r_v.numel() > 1 else r_v
    qm = (((bm + (r_m << 4)) >> 20) - base_m).clamp(min=0)
    qm = qm | torch.where(m.view(-1, BLOCK) < 0, 128, 0)
    qv = (((bv + (r_v << 4)) >> 20) - base_v).clamp(min=1)
    qv = torch.where(bv > 0, qv, 0)
    return qm.view(-1).to(torch.uint8), qv.view(-1).to(torch.uint8), torch.cat([em, ev], 1).to(torch.uint8)


def _decode(q_m: torch.Tensor, q_v: torch.Tensor, scales: torch.Tensor):
    """The float32 values that codes stand for (each has 4 significant bits: bfloat16 holds it exactly)."""
    e = scales.long()
    base_m, base_v = ((e[:, i, None] - b).clamp(min=0) * 8 for i, b in ((0, 15), (1, 31)))
    qm, qv = q_m.long().view(-1, BLOCK), q_v.long().view(-1, BLOCK)
    c = qm & 127
    m = torch.where(c > 0, (c + base_m) << 20, 0).to(torch.int32).view(torch.float32)
    m = torch.where(qm > 127, -m, m)
    v = torch.where(qv > 0, (qv + base_v) << 20, 0).to(torch.int32).view(torch.float32)
    return m.view(-1), v.view(-1)


def _plain_update(p, m, v, decay, step: int) -> torch.Tensor:
    b1, b2 = ADAMW["betas"]
    d = v.sqrt() * (1.0 / math.sqrt(1.0 - b2 ** step)) + ADAMW["eps"]
    return p * (1.0 - ADAMW["lr"] * ADAMW["weight_decay"] * decay) - (ADAMW["lr"] / (1.0 - b1 ** step)) * (m / d)


def _plain_adamw(s: dict):
    case, na, (b1, b2) = s["case"], s["na"], ADAMW["betas"]
    s["step"] += 1
    out = {}
    g = torch.cat([s["ga"], s["gb"].float()])
    if case["clip"]:
        out["norm"] = _plain_grad_norm(s)
        g = g * out["norm"][1]
    m, v = (s["m"], s["v"]) if case["bits"] == 32 else _decode(s["m"], s["v"], s["scales"])
    m = m * b1 + g * (1.0 - b1)
    v = v * b2 + (g * (1.0 - b2)) * g
    del g
    s["pa"] = _plain_update(s["pa"], m[:na], v[:na], s["decay_a"], s["step"])
    pb = _plain_update(s["pb"].float() if s["master"] is None else s["master"], m[na:], v[na:], 1.0, s["step"])
    s["pb"] = pb.to(s["pb"].dtype)
    if s["master"] is not None:
        s["master"] = out["master"] = pb
    del pb
    if case["bits"] == 8:
        r = _random(s)
        s["m"], s["v"], s["scales"] = _encode(m, v, r & 0xFFFF, r >> 16)
        del r
        m, v = _decode(s["m"], s["v"], s["scales"])
        m, v = m.to(torch.bfloat16), v.to(torch.bfloat16)
    else:
        s["m"], s["v"] = m, v
    return {**out, "pa": s["pa"], "pb": s["pb"], "m": m, "v": v}


def run(state):
    kind = state["case"]["kind"]
    if not own:
        return {"norm": _plain_norm, "norm_bwd": _plain_norm_bwd, "adamw": _plain_adamw,
                "grad_norm": _plain_grad_norm}[kind](state)
    kernels = _module("kernels")
    if kind == "norm":
        y, mean, rstd = kernels.layer_norm(state["x"], state["w"], state["b"], EPS)
        return {"y": y, "mean": mean, "rstd": rstd}
    if kind == "norm_bwd":
        dx, dw, db = kernels.layer_norm_bwd(state["dy"], state["x"], state["w"], state["mean"], state["rstd"],
                                            dres=state["dres"])
        return {"dx": dx, "dw": dw, "db": db}
    if kind == "grad_norm":
        return kernels.grad_norm(list(state["grads"].values()), MAX_NORM)
    opt, buffers = state["opt"], state["buffers"]
    opt.step()
    out = {"norm": opt.grad_norm} if state["case"]["clip"] else {}
    if state["case"]["master"]:
        out["master"] = buffers["master"]
    m, v = opt.moments() if state["case"]["bits"] == 8 else (buffers["exp_avg"], buffers["exp_avg_sq"])
    return {**out, "pa": state["pa"], "pb": state["pb"], "m": m, "v": v}


# ----------------------------------------------------------------------------- what a pass cannot do without


def work(case: dict) -> dict:
    size = {"float32": 4, "bfloat16": 2}[case["dtype"]]
    h = case["hidden"]
    if case["kind"] in ("norm", "norm_bwd"):
        n = case["tokens"] * h
        if case["kind"] == "norm":
            return {"bytes": 2 * n * size + 8 * case["tokens"] + 8 * h, "flops": 8 * n}
        return {"bytes": (3 + case["residual"]) * n * size + 8 * case["tokens"] + 12 * h, "flops": 14 * n}
    n, r = (case["experts"] + case["shared"]) * 3 * h * case["ffn"], (case["experts"] + 2) * h
    if case["kind"] == "grad_norm":
        return {"bytes": n * size + 4 * r, "flops": 2 * (n + r)}
    # Gradient and weight in, weight out (with a master: the master in and out, the weight out); the moments
    # in and out, those of 8 bits also as the bfloat16 values they stand for.
    per = (2 + 2 * size if not case["master"] else 8 + 2 * size) if size == 2 else 12
    state = 16 if case["bits"] == 32 else 4 + 4
    return {"bytes": n * (per + state) + r * (12 + state), "flops": 14 * (n + r)}


# ----------------------------------------------------------------------------- from the definitions, in 64 bits


def _exact_norm(case: dict, seed: int):
    s = _norm_inputs(case, seed)
    x, w = s["x"].double(), s["w"].double()
    if case["kind"] == "norm":
        mean = x.mean(1)
        rstd = ((x - mean[:, None]).square().mean(1) + EPS).rsqrt()
        return {"y": torch.addcmul(s["b"].double(), (x - mean[:, None]) * rstd[:, None], w), "mean": mean,
                "rstd": rstd}
    # d/dx of sum(dy * y) with the statistics as functions of x, at the ones that were kept.
    dy, mean, rstd = s["dy"].double(), s["mean"].double()[:, None], s["rstd"].double()[:, None]
    h = case["hidden"]
    c = x - mean
    a = dy * w
    d_rstd = (a * c).sum(1, keepdim=True)
    dx = a * rstd - (a.sum(1, keepdim=True) * rstd) / h - c * rstd.pow(3) * d_rstd / h
    if s["dres"] is not None:
        dx = dx + s["dres"].double()
    return {"dx": dx, "dw": (dy * c * rstd).sum(0), "db": dy.sum(0)}


def _exact_code(x: torch.Tensor, r: torch.Tensor, binades: int, keep: bool) -> torch.Tensor:
    """The values that magnitudes ``x`` [blocks, BLOCK] are stored as: a multiple of 1/8 of their binade, one
    up where the fraction left plus the random one (r / 2^16) reaches one; nothing under the block's lowest
    binade but zero, or (keep) the smallest value there."""
    mant, e = torch.frexp(x.amax(1, keepdim=True))
    e = e - 1 + (2 * mant > 1.875).int()        # the block's exponent: x rounded up fits 1.875 * 2^e
    low = torch.clamp(e - (binades - 1), min=-127).double()
    _, ex = torch.frexp(x)
    step = torch.exp2(torch.clamp(ex.double() - 1, min=-126) - 3)
    q = step * torch.floor(x / step + r.double() / 65536.0)
    least = torch.where(low > -127, torch.exp2(low) * 1.125, 2.0 ** -129)
    small = least if keep else torch.zeros_like(least)
    return torch.where(x == 0, 0.0, torch.where(q < least, small, q))


def _exact_adamw(case: dict, seed: int):
    s = _optim_inputs(case, seed)
    b1, b2 = ADAMW["betas"]
    na, t = s["na"], STEPS_DONE + 1
    out = {}
    g = torch.cat([s["ga"].double(), s["gb"].double()])
    if case["clip"]:
        norm = g.norm()
        coef = torch.clamp(MAX_NORM / (norm + 1e-6), max=1.0)
        out["norm"] = torch.stack([norm, coef])
        g *= coef
    if case["bits"] == 8:
        m, v = (x.double() for x in _decode(s["m"], s["v"], s["scales"]))
    else:
        m, v = s["m"].double(), s["v"].double()
    m.mul_(b1).add_(g, alpha=1 - b1)
    v.mul_(b2).add_(g.square_(), alpha=1 - b2)
    del g
    wd = torch.ones(s["n"], dtype=torch.float64, device=DEV)
    wd[:na] = s["decay_a"].double()
    p = torch.cat([s["pa"].double(), (s["pb"] if s["master"] is None else s["master"]).double()])
    p.mul_(1 - ADAMW["lr"] * ADAMW["weight_decay"] * wd)
    del wd
    p -= ADAMW["lr"] / (1 - b1 ** t) * m / ((v / (1 - b2 ** t)).sqrt() + ADAMW["eps"])
    if s["master"] is not None:
        out["master"] = p[na:]
    if case["bits"] == 8:
        s["step"] = t
        r = _random(s).view(-1, BLOCK)
        sign = torch.where(m < 0, -1.0, 1.0)
        m = _exact_code(m.abs().view(-1, BLOCK), r & 0xFFFF, 16, False).view(-1) * sign
        v = _exact_code(v.view(-1, BLOCK), r >> 16, 32, True).view(-1)
    return {**out, "pa": p[:na], "pb": p[na:], "m": m, "v": v}


def exact(case: dict, seed: int):
    if case["kind"] in ("norm", "norm_bwd"):
        return _exact_norm(case, seed)
    if case["kind"] == "adamw":
        return _exact_adamw(case, seed)
    s = _optim_inputs(case, seed)
    norm = torch.hypot(s["ga"].double().norm(), s["gb"].double().norm())
    return torch.stack([norm, torch.clamp(MAX_NORM / (norm + 1e-6), max=1.0)])
