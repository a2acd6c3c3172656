"""The router losses' and the 4-bit entry points without a GPU: arguments are refused before any launch, sizes are
pure functions, and the oracle's 4-bit format is pinned to values worked out by hand."""

from __future__ import annotations

import ctypes
import math
from types import SimpleNamespace

import pytest
import torch

from oracle import mx4_ref as R4
from resihp_megatron_amd import _capi as C
from resihp_megatron_amd import kernels as K
from resihp_megatron_amd import layer as L
from resihp_megatron_amd import moe

FAKE = ctypes.c_void_p(4096)    # 16-byte aligned, never dereferenced: validation fails first
ODD = ctypes.c_void_p(4104)


def _loss(T=8, E=8, k=2, S=1, dtype=C.F32, score=C.SCORE_SIGMOID, logits=FAKE, topi=FAKE, seqs=None, out=FAKE, ws=FAKE,
          ws_bytes=1 << 30):
    C.call("rhp_router_loss", logits, dtype, topi, None, seqs, T, E, k, S, score, out, out, out, out, ws, ws_bytes, None)


@pytest.mark.parametrize("kw,msg", [
    (dict(dtype=C.BF16), "float32 or float64"),
    (dict(T=-1), "T >= 0"),
    (dict(T=1 << 31), "T >= 0"),
    (dict(E=0), "E <= 1024"),
    (dict(E=1025), "E <= 1024"),
    (dict(k=0), "k <= 16"),
    (dict(k=17), "k <= 16"),
    (dict(score=7), "score function"),
    (dict(S=0), "sequences"),
    (dict(S=2), "sequences"),
    (dict(S=(1 << 20) + 1, seqs=FAKE), "sequences"),
    (dict(logits=None), "null pointer"),
    (dict(topi=None), "null pointer"),
    (dict(logits=ctypes.c_void_p(4098)), "unaligned logits"),
    (dict(out=None), "null pointer"),
    (dict(ws=None), "workspace"),
    (dict(ws=ODD), "workspace"),
    (dict(ws_bytes=16), "workspace"),
])
def test_router_loss_rejects_bad_arguments(kw, msg):
    with pytest.raises(RuntimeError, match=msg):
        _loss(**kw)


def test_router_loss_bwd_rejects_bad_arguments():
    call = lambda counts, tokens, d, T=8: C.call(  # noqa: E731
        "rhp_router_loss_bwd", FAKE, FAKE, FAKE, C.F32, FAKE, None, None, T, 8, 2, 1, C.SCORE_SOFTMAX, counts, tokens, d,
        None)
    for args in ((None, FAKE, ODD), (FAKE, None, ODD), (FAKE, FAKE, None), (FAKE, FAKE, FAKE)):
        with pytest.raises(RuntimeError, match="null pointer, or dlogits is logits"):
            call(*args)
    call(None, None, None, T=0)   # nothing to do


@pytest.mark.parametrize("args,msg", [
    (dict(xd=C.E4M3), "unsupported dtype"),
    (dict(rd=C.F64), "float64 router"),
    (dict(xd=C.F64), "float64 router"),
    (dict(T=-1), "T >= 0"),
    (dict(E=1025), "E <= 1024"),
    (dict(h=1 << 23), "2\\^22 columns"),
    (dict(dl=None), "null pointer"),
    (dict(w=None), "router's weight"),
    (dict(x=None), "the tokens"),
    (dict(x=ODD), "16-byte aligned"),
    (dict(T=1 << 20, ws=None), "workspace"),
    (dict(T=1 << 20, ws_bytes=1024), "workspace"),
    (dict(T=1 << 30, h=65), "2 M tokens"),
])
def test_router_logits_bwd_rejects_bad_arguments(args, msg):
    a = dict(dl=FAKE, x=FAKE, xd=C.BF16, w=FAKE, rd=C.F32, T=8, h=64, E=8, ws=FAKE, ws_bytes=1 << 40) | args
    with pytest.raises(RuntimeError, match=msg):
        C.call("rhp_router_logits_bwd", a["dl"], a["x"], a["xd"], a["w"], a["rd"], a["T"], a["h"], a["E"],
               ctypes.c_void_p(8192), ctypes.c_void_p(12288), a["ws"], a["ws_bytes"], None)


@pytest.mark.parametrize("args,msg", [
    (dict(dtype=C.F64), "unsupported dtype"),
    (dict(rows=-1), "bad sizes"),
    (dict(rows=(1 << 31) - 16384), "bad sizes"),
    (dict(cols=0), "bad sizes"),
    (dict(cols=(1 << 31) - 256), "bad sizes"),
    (dict(offsets=FAKE, G=65), "1 to 64"),
    (dict(offsets=FAKE, G=0), "1 to 64"),
    (dict(offsets=FAKE, G=1, n=2), "of one matrix"),
    (dict(rq=None, cq=None), "null pointer"),
    (dict(rs=None), "codes without scales"),
    (dict(cs=None), "codes without scales"),
    (dict(rq=ODD), "16-byte aligned"),
    (dict(x=[4097]), "aligned to its elements"),
    (dict(x=[0]), "null"),
    (dict(rows=1 << 30, cols=1 << 20), "too many tiles"),
])
def test_quantize_rejects_bad_arguments(args, msg):
    a = dict(x=[4096], n=1, dtype=C.BF16, rows=8, cols=8, offsets=None, G=0, rq=FAKE, rs=FAKE, cq=FAKE, cs=FAKE) | args
    with pytest.raises(RuntimeError, match=msg):
        C.call("rhp_mx4_quantize", a["n"], C.ptr_array(a["x"] * a["n"]), a["dtype"], a["rows"], a["cols"], a["offsets"],
               a["G"], a["rq"], a["rs"], a["cq"], a["cs"], None)


@pytest.mark.parametrize("args,msg", [
    (dict(dtype=C.F64), "unsupported dtype"),
    (dict(cols=0), "bad sizes"),
    (dict(q=None), "null pointer"),
    (dict(q=ODD), "16-byte aligned"),
    (dict(out=ctypes.c_void_p(4097)), "16-byte aligned, the output"),
    (dict(n=1 << 16, rows=1 << 16), "2\\^35"),
])
def test_dequantize_rejects_bad_arguments(args, msg):
    a = dict(q=FAKE, n=1, rows=8, cols=8, dtype=C.BF16, out=FAKE) | args
    with pytest.raises(RuntimeError, match=msg):
        C.call("rhp_mx4_dequantize", a["q"], FAKE, a["n"], a["rows"], a["cols"], a["dtype"], a["out"], None)


@pytest.mark.parametrize("args,msg", [
    (dict(G=0), "1 to 64"),
    (dict(G=65), "1 to 64"),
    (dict(epi=5), "epilogue"),
    (dict(N=12), "multiple of 8"),
    (dict(K=0), "bad sizes"),
    (dict(a=None), "null pointer"),
    (dict(out=None), "null pointer"),
    (dict(act=FAKE), "forward activations"),
    (dict(epi=1), "forward activations"),
    (dict(epi=3), "backward ones read aux"),
    (dict(a=ODD), "16-byte aligned"),
    (dict(N=1 << 20, K=1 << 14), "2 GiB"),
])
def test_gemm_rejects_bad_arguments(args, msg):
    a = dict(epi=0, G=2, rows=8, N=64, K=64, a=FAKE, out=FAKE, act=None, aux=None) | args
    with pytest.raises(RuntimeError, match=msg):
        C.call("rhp_mx4_gemm", a["epi"], a["G"], FAKE, a["rows"], a["N"], a["K"], a["a"], FAKE, FAKE, FAKE, a["out"],
               a["act"], a["aux"], None)


@pytest.mark.parametrize("args,msg", [
    (dict(G=65), "1 to 64"),
    (dict(N=12), "multiple of 8"),
    (dict(out=None), "unaligned output"),
    (dict(a=None), "null pointer"),
    (dict(a=ODD), "16-byte aligned"),
    (dict(rows=1 << 24, N=1 << 10), "2 GiB"),
])
def test_wgrad_rejects_bad_arguments(args, msg):
    a = dict(G=2, rows=8, M=64, N=64, a=FAKE, out=FAKE) | args
    with pytest.raises(RuntimeError, match=msg):
        C.call("rhp_mx4_wgrad", a["G"], FAKE, a["rows"], a["M"], a["N"], a["a"], FAKE, FAKE, FAKE, a["out"], None)


@pytest.mark.parametrize("args,msg", [
    (dict(G=65), "1 to 64"),
    (dict(K=60), "multiples of 8"),
    (dict(N=60), "multiples of 8"),
    (dict(act=5), "unknown activation"),
    (dict(x=None), "null pointer"),
    (dict(x=ODD), "16-byte aligned"),
    (dict(rows=(1 << 31) - 4096), "too many rows"),
    (dict(K=1 << 23), "2\\^23 columns"),
])
def test_rows_gemm_rejects_bad_arguments(args, msg):
    a = dict(G=2, rows=8, N=64, K=64, act=-1, x=FAKE) | args
    with pytest.raises(RuntimeError, match=msg):
        C.call("rhp_mx4_rows_gemm", a["G"], FAKE, a["rows"], a["N"], a["K"], a["act"], a["x"], FAKE, FAKE, FAKE, None)


def test_sizes():
    lib = C.lib()
    assert [lib.rhp_mx4_padded_rows(r, g) for r, g in ((0, 1), (1, 1), (128, 1), (129, 1), (1, 2), (300, 4))] == \
        [0, 128, 128, 256, 128, 768]
    # every way to place the rows fits: at most 127 places more than rows for each group
    assert all(lib.rhp_mx4_padded_rows(r, 3) >= sum(-(-c // 128) * 128 for c in (a, b, r - a - b))
               for r in (5, 130, 400) for a in range(0, r, 7) for b in range(0, r - a, 11))
    # 64 tokens a block at least, one partial row of E sums, E counts, lse^2 and tokens for a block and a sequence
    assert lib.rhp_router_loss_workspace_bytes(64, 8, 1, C.F32) == 2 * 9 * 8
    assert lib.rhp_router_loss_workspace_bytes(1 << 20, 64, 3, C.F64) == (256 + 3) * 65 * 12
    assert lib.rhp_router_loss_workspace_bytes(-1, 8, 1, C.F32) == 0
    assert lib.rhp_router_logits_bwd_workspace_bytes(64, 2048, 64, C.BF16) == 0      # one slice
    assert lib.rhp_router_logits_bwd_workspace_bytes(16384, 2048, 64, C.BF16) == 16 * 64 * 2048 * 4
    assert lib.rhp_router_logits_bwd_workspace_bytes(-1, 64, 8, C.F32) == 0


def test_python_entry_points_refuse_cpu_tensors_and_what_is_no_mx4():
    x, off = torch.zeros(8, 64, dtype=torch.bfloat16), torch.tensor([0, 8], dtype=torch.int32)
    q = K.Mx4(torch.zeros(8, 32, dtype=torch.uint8), torch.zeros(1, 8, 4, dtype=torch.uint8), 64)
    for call in (lambda: K.mx4_quantize(x), lambda: K.mx4_dequantize(q), lambda: K.mx4_gemm(q, q, off),
                 lambda: L.mx4_linear(x, x[None], off), lambda: L.Mx4Experts([torch.zeros(32, 64)], [torch.zeros(64, 16)]),
                 lambda: L.router_loss(torch.zeros(8, 4), torch.zeros(8, 2, dtype=torch.int32)),
                 lambda: K.router_logits_bwd(torch.zeros(8, 4), x, torch.zeros(4, 64))):
        with pytest.raises(RuntimeError, match="HIP device"):
            call()
    for call in (lambda: K.mx4_dequantize(x), lambda: K.mx4_gemm(x, q, off), lambda: K.mx4_wgrad(x, q, off),
                 lambda: K.mx4_gemm_act(x, q, off, "gelu"), lambda: K.mx4_rows_gemm(x, x, off)):
        with pytest.raises(RuntimeError, match="must be an Mx4, got Tensor"):
            call()
    for call in (lambda: K.mx4_quantize(x, "diagonal"), lambda: K.mx4_quantize([])):
        with pytest.raises(RuntimeError):
            call()


@pytest.mark.parametrize("length,rows,groups", [(128, 1000, 1), (1024, 1000, 2), (1152, 1000, 1), (128, 0, 1), (128, -5, 1)])
def test_wgrad_refuses_matrices_whose_places_are_not_those_of_their_groups(length, rows, groups, monkeypatch):
    """The kernel goes through the places that rows and groups ask for: codes of fewer would be read past their end."""
    monkeypatch.setattr(K, "_need_cuda", lambda *ts: torch.device("cpu"))
    monkeypatch.setattr(K, "_call", lambda *a: pytest.fail("a launch"))
    q = K.Mx4(torch.zeros(8, length // 2, dtype=torch.uint8), torch.zeros(length // 128, 8, 4, dtype=torch.uint8), length, rows,
              groups)
    with pytest.raises(RuntimeError, match="places"):
        K.mx4_wgrad(q, q, torch.zeros(groups + 1, dtype=torch.int32))


def test_received_rows_do_not_run_in_4_bits_silently():
    for bits, msg in ((4, "model's dtype"), (8, "experts_bits must be")):
        runtime = SimpleNamespace(cfg=moe.MoEConfig(experts_bits=bits))
        with pytest.raises(ValueError, match=msg):
            moe.EPRuntime.expert_outputs(runtime, None, None)


# ----------------------------------------------------------------------------- the oracle's format

def test_oracle_codes_by_hand():
    """A block whose largest magnitude is 6: scale 1 (floor(log2 6) - 2 = 0); ties go to the even code."""
    block = torch.tensor([0.0, 0.25, 0.26, 0.5, 0.75, 1.0, 1.25, 1.5, 1.75, 2.0, 2.5, 2.6, 3.0, 3.5, 4.0, 5.0, 5.1, 6.0, -0.25,
                          -0.3, -6.0, -0.0] + [0.0] * 10)
    code, scale = R4.quantize(block[None])
    assert scale.tolist() == [[127]]
    assert code[0, 0, :22].tolist() == [0, 0, 1, 1, 2, 2, 2, 3, 4, 4, 4, 5, 5, 6, 6, 6, 7, 7, 8, 9, 15, 8]
    # 7.9 shares floor(log2) with 4: its scale is 1 and it saturates to 6.
    assert R4.round4(torch.tensor([[7.9, 4.0]])).tolist() == [[6.0, 4.0]]


@pytest.mark.parametrize("top,code", [(0.0, 0), (2.0 ** -149, 0), (2.0 ** -126, 0), (2.0 ** -125, 0), (2.0 ** -124, 1),
                                      (1.0, 125), (3.9, 126), (4.0, 127), (3.3e38, 252)])
def test_oracle_scales_by_hand(top, code):
    assert R4.quantize(torch.tensor([[top, 0.0]], dtype=torch.float64))[1].item() == code


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_oracle_blocks_that_are_not_finite(bad):
    x = torch.ones(2, 40)
    x[1, 33] = bad
    v = R4.round4(x)
    assert v[0].tolist() == [1.0] * 40 and v[1, :32].tolist() == [1.0] * 32 and torch.isnan(v[1, 32:]).all()


def test_oracle_rounding_is_off_by_at_most_half_a_step():
    x = torch.randn(64, 96, generator=torch.Generator().manual_seed(0), dtype=torch.float64)
    code, scale = R4.quantize(x)
    s = torch.exp2(scale.double() - 127).repeat_interleave(32, 1)
    err, a = (R4.values(code, scale, 96) - x).abs(), x.abs() / s
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0)) * s
    assert (err <= step / 2 + (a > 6) * s).all()   # past 6 the code saturates: off by less than 2


def test_oracle_bytes():
    code = torch.arange(64).view(1, 2, 32) % 16
    codes, scales = R4.pack(code, torch.tensor([[7, 255]]))
    assert codes.shape == (1, 32) and codes[0, :3].tolist() == [0x10, 0x32, 0x54]
    assert scales.tolist() == [[[7, 255, 0, 0]]]
    assert R4.padded([1, 0, 129, 3]) == [0, 128, 128, 384]
