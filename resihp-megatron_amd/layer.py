"""The fused MoE layer: route -> dispatch -> permute -> grouped expert GEMMs -> combine, and its backward.

One ``torch.autograd.Function`` drives the gfx950 kernels of
``libresihp_moe.so``.  Its semantics are those of ``reference_forward``
(resihp/runtime/moe.py:90-101) for the experts in the local window
[e0, e1): ``out = x + sum over local slots of gate * expert(x) + sum of shared
experts(x)``.  With the full window it is the whole layer; with a partial
window it is one GPU's expert-parallel share with its tokens already received.

Expert weights stay separate tensors (one per expert and matrix), so the
autograd graph, the optimizer and expert re-placement see per-expert
parameters exactly as in the reference; the kernels reach them through
per-group pointers.
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import NamedTuple

import torch
from torch.autograd.function import once_differentiable

from . import kernels as K
from .fp8 import ACT, DH, DY, X, Fp8State


@dataclass(frozen=True)
class LayerMeta:
    num_experts: int
    top_k: int
    ffn: int
    act: str = "gelu"
    score: str = "softmax"
    normalize: bool = True
    gate_scale: float = 1.0
    e0: int = 0
    e1: int | None = None
    n_src: int = 1
    num_shared: int = 0
    shared_ffn: int = 0

    @property
    def window(self) -> tuple[int, int]:
        return self.e0, self.num_experts if self.e1 is None else self.e1

    @property
    def full(self) -> bool:
        return self.window == (0, self.num_experts)


class Norm(NamedTuple):
    """The layer norm in front of a pre-norm block (resihp/runtime/reference_model.py:195-234)."""

    weight: torch.Tensor | None
    bias: torch.Tensor | None
    eps: float = 1e-5


class LossTokens(NamedTuple):
    """What a layer's router losses are taken over (``router_loss``): the tokens that count, and sequences."""

    mask: torch.Tensor | None = None
    seq_offsets: torch.Tensor | None = None


class RouterLosses(NamedTuple):
    """Balance loss, z loss and the counts [S, E] they are made of, which the backward reads (unchanged until then)."""

    balance: torch.Tensor
    z: torch.Tensor
    counts: torch.Tensor


def _fc1_rows(act: str, f: int) -> int:
    return 2 * f if act == "swiglu" else f


# The backward's input-gradient and weight-gradient products are independent.  Run concurrently, the
# weight gradients go to a second stream of the device (default priority), so their tiles fill the CUs
# the input-gradient products leave idle: every CU reaches a tile's epilogue at the same time, so the
# epilogues' HBM traffic comes in bursts, and the last round of a launch leaves CUs empty.  That pays
# for short reductions (measured: dsv2lite +1.4 %, the EP-128 share +2.7 %); input-gradient products
# whose reduction is long enough for the K split of their last round (h or the fc1 rows >= 8192) fill
# that round themselves and lose L2 locality to a concurrent launch (Mixtral shape: -4 %), so they keep
# the GPU to themselves.  "auto" chooses by that rule; True / False force it.
CONCURRENT_BACKWARD: bool | str = "auto"
SPLIT_MIN_K = 8192   # the reduction length from which the input-gradient products split their last round


def _concurrent(h: int, F1: int) -> bool:
    if CONCURRENT_BACKWARD == "auto":
        return max(h, F1) < SPLIT_MIN_K
    return bool(CONCURRENT_BACKWARD)
# Add the router term of the input gradient in fc1's input-gradient epilogue (layers whose experts are
# all local) instead of reading k router rows per token in the token backward.
FOLD_ROUTER_TERM = True
_side_streams: dict[int, torch.cuda.Stream] = {}


def _side_stream(dev: torch.device) -> torch.cuda.Stream:
    idx = dev.index if dev.index is not None else torch.cuda.current_device()
    st = _side_streams.get(idx)
    if st is None:
        st = torch.cuda.Stream(device=idx)
        _side_streams[idx] = st
    return st


def expert_backward(dys, acts, hpres, offsets, rows_from_offsets: bool, rows_cap: int, fc1s, fc2s, f: int,
                    act: str, dhpre, xs, dxs, dw1, dw2, router=None) -> None:
    """The expert FFN backward (fc2 then fc1, input and weight gradients) of a group launch.

    The weight gradients go to the side stream when the products run concurrently (CONCURRENT_BACKWARD);
    the current stream waits for them before returning, so every output is ordered on it as usual.
    ``router`` = (router_w, e0, perm, dl) folds the router term into fc1's input gradient."""
    fc1s, fc2s, dw1, dw2 = K.group(fc1s), K.group(fc2s), K.group(dw1), K.group(dw2)

    def fc1_dgrad():
        if router is None:
            K.expert_fc1_bwd(dhpre, xs, offsets, rows_from_offsets, rows_cap, fc1s, f, act, dxs, None)
        else:
            K.expert_fc1_dgrad_router(dhpre, offsets, rows_cap, fc1s, f, act, *router, dxs)

    if not _concurrent(fc1s[0].shape[1], fc1s[0].shape[0]):
        K.expert_fc2_bwd(dys, acts, hpres, offsets, rows_from_offsets, rows_cap, fc2s, act, dhpre, dw2)
        if dxs:
            fc1_dgrad()
        K.expert_fc1_bwd(dhpre, xs, offsets, rows_from_offsets, rows_cap, fc1s, f, act, None, dw1)
        return
    main = torch.cuda.current_stream(offsets.device)
    side = _side_stream(offsets.device)
    side.wait_stream(main)
    with torch.cuda.stream(side):
        K.expert_fc2_bwd(dys, acts, hpres, offsets, rows_from_offsets, rows_cap, fc2s, act, None, dw2)
    K.expert_fc2_bwd(dys, acts, hpres, offsets, rows_from_offsets, rows_cap, fc2s, act, dhpre, None)
    side.wait_stream(main)
    with torch.cuda.stream(side):
        K.expert_fc1_bwd(dhpre, xs, offsets, rows_from_offsets, rows_cap, fc1s, f, act, None, dw1)
    if dxs:
        fc1_dgrad()
    main.wait_stream(side)


def _fp8_weight_casts(st: Fp8State, fc1s, fc2s, main: torch.cuda.Stream):
    """Starts the casts of the expert weights on the side stream: fc1's while the routing, dispatch and
    permute run, fc2's while fc1's product runs.  Returns the code buffers and the events that mark them
    written (the buffers are allocated on the caller's stream, which waits for the events before use)."""
    w1q, w2q = st.weight_codes(fc1s), st.weight_codes(fc2s)
    side = _side_stream(main.device)
    side.wait_stream(main)
    with torch.cuda.stream(side):
        st.cast_weights("fc1", fc1s, w1q)
        ev1 = torch.cuda.Event()
        ev1.record(side)
        st.cast_weights("fc2", fc2s, w2q)
        ev2 = torch.cuda.Event()
        ev2.record(side)
    return w1q, w2q, ev1, ev2


def _fp8_forward(st: Fp8State, meta: LayerMeta, offsets, P, xq, fc1s, fc2s, hpre, y, wcast):
    """Expert FFN forward in fp8 on the permuted input's codes ``xq``; returns what the backward needs
    (the row-major codes).

    The fc1 product's epilogue casts the activation straight to fp8 (no bf16 activation rows).  Every
    operand is kept as row-major codes only: the backward products read them N-contiguous and transpose
    in LDS (fp8 product modes 2 and 3).
    """
    G, f = st.G, meta.ffn
    h = xq.shape[1]
    w1q, w2q, ev1, ev2 = wcast
    main = torch.cuda.current_stream(xq.device)
    sw1 = st.scale_inv[st.w1(0):st.w1(0) + G]
    sw2 = st.scale_inv[st.w2(0):st.w2(0) + G]
    # The product casts tile each expert's rows in blocks of 128 (the padded offsets); no transposed copy
    # is written.
    poff = K.fp8_padded_offsets(offsets)
    aq = None
    if P > 0:
        epi = "swiglu_fwd" if meta.act == "swiglu" else "gelu_fwd"
        main.wait_event(ev1)
        aq, _ = st.gemm_cast(ACT, epi, offsets, poff, P, [xq] * G, "e4m3", w1q, f, h, f, st.scale_inv[X:X + 1],
                             sw1, cs=[hpre] * G, transposed=False)
        main.wait_event(ev2)
        K.fp8_gemm(0, "store", offsets, P, [aq] * G, "e4m3", w2q, "e4m3", h, f, 0, f, [y] * G,
                   st.scale_inv[ACT:ACT + 1], sw2)
    main.wait_event(ev2)   # the weight casts are complete (and their amax raised) before the layer returns
    return dict(poff=poff, xq=xq, aq=aq, w1q=w1q, w2q=w2q, sw1=sw1, sw2=sw2)


def _fp8_backward(st: Fp8State, q8: dict, meta: LayerMeta, offsets, P, dyq, hpre, dxp, dw1, dw2):
    """Expert FFN backward in fp8 (e5m2 gradients, e4m3 weights and activations) from the codes ``dyq`` of
    the output rows' gradient.

    The fc2 input-gradient product's epilogue casts the pre-activation gradient straight to fp8.  The
    input-gradient products read the row-major weight codes as [K, N] (mode 2) and the weight gradients
    the row-major activation and gradient codes (mode 3).
    """
    G, f = st.G, meta.ffn
    h = dyq.shape[1]
    F1 = _fc1_rows(meta.act, f)
    if P == 0:
        for w in (*dw1, *dw2):
            w.zero_()
        return
    s = st.scale_inv
    poff = q8["poff"]
    epi = "swiglu_bwd" if meta.act == "swiglu" else "gelu_bwd"
    dhq, _ = st.gemm_cast(DH, epi, offsets, poff, P, [dyq] * G, "e5m2", q8["w2q"], f, h, f, s[DY:DY + 1],
                          q8["sw2"], auxs=[hpre] * G, transposed=False, x_kn=True)
    K.fp8_gemm(3, "store", offsets, P, [dyq], "e5m2", [q8["aq"]], "e4m3", f, 0, h, f, list(dw2), s[DY:DY + 1],
               s[ACT:ACT + 1])
    if dxp is not None:
        K.fp8_gemm(2, "store", offsets, P, [dhq] * G, "e5m2", q8["w1q"], "e4m3", h, F1, 0, f, [dxp] * G,
                   s[DH:DH + 1], q8["sw1"])
    K.fp8_gemm(3, "store", offsets, P, [dhq], "e5m2", [q8["xq"]], "e4m3", h, 0, F1, f, list(dw1), s[DH:DH + 1],
               s[X:X + 1])


def _mx4_tensors(*qs) -> tuple[list[torch.Tensor], list]:
    """The tensors of 4-bit matrices (or Nones), to be saved for a backward, and what else they are made of."""
    return ([t for q in qs if q is not None for t in (q.codes, q.scales)],
            [None if q is None else (q.length, q.rows, q.groups) for q in qs])


def _mx4_again(tensors, rest) -> list:
    """The matrices of ``_mx4_tensors``."""
    it = iter(tensors)
    return [None if r is None else K.Mx4(next(it), next(it), *r) for r in rest]


def _mx4_forward(meta: LayerMeta, offsets, xp, fc1s, fc2s, keep: bool, need_x: bool):
    """Expert FFN forward on operands in 4 bits from the permuted rows; returns (y, the activation's input for the
    backward, 4-bit matrices for it).

    Each operand is read once: the rows and activations are quantised along their rows for the forward products
    and along their columns, by expert, for the weights' gradients; the weights along their rows and, for the
    input gradients, their columns."""
    def quantize(t, both, groups=None):
        return K.mx4_quantize(t, "both", groups) if both else (K.mx4_quantize(t), None)

    xr, xc = quantize(xp, keep, offsets)
    w1, w1t = quantize(fc1s, keep and need_x)
    a, hpre = K.mx4_gemm_act(xr, w1, offsets, meta.act, keep)
    ar, ac = quantize(a, keep, offsets)
    w2, w2t = quantize(fc2s, keep)
    return K.mx4_gemm(ar, w2, offsets), hpre, (xc, ac, w1t, w2t)


def _mx4_backward(q4, hpre, meta: LayerMeta, offsets, dy, need_x: bool):
    """Expert FFN backward on operands in 4 bits: (dxp or None, dw1 [G, F1, h], dw2 [G, h, f])."""
    xc, ac, w1t, w2t = q4
    dr, dc = K.mx4_quantize(dy, "both", offsets)
    dh = K.mx4_gemm_act_bwd(dr, w2t, offsets, meta.act, hpre)
    dw2 = K.mx4_wgrad(dc, ac, offsets)
    hr, hc = K.mx4_quantize(dh, "both", offsets) if need_x else (None, K.mx4_quantize(dh, "cols", offsets))
    dxp = K.mx4_gemm(hr, w1t, offsets) if need_x else None
    return dxp, K.mx4_wgrad(hc, xc, offsets), dw2


def _fc1_fwd(xs, offsets, rows_from_offsets: bool, rows_cap: int, fc1s, f: int, act: str, hpres, acts) -> None:
    """fc1's forward product; ``hpres`` None: without what a backward needs."""
    if hpres is None:
        K.expert_fc1_act(xs, offsets, rows_from_offsets, rows_cap, fc1s, f, act, acts)
    else:
        K.expert_fc1_fwd(xs, offsets, rows_from_offsets, rows_cap, fc1s, f, act, hpres, acts)


class _MoELayerFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, meta: LayerMeta, opts, x, router_w, bias, norm_w, norm_b, *weights):
        fp8, mx4, losses, grad_mode, norm_eps = opts
        # Without a backward to come (no_grad, or no input that needs a gradient) fc1 writes only the
        # activation rows, and nothing is saved.
        keep = fp8 is not None or (grad_mode and any(ctx.needs_input_grad))
        e0, e1 = meta.window
        G = e1 - e0
        S = meta.num_shared
        W = 0 if isinstance(mx4, Mx4Experts) else G   # the routed experts' weights among ``weights``
        fc1s, fc2s = K.group(weights[:W]), K.group(weights[W:2 * W])
        sfc1s, sfc2s = list(weights[2 * W:2 * W + S]), list(weights[2 * W + S:2 * W + 2 * S])
        T, h = x.shape
        k, f = meta.top_k, meta.ffn
        fs = meta.shared_ffn or f
        shared_off = shared_h = shared_a = shared_y = None
        K.need_device(x, router_w, fc1s, fc2s, sfc1s, sfc2s)
        main = torch.cuda.current_stream(x.device)
        # Behind a norm the layer works on its output; x itself is only the residual.
        res, mean, rstd = x, None, None
        if norm_eps is not None:
            x, mean, rstd = K.layer_norm(res, norm_w, norm_b, norm_eps)
        # Shared experts need only x: concurrently with the routing and the routed experts on a side
        # stream where the products run concurrently, else after them.
        shared_side = S > 0 and T > 0 and _concurrent(h, _fc1_rows(meta.act, fs))
        if S:
            shared_off = torch.arange(S + 1, dtype=torch.int32, device=x.device) * T
            shared_h = [x.new_empty(T, _fc1_rows(meta.act, fs)) for _ in range(S)] if keep else None
            shared_a = [x.new_empty(T, fs) for _ in range(S)]
            shared_y = [x.new_empty(T, h) for _ in range(S)]
        if shared_side:
            side = _side_stream(x.device)
            side.wait_stream(main)
            with torch.cuda.stream(side):
                _fc1_fwd([x] * S, shared_off, False, T, sfc1s, fs, meta.act, shared_h, shared_a)
                K.expert_fc2_fwd(shared_a, shared_off, False, T, sfc2s, shared_y)
        # fp8 experts (never with shared experts): the weight casts start now, on the side stream.
        wcast = _fp8_weight_casts(fp8, weights[:G], weights[G:2 * G], main) if fp8 is not None else None
        logits, topi, gates = K.route(x, router_w, bias, k, meta.score, meta.normalize, meta.gate_scale)
        loss = None if losses is None else K.router_loss(logits, topi, meta.score, *losses)
        plan = K.dispatch(topi, meta.num_experts, e0, e1, meta.n_src)
        # The reference materialises counts on the host here too (moe.py:210-211);
        # with every expert local the row count is known without a sync.
        P = T * k if meta.full else int(plan.offsets[-1].item())
        F1 = _fc1_rows(meta.act, f)
        # fp8 experts read only the input rows' codes: the permute writes them instead of bf16 rows.
        xp = K.permute(x, plan.pair_row, k, P) if fp8 is None else x.new_empty(0, h)
        hpre = x.new_empty(P, F1) if keep and mx4 is None else None
        # The fp8 and 4-bit paths keep only the activation's codes.
        act = x.new_empty(0 if fp8 is not None or mx4 is not None else P, f)
        y = x.new_empty(P, h) if mx4 is None else None
        q8, q4 = None, ()
        if isinstance(mx4, Mx4Experts):
            y = mx4_experts(xp, plan.offsets, mx4)
        elif mx4 is not None:
            y, hpre, q4 = _mx4_forward(meta, plan.offsets, xp, weights[:G], weights[G:2 * G], keep,
                                       any(ctx.needs_input_grad[i] for i in (2, 5, 6)))
            xp = x.new_empty(0, h)
        elif fp8 is not None:
            xq = fp8.permute(X, x, plan.pair_row, k, P)
            q8 = _fp8_forward(fp8, meta, plan.offsets, P, xq, fc1s, fc2s, hpre, y, wcast)
            q8["xq"] = xq
        elif P > 0:
            _fc1_fwd([xp] * G, plan.offsets, True, P, fc1s, f, meta.act, [hpre] * G if keep else None, [act] * G)
            K.expert_fc2_fwd([act] * G, plan.offsets, True, P, fc2s, [y] * G)
        if S and T > 0 and not shared_side:
            _fc1_fwd([x] * S, shared_off, False, T, sfc1s, fs, meta.act, shared_h, shared_a)
            K.expert_fc2_fwd(shared_a, shared_off, False, T, sfc2s, shared_y)
        if shared_side:
            main.wait_stream(_side_stream(x.device))
        out = K.combine(y, res, gates, topi, plan.pair_row, shared_y or [])
        ctx.mark_non_differentiable(plan.counts)
        outs = out, plan.counts
        if loss is not None:
            ctx.mark_non_differentiable(plan.counts, loss.counts)
            outs = *outs, loss.balance, loss.z, loss.counts
        if not keep:
            return outs
        ctx.meta = meta
        ctx.fp8 = (fp8, q8)
        codes, ctx.mx4 = _mx4_tensors(*q4)
        if loss is not None:
            ctx.set_materialize_grads(False)   # a loss that nothing came back for costs nothing
        ctx.norm_dtype = None if norm_b is None else norm_b.dtype
        ctx.dims = (T, h, P, G, S)
        ctx.save_for_backward(x, router_w, logits, topi, gates, plan.perm, plan.offsets, plan.pair_row, xp, hpre,
                              act, y, *(losses or LossTokens()),
                              *((None, None) if loss is None else (loss.counts, loss.tokens)), *codes,
                              *((shared_off, *shared_h, *shared_a) if S else ()), *weights,
                              *(() if mean is None else (res, norm_w, mean, rstd)))
        return outs

    @staticmethod
    @once_differentiable
    def backward(ctx, dout, _dcounts, d_balance=None, d_z=None, _dloss_counts=None):
        meta = ctx.meta
        T, h, P, G, S = ctx.dims
        (x, router_w, logits, topi, gates, perm, offsets, pair_row, xp, hpre, act, y, *ws) = ctx.saved_tensors
        n4 = 4 + 2 * sum(r is not None for r in ctx.mx4)
        # The LossTokens, what the losses' backward needs, 4-bit matrices, the shared experts' offsets and rows.
        over, (counts, tokens), codes, ws = ws[:2], ws[2:4], ws[4:n4], ws[n4:]
        shared_off = shared_h = shared_a = None
        if S:
            shared_off, shared_h, shared_a, ws = ws[0], ws[1:1 + S], ws[1 + S:1 + 2 * S], ws[1 + 2 * S:]
        normed = len(ws) > 2 * (G + S)
        if normed:
            *ws, res, norm_w, mean, rstd = ws
        fc1s, fc2s = ws[:G], ws[G:2 * G]
        sfc1s, sfc2s = ws[2 * G:2 * G + S], ws[2 * G + S:]
        f = meta.ffn
        fs = meta.shared_ffn or f
        dout = x.new_zeros(T, h) if dout is None else dout.contiguous()
        need_norm = ctx.needs_input_grad[5:7]
        need_x = ctx.needs_input_grad[2] or any(need_norm)
        main = torch.cuda.current_stream(x.device)
        sdw1 = [torch.empty_like(w) for w in sfc1s]
        sdw2 = [torch.empty_like(w) for w in sfc2s]
        shared_dx = []
        shared_side = S > 0 and T > 0 and _concurrent(h, _fc1_rows(meta.act, fs))
        if S and T > 0:
            dh = [x.new_empty(T, _fc1_rows(meta.act, fs)) for _ in range(S)]
            shared_dx = [x.new_empty(T, h) for _ in range(S)] if need_x else []
        if shared_side:
            # The shared experts' whole backward (it needs only dout) on the side stream, ahead of the
            # routed experts' weight gradients that expert_backward queues there.
            side = _side_stream(x.device)
            side.wait_stream(main)
            with torch.cuda.stream(side):
                K.expert_fc2_bwd([dout] * S, shared_a, shared_h, shared_off, False, T, list(sfc2s), meta.act, dh, sdw2)
                K.expert_fc1_bwd(dh, [x] * S, shared_off, False, T, list(sfc1s), fs, meta.act, shared_dx or None, sdw1)
        fp8, q8 = ctx.fp8
        if fp8 is None:
            dy, dgates = K.combine_bwd(dout, y, gates, pair_row, P)
        else:   # the fp8 products read only the codes of the rows' gradient
            dy, dgates = fp8.combine_bwd(DY, dout, y, gates, pair_row, P)
        dl = K.route_bwd(dgates, gates, logits, topi, meta.score, meta.normalize, meta.gate_scale)
        # What the losses send through all logits: one more row source of the token backward, and a term of the
        # router's gradient.
        loss_dx, loss_dwr = [], None
        if d_balance is not None or d_z is not None:
            dense = K.router_loss_bwd(d_balance, d_z, logits, topi, counts, tokens, meta.score, *over)
            rdx, loss_dwr = K.router_logits_bwd(dense, x, router_w, need_x, ctx.needs_input_grad[3])
            loss_dx = [rdx] if need_x else []
        dwr = None
        if ctx.needs_input_grad[3]:
            # The router's weight gradient needs only dl and x: on the side stream, beside the expert
            # products, instead of an HBM-bound pass that ends the backward on its own.
            side = _side_stream(x.device)
            side.wait_stream(main)
            with torch.cuda.stream(side):
                if meta.full:
                    rperm, roff = perm, offsets
                else:
                    full_plan = K.dispatch(topi, meta.num_experts)
                    rperm, roff = full_plan.perm, full_plan.offsets
                dwr = K.router_wgrad(dl, rperm, roff, x, meta.num_experts, router_w.dtype)
        # With every expert local each routed slot has a row, so fc1's input-gradient product can add the
        # router term to its rows (the token backward then sums it with the rows).
        fold = (need_x and meta.full and ctx.fp8[0] is None and not ctx.mx4 and P > 0 and x.dtype != torch.float64
                and router_w.dtype == torch.float32 and FOLD_ROUTER_TERM)
        if not ctx.mx4:
            dw2 = [torch.empty_like(w) for w in fc2s]
            dw1 = [torch.empty_like(w) for w in fc1s]
            dxp = x.new_empty(P, h) if need_x else None
        if ctx.mx4:
            dxp, dw1, dw2 = _mx4_backward(_mx4_again(codes, ctx.mx4), hpre, meta, offsets, dy, need_x)
            dw1, dw2 = dw1.unbind(), dw2.unbind()
        elif fp8 is not None:
            _fp8_backward(fp8, q8, meta, offsets, P, dy, hpre, dxp, dw1, dw2)
        elif P > 0:
            dhpre = x.new_empty(P, _fc1_rows(meta.act, f))
            expert_backward([dy] * G, [act] * G, [hpre] * G, offsets, True, P, fc1s, fc2s, f, meta.act, [dhpre] * G,
                            [xp] * G, [dxp] * G if need_x else None, dw1, dw2,
                            router=(router_w, meta.window[0], perm, dl) if fold else None)
        else:
            for w in (*dw1, *dw2):
                w.zero_()
        if S and T > 0 and not shared_side:
            expert_backward([dout] * S, shared_a, shared_h, shared_off, False, T, sfc1s, sfc2s, fs, meta.act, dh,
                            [x] * S, shared_dx or None, sdw1, sdw2)
        if shared_side:
            main.wait_stream(_side_stream(x.device))
        extra = [*shared_dx, *loss_dx]
        if len(extra) > K.MAX_SHARED:   # one row source more than the token backward reads
            extra[-2:] = [extra[-2] + extra[-1]]
        dx = K.token_bwd(dout, dxp, pair_row, None if fold else dl, topi, router_w, extra,
                         residual=not normed) if need_x else None
        dnw = dnb = None
        if normed and need_x:
            dx, dnw, dnb = K.layer_norm_bwd(dx, res, norm_w, mean, rstd, dres=dout, need_x=ctx.needs_input_grad[2],
                                            need_weight=need_norm[0], need_bias=need_norm[1], dtype=ctx.norm_dtype)
        if dwr is not None:
            main.wait_stream(_side_stream(x.device))
            dwr.record_stream(main)   # made on the side stream, used on the caller's
            if loss_dwr is not None:
                dwr += loss_dwr
        return (None, None, dx, dwr, None, dnw, dnb, *dw1, *dw2, *sdw1, *sdw2)


class _LayerNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, eps, x, weight, bias):
        y, mean, rstd = K.layer_norm(x, weight, bias, eps)
        ctx.norm_dtype = None if bias is None else bias.dtype
        ctx.save_for_backward(x, weight, mean, rstd)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, mean, rstd = ctx.saved_tensors
        _, need_x, need_w, need_b = ctx.needs_input_grad
        return None, *K.layer_norm_bwd(dy.contiguous(), x, weight, mean, rstd, need_x=need_x, need_weight=need_w,
                                       need_bias=need_b, dtype=ctx.norm_dtype)


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
               eps: float = 1e-5) -> torch.Tensor:
    """Layer norm over the last dimension of ``x`` (with autograd), in float32 (float64 for float64) whatever
    x's dtype.  ``weight`` and ``bias``: [h] in x's dtype, or float32 with bfloat16 rows, or None."""
    if x.dim() == 0 or x.shape[-1] == 0:
        raise K.KernelArgumentError("layer_norm needs at least one element a row")
    h = x.shape[-1]
    rows = x.reshape(-1, h).contiguous()
    return _LayerNormFn.apply(float(eps), rows, None if weight is None else weight.contiguous(),
                              None if bias is None else bias.contiguous()).view(x.shape)


class _RouterLossFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, score, logits, topi, mask, seq_offsets):
        loss = K.router_loss(logits, topi, score, mask, seq_offsets)
        ctx.score = score
        ctx.save_for_backward(logits, topi, mask, seq_offsets, loss.counts, loss.tokens)
        ctx.mark_non_differentiable(loss.counts)
        ctx.set_materialize_grads(False)
        return loss.balance, loss.z, loss.counts

    @staticmethod
    @once_differentiable
    def backward(ctx, d_balance, d_z, _dcounts):
        if d_balance is None and d_z is None:
            return None, None, None, None, None
        logits, topi, mask, seq_offsets, counts, tokens = ctx.saved_tensors
        d = K.router_loss_bwd(d_balance, d_z, logits, topi, counts, tokens, ctx.score, mask, seq_offsets)
        return None, d, None, None, None


def router_loss(logits: torch.Tensor, topi: torch.Tensor, score: str = "softmax", mask: torch.Tensor | None = None,
                seq_offsets: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Balance loss, z loss and per-expert counts of a router (differentiable in ``logits`` [T, E]); the choice
    ``topi`` [T, k] and the counts carry no gradient.  See ``kernels.router_loss`` for the formulas, ``mask`` [T]
    and ``seq_offsets`` [S + 1]; the counts are int32 [S, E]."""
    c = lambda t: None if t is None else t.contiguous()  # noqa: E731
    return _RouterLossFn.apply(score, logits.contiguous(), c(topi), c(mask), c(seq_offsets))


class _Mx4LinearFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, offsets, stacked, *weights):
        w = weights[0] if stacked else weights
        need_x, need_w = ctx.needs_input_grad[0], any(ctx.needs_input_grad[3:])
        # Each operand is read once for all the products it takes part in: x along its rows for y and along its
        # columns for the weights' gradients, the weights along their rows for y and their columns for dx.
        xr, xc = K.mx4_quantize(x, "both", offsets) if need_w else (K.mx4_quantize(x), None)
        wr, wc = K.mx4_quantize(w, "both") if need_x else (K.mx4_quantize(w), None)
        codes, ctx.mx4 = _mx4_tensors(xc, wc)
        ctx.stacked = stacked
        ctx.save_for_backward(offsets, *codes)
        return K.mx4_gemm(xr, wr, offsets)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        offsets, *codes = ctx.saved_tensors
        (xc, wc), stacked = _mx4_again(codes, ctx.mx4), ctx.stacked
        need_x, need_w = ctx.needs_input_grad[0], ctx.needs_input_grad[3:]
        along = "both" if need_x and any(need_w) else "rows" if need_x else "cols"
        q = K.mx4_quantize(dy.contiguous(), along, None if along == "rows" else offsets)
        dr, dc = q if along == "both" else (q, None) if need_x else (None, q)
        dx = K.mx4_gemm(dr, wc, offsets) if need_x else None
        if not any(need_w):
            return dx, None, None, *(None for _ in need_w)
        dw = K.mx4_wgrad(dc, xc, offsets)
        return dx, None, None, *((dw,) if stacked else (d if n else None for d, n in zip(dw.unbind(), need_w)))


def mx4_linear(x: torch.Tensor, weights, offsets: torch.Tensor) -> torch.Tensor:
    """y[r] = x[r] @ w[g]^T for the rows r of group g ([offsets[g], offsets[g + 1])), with every product, forward
    and backward, on operands in 4 bits with a power of two a block of 32 (with autograd: dx and dw are the
    products of the quantised gradient with the operands quantised along the other dimension).

    ``x`` [rows, K] and the ``weights`` (a list of [N, K], or stacked [G, N, K]) are bfloat16, K and N multiples of
    8, at most 64 groups.  Rows of no group are not computed: their y and dx are unspecified."""
    stacked = isinstance(weights, torch.Tensor)
    shape = weights.shape[1:] if stacked else weights[0].shape if len(weights) else ()
    if x.dim() != 2 or len(shape) != 2 or shape[1] != x.shape[1]:
        raise K.KernelArgumentError("mx4_linear needs x [rows, K] and weights [N, K]")
    if x.dtype != torch.bfloat16 or any(w.dtype != torch.bfloat16 for w in ((weights,) if stacked else weights)):
        raise K.KernelArgumentError("mx4_linear needs bfloat16 rows and weights")
    if shape[0] % 8 or shape[1] % 8:
        raise K.KernelArgumentError(f"mx4_linear needs sizes that are multiples of 8, got {tuple(shape)}")
    return _Mx4LinearFn.apply(x.contiguous(), offsets.contiguous(), stacked,
                              *((weights.contiguous(),) if stacked else (w.contiguous() for w in weights)))


class Mx4Experts:
    """Expert weights in 4 bits for serving: ``fc1s`` [ffn (SwiGLU: 2 ffn), hidden] and ``fc2s`` [hidden, ffn] of up
    to 64 experts (bfloat16 or float32 lists), quantised once along their rows; the originals are not kept."""

    def __init__(self, fc1s, fc2s, act: str = "swiglu"):
        if len(fc1s) != len(fc2s) or not len(fc1s):
            raise ValueError("need one fc1 and one fc2 weight per expert")
        h, f = fc2s[0].shape
        if tuple(fc1s[0].shape) != (_fc1_rows(act, f), h):
            raise ValueError(f"fc1 must be [{_fc1_rows(act, f)}, {h}], got {tuple(fc1s[0].shape)}")
        self.act, self.hidden, self.ffn = act, h, f
        self.fc1, self.fc2 = (K.mx4_quantize([w.detach().contiguous() for w in ws]) for ws in (fc1s, fc2s))

    def __len__(self) -> int:
        return self.fc1.shape[0]


def mx4_experts(x: torch.Tensor, offsets: torch.Tensor, experts: Mx4Experts) -> torch.Tensor:
    """fc2(act(fc1(x[r]))) of expert g for the bfloat16 rows r in [offsets[g], offsets[g + 1]), from weights in 4
    bits.  Without autograd: rows that need a gradient are refused.  Rows of no expert are not computed.

    The activations are rounded to bfloat16 between the two products, as the bfloat16 layer rounds them: the matrix
    instructions of the second take them so, and the error, 0.0023 of y's size against 0.0017 with them in float32,
    stays far below the 4 bits' own.  The sums of one product are ordered by its sizes and the mean rows of an expert,
    so a row served alone and in a larger batch may differ in its last bit."""
    if torch.is_grad_enabled() and x.requires_grad:
        raise ValueError("mx4_experts serves without autograd: call it under torch.no_grad() or on x.detach()")
    act = K.mx4_rows_gemm(x, experts.fc1, offsets, experts.act)
    return K.mx4_rows_gemm(act, experts.fc2, offsets)


class _ExpertChunksFn(torch.autograd.Function):
    """The receiving side of expert parallelism: the expert FFN over a source-major received buffer.

    resihp/runtime/moe.py:213-224 runs ``expert_ffn`` on every (source, expert) chunk of the received
    rows in order and returns the outputs in that order.  Here every local expert is one group of the
    grouped GEMMs over the chunks' expert-major order (the recv plan), and the products read and write
    received rows through the plan's row map: fc1 gathers its input rows, fc2 scatters its outputs
    back into the received order, and in the backward fc2's input-gradient product gathers the output
    gradient rows and fc1's scatters the input gradient.  Only the weight gradients need expert-major
    copies (of the inputs and of the output gradients); those gathers run on the side stream, beside
    the products.
    """

    @staticmethod
    def forward(ctx, act, f, rows, recv_counts, recv, *weights):
        G = len(weights) // 2
        fc1s, fc2s = K.group(weights[:G]), K.group(weights[G:])
        plan = K.recv_plan(recv_counts, rows)
        P, h = plan.rows, recv.shape[1]
        if recv.shape[0] != P:
            raise K.KernelArgumentError(f"the received buffer has {recv.shape[0]} rows, the counts {P}")
        F1 = _fc1_rows(act, f)
        xs = recv.new_empty(P, h)
        hpre = recv.new_empty(P, F1)
        a = recv.new_empty(P, f)
        y = recv.new_empty(P, h)
        if P > 0:
            main = torch.cuda.current_stream(recv.device)
            side = _side_stream(recv.device)
            side.wait_stream(main)
            with torch.cuda.stream(side):
                K.gather_rows(recv, plan.sort_row, out=xs)   # expert-major inputs, for the fc1 weight gradient
            K.expert_fc1_fwd_gather(recv, plan.sort_row, plan.offsets, P, fc1s, f, act, hpre, a)
            K.expert_fc2_fwd_scatter(a, plan.offsets, P, fc2s, y, plan.sort_row)
            main.wait_stream(side)
        ctx.act, ctx.f, ctx.P = act, f, P
        ctx.save_for_backward(plan.offsets, plan.sort_row, xs, hpre, a, *weights)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy_recv):
        offsets, sort_row, xs, hpre, a, *ws = ctx.saved_tensors
        G = len(ws) // 2
        fc1s, fc2s = ws[:G], ws[G:]
        act, f, P = ctx.act, ctx.f, ctx.P
        dw1 = [torch.empty_like(w) for w in fc1s]
        dw2 = [torch.empty_like(w) for w in fc2s]
        drecv = None
        need_x = ctx.needs_input_grad[4]
        grads = (*dw1, *dw2)
        if P > 0:
            fc1s, fc2s, dw1, dw2 = K.group(fc1s), K.group(fc2s), K.group(dw1), K.group(dw2)
            dy_recv = dy_recv.contiguous()
            h = xs.shape[1]
            dys = torch.empty_like(xs)          # expert-major output gradients, for the fc2 weight gradient
            dhpre = torch.empty_like(hpre)
            main = torch.cuda.current_stream(xs.device)
            if _concurrent(h, hpre.shape[1]):
                # Weight gradients (and the gather they need) on the side stream, input gradients here.
                side = _side_stream(xs.device)
                side.wait_stream(main)
                with torch.cuda.stream(side):
                    K.gather_rows(dy_recv, sort_row, out=dys)
                    K.expert_fc2_bwd([dys] * G, [a] * G, [hpre] * G, offsets, True, P, fc2s, act, None, dw2)
                K.expert_fc2_dgrad_gather(dy_recv, sort_row, offsets, P, fc2s, act, hpre, dhpre)
                side.wait_stream(main)
                with torch.cuda.stream(side):
                    K.expert_fc1_bwd([dhpre] * G, [xs] * G, offsets, True, P, fc1s, f, act, None, dw1)
                if need_x:
                    drecv = torch.empty_like(dy_recv)
                    K.expert_fc1_dgrad_scatter(dhpre, offsets, P, fc1s, f, act, drecv, sort_row)
                main.wait_stream(side)
            else:
                K.gather_rows(dy_recv, sort_row, out=dys)
                K.expert_fc2_dgrad_gather(dy_recv, sort_row, offsets, P, fc2s, act, hpre, dhpre)
                K.expert_fc2_bwd([dys] * G, [a] * G, [hpre] * G, offsets, True, P, fc2s, act, None, dw2)
                K.expert_fc1_bwd([dhpre] * G, [xs] * G, offsets, True, P, fc1s, f, act, None, dw1)
                if need_x:
                    drecv = torch.empty_like(dy_recv)
                    K.expert_fc1_dgrad_scatter(dhpre, offsets, P, fc1s, f, act, drecv, sort_row)
        else:
            for w in (*dw1, *dw2):
                w.zero_()
            drecv = torch.zeros_like(xs)
        return (None, None, None, None, drecv, *grads)


def expert_chunks(recv: torch.Tensor, recv_counts: torch.Tensor, fc1s: list[torch.Tensor],
                  fc2s: list[torch.Tensor], act: str = "swiglu", rows: int | None = None) -> torch.Tensor:
    """Expert outputs of a received buffer, in the received order (with autograd).

    ``recv`` holds the rows the all-to-all delivered, source-major: chunk (s, i) of
    ``recv_counts[s, i]`` rows for local expert i (``fc1s[i]``, ``fc2s[i]``), rows in the sender's
    (token, slot) order, as resihp/runtime/moe.py:199-212 builds and exchanges them.
    ``recv_counts`` is an int32 ``[n_src, L]`` device tensor; ``rows``, its sum, may be given to spare
    reading the counts on the host.
    """
    if len(fc1s) != len(fc2s) or recv_counts.dim() != 2 or recv_counts.shape[1] != len(fc1s):
        raise ValueError("need one fc1 and one fc2 weight per column of recv_counts")
    f = fc2s[0].shape[1]
    return _ExpertChunksFn.apply(act, f, rows, recv_counts.contiguous(), recv.contiguous(), *fc1s, *fc2s)


def moe_layer(meta: LayerMeta, x: torch.Tensor, router_w: torch.Tensor, bias: torch.Tensor | None,
              fc1s: list[torch.Tensor], fc2s: list[torch.Tensor], shared_fc1s: list[torch.Tensor] = (),
              shared_fc2s: list[torch.Tensor] = (), fp8: Fp8State | None = None,
              norm: Norm | None = None, mx4: "Mx4Experts | bool | None" = None,
              losses: LossTokens | None = None) -> tuple:
    """Layer output and the int32 per-expert counts (``counts[E]`` counts invalid ids).

    With ``losses`` (``LossTokens()``: all tokens in one sequence) a third value, the router's ``RouterLosses``:
    the balance and z loss, differentiable through the router's logits into x and ``router_w``, and their counts.

    With ``mx4`` = True the routed experts' products, forward and backward, run on operands in 4 bits with a power
    of two a block of 32 (bfloat16 tokens; hidden and ffn multiples of 8); with an ``Mx4Experts`` the layer serves
    from those weights (``fc1s`` and ``fc2s`` empty), without autograd.

    With ``norm`` the layer is a pre-norm block: it routes and computes on layer_norm(x), and x itself is
    the residual; the backward adds the residual's gradient inside the norm's.

    With ``fp8`` the routed experts run in fp8 (e4m3 weights and activations, e5m2 gradients) with the
    delayed scaling of that state; the caller ends each iteration with ``fp8.finish_iteration()``.
    """
    e0, e1 = meta.window
    if mx4 is False:
        mx4 = None
    if not (mx4 is None or mx4 is True or isinstance(mx4, Mx4Experts)):
        raise ValueError(f"mx4 must be True or an Mx4Experts, not {type(mx4).__name__}")
    if mx4 is not None and fp8 is not None:
        raise ValueError("experts run in fp8 or in 4 bits, not both")
    if fp8 is not None:
        if fp8.G != e1 - e0:
            raise ValueError(f"the fp8 state holds {fp8.G} experts, the window {e1 - e0}")
        if meta.num_shared:
            raise ValueError("fp8 experts: shared experts are not supported")
        h, F1 = fc1s[0].shape[1], _fc1_rows(meta.act, meta.ffn)
        if x.dtype != torch.bfloat16 or h % K.FP8_ALIGN or meta.ffn % K.FP8_ALIGN:
            raise ValueError(f"fp8 experts need bf16 tokens and hidden/ffn sizes that are multiples of {K.FP8_ALIGN}")
    serve = isinstance(mx4, Mx4Experts)
    if mx4 is not None:
        if x.dtype != torch.bfloat16 or x.shape[-1] % 8 or meta.ffn % 8 or e1 - e0 > K.C.MAX_GROUPS_PER_LAUNCH:
            raise ValueError("experts in 4 bits need bf16 tokens, hidden/ffn sizes that are multiples of 8 and at most "
                             f"{K.C.MAX_GROUPS_PER_LAUNCH} experts")
    if serve:
        if len(fc1s) or len(fc2s):
            raise ValueError("an Mx4Experts brings the experts' weights: fc1s and fc2s must be empty")
        if (len(mx4), mx4.hidden, mx4.ffn, mx4.act) != (e1 - e0, x.shape[-1], meta.ffn, meta.act):
            raise ValueError(f"the 4-bit weights are of {len(mx4)} experts, {mx4.hidden} x {mx4.ffn}, {mx4.act}; the layer "
                             f"needs {e1 - e0}, {x.shape[-1]} x {meta.ffn}, {meta.act}")
        if torch.is_grad_enabled() and any(t is not None and t.requires_grad
                                           for t in (x, router_w, *shared_fc1s, *shared_fc2s, *(norm or ())[:2])):
            raise ValueError("an Mx4Experts serves without autograd: call the layer under torch.no_grad()")
    elif len(fc1s) != e1 - e0 or len(fc2s) != e1 - e0:
        raise ValueError(f"need one fc1 and one fc2 weight per local expert ({e1 - e0})")
    if len(shared_fc1s) != meta.num_shared or len(shared_fc2s) != meta.num_shared:
        raise ValueError(f"need {meta.num_shared} shared expert weight pairs")
    norm_w, norm_b, eps = (None, None, None) if norm is None else norm
    if losses is not None:
        losses = LossTokens(*(None if t is None else t.contiguous() for t in losses))
    outs = _MoELayerFn.apply(meta, (fp8, mx4, losses, torch.is_grad_enabled(), None if eps is None else float(eps)),
                             x.contiguous(), router_w.contiguous(),
                             None if bias is None else bias.detach().contiguous(),
                             None if norm_w is None else norm_w.contiguous(),
                             None if norm_b is None else norm_b.contiguous(), *fc1s, *fc2s, *shared_fc1s, *shared_fc2s)
    return outs if losses is None else (*outs[:2], RouterLosses(*outs[2:]))
