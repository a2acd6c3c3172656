"""The router losses and the 4-bit operators as programs use them: captured and replayed with their backward, on
other streams, from views, with long and ragged shares, and with inputs changed between forward and backward."""

from __future__ import annotations

import pytest
import torch

from oracle import mx4_ref as R4
from resihp_megatron_amd import kernels as K
from resihp_megatron_amd import layer as L
from resihp_megatron_amd import moe

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16 = torch.bfloat16


def rand(*shape, seed=0, dtype=BF16, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g, dtype=torch.float64) * std).to(dtype).to(DEV)


def offsets_of(counts):
    return torch.tensor([0, *torch.tensor(counts).cumsum(0).tolist()], dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("which", ["linear", "loss"])
def test_forward_and_backward_captured_together(which):
    """Replays with new inputs, eager work between them; every replay's outputs and gradients are the eager ones."""
    if which == "linear":
        off, weight = offsets_of([70, 0, 130]), rand(200, 64, seed=90)
        inputs = lambda i: [rand(200, 96, seed=i), rand(3, 64, 96, seed=50 + i, std=0.1)]  # noqa: E731
        call = lambda x, w: (L.mx4_linear(x, w, off),)  # noqa: E731
    else:
        off, weight = offsets_of([50, 100]), torch.tensor(0.7, device=DEV)
        topi = rand(150, 24, seed=91).topk(3, 1).indices.int()
        inputs = lambda i: [rand(150, 24, seed=i, dtype=torch.float32)]  # noqa: E731
        call = lambda x: L.router_loss(x, topi, "sigmoid", None, off)[:2]  # noqa: E731

    def run(ts):
        outs = call(*ts)
        return [o.detach() for o in outs] + list(torch.autograd.grad(outs, ts, [weight] * len(outs)))

    held = [t.requires_grad_() for t in inputs(0)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(held)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run(held)
    for i in range(1, 4):
        fresh = inputs(i)
        with torch.no_grad():
            for a, b in zip(held, fresh):
                a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, run([t.requires_grad_() for t in fresh])))


def test_training_layer_captured():
    """The layer on 4-bit operands with its losses, forward and backward in one graph, replayed on new tokens."""
    cfg = moe.MoEConfig(hidden=64, ffn=48, num_experts=6, top_k=2, dtype=BF16, act="swiglu", num_shared=1, device=DEV)
    specs = moe.moe_specs(cfg)
    params = {k: moe.init_param(cfg, s).requires_grad_(s.trainable) for k, s in specs.items()}
    fc1s, fc2s, s1, s2 = moe._weights(cfg, params, range(6))
    dout, coef = rand(50, 64, seed=7), torch.tensor(0.3, device=DEV)

    def run(x):
        out, counts, losses = L.moe_layer(moe._layer_meta(cfg), x, params["router.weight"], None, fc1s, fc2s, s1, s2,
                                          mx4=True, losses=L.LossTokens())
        leaves = [x, params["router.weight"], *fc1s, *fc2s, *s1, *s2]
        outs = [out, losses.balance, losses.z]
        return [t.detach() for t in (*outs, counts)] + list(torch.autograd.grad(outs, leaves, [dout, coef, coef]))

    held = rand(50, 64, seed=1).requires_grad_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(held)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run(held)
    for i in range(3):
        fresh = rand(50, 64, seed=20 + i)
        with torch.no_grad():
            held.copy_(fresh)
        graph.replay()
        torch.cuda.synchronize()
        want = run(fresh.requires_grad_())
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("tokens", [0, 1])
@pytest.mark.parametrize("mx4", [None, True])
def test_layer_with_no_token_and_with_one(tokens, mx4):
    cfg = moe.MoEConfig(hidden=64, ffn=48, num_experts=6, top_k=2, dtype=BF16, act="swiglu", device=DEV)
    params = {k: moe.init_param(cfg, s).requires_grad_(s.trainable) for k, s in moe.moe_specs(cfg).items()}
    fc1s, fc2s, *_ = moe._weights(cfg, params, range(6))
    x = rand(tokens, 64, seed=3).requires_grad_()
    out, counts, losses = L.moe_layer(moe._layer_meta(cfg), x, params["router.weight"], None, fc1s, fc2s, mx4=mx4,
                                      losses=L.LossTokens())
    leaves = [x, params["router.weight"], *fc1s, *fc2s]
    got = torch.autograd.grad(out.float().sum() + losses.balance + losses.z, leaves)
    assert out.shape == got[0].shape == (tokens, 64) and counts.sum() == 2 * tokens
    chosen = (counts[:6] > 0).tolist()
    assert [bool(g.any()) for g in got[2:8]] == chosen and all(torch.isfinite(g).all() for g in got)
    if not tokens:
        assert losses.balance == 0 and losses.z == 0 and not got[1].any()


def test_two_graphs_in_turn():
    """Two captured losses and products replayed in turn keep their own workspaces."""
    xs = [rand(300, 16, seed=i, dtype=torch.float32) for i in (1, 2)]
    ts = [x.topk(2, 1).indices.int() for x in xs]
    ds = [rand(300, 16, seed=i, dtype=torch.float32) for i in (3, 4)]
    tokens, w = rand(300, 64, seed=5), rand(16, 64, seed=6, dtype=torch.float32)
    call = lambda i: (*L.router_loss(xs[i], ts[i]), *K.router_logits_bwd(ds[i], tokens, w))  # noqa: E731
    call(0)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for i in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(call(i))
    for i in (0, 1, 1, 0):
        graphs[i].replay()
        graphs[1 - i].replay()
        torch.cuda.synchronize()
        for j in range(2):
            assert all(torch.equal(a, b) for a, b in zip(outs[j], call(j)))


def test_on_another_stream():
    x, w, off = rand(65, 64, seed=1), rand(2, 32, 64, seed=2), offsets_of([30, 35])
    want = L.mx4_linear(x, w, off)
    experts = L.Mx4Experts(list(rand(2, 32, 64, seed=3)), list(rand(2, 64, 16, seed=4)))
    served = L.mx4_experts(x, off, experts)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got, got_served = L.mx4_linear(x, w, off), L.mx4_experts(x, off, experts)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want) and torch.equal(got_served, served)


def test_views_and_strides():
    """mx4_linear and router_loss take any strides and element-aligned views; the serving product refuses them by name."""
    base = rand(41, 130, seed=1)
    x, w, off = base[1:, 1:97], rand(96, 2, 64, seed=2).permute(1, 2, 0), offsets_of([17, 23])
    assert torch.equal(L.mx4_linear(x, w, off), L.mx4_linear(x.clone(), w.contiguous(), off))
    logits = rand(9, 30, seed=3, dtype=torch.float32)[:, 1:22]
    topi = torch.stack([logits.topk(4, 1).indices.int()] * 2, 2)[:, ::2, 0]
    mask = torch.arange(18, device=DEV)[::2] % 4 == 0
    a, b = L.router_loss(logits, topi, mask=mask), L.router_loss(logits.clone(), topi.clone(), mask=mask.clone())
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    with pytest.raises(RuntimeError, match="contiguous"):
        K.mx4_rows_gemm(base[:, :96], K.mx4_quantize(w.contiguous()), offsets_of([41, 0]))


def test_inputs_changed_between_forward_and_backward():
    """Operands in 4 bits are copies, so x and the weights may change; offsets, logits and masks may not, and say so."""
    x, w, off = rand(40, 64, seed=1).requires_grad_(), rand(1, 32, 64, seed=2).requires_grad_(), offsets_of([40])
    dy = rand(40, 32, seed=3)
    want = torch.autograd.grad(L.mx4_linear(x, w, off), (x, w), dy)
    y = L.mx4_linear(x, w, off)
    with torch.no_grad():
        x.add_(1.0)
        w.mul_(2.0)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(y, (x, w), dy), want))
    y = L.mx4_linear(x, w, off)
    off.add_(0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, x, dy)
    logits, mask = rand(8, 4, seed=4, dtype=torch.float32).requires_grad_(), torch.ones(8, dtype=torch.bool, device=DEV)
    loss = L.router_loss(logits, torch.zeros(8, 1, dtype=torch.int32, device=DEV), mask=mask)
    mask[2] = False
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss[0].backward()


def test_backward_frees_what_the_forward_kept():
    """Once the backward has run, the outputs alone hold no 4-bit operands, and a second backward says why it cannot."""
    x, w = rand(4096, 1024, seed=1).requires_grad_(), rand(2, 1024, 1024, seed=2).requires_grad_()
    off = offsets_of([2000, 2096])
    y = L.mx4_linear(x, w, off)
    kept = torch.cuda.memory_allocated()
    torch.autograd.grad(y, (x, w), torch.ones_like(y))
    assert torch.cuda.memory_allocated() <= kept - 4096 * 1024 // 2 - 2 * 1024 * 1024 // 2   # x's and the weights' codes
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(y, x, torch.ones_like(y))


def test_second_derivatives_are_refused():
    x, w = rand(16, 32, seed=1).requires_grad_(), rand(1, 32, 32, seed=2).requires_grad_()
    dx, = torch.autograd.grad(L.mx4_linear(x, w, offsets_of([16])).float().pow(2).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        dx.sum().backward()


def test_rows_of_no_group_and_offsets_that_skip():
    """Groups that leave rows out before, between and behind: those rows' outputs stay, the groups' are their own."""
    x, w = rand(300, 64, seed=1), rand(3, 32, 64, seed=2)
    off = torch.tensor([10, 10, 140, 260], dtype=torch.int32, device=DEV)   # rows 0 to 9 and 260 on of no group
    y = torch.full((300, 32), 3.0, dtype=BF16, device=DEV)
    K.mx4_gemm(K.mx4_quantize(x), K.mx4_quantize(w), off, y)
    z = torch.full_like(y, 3.0)
    K.mx4_rows_gemm(x, K.mx4_quantize(w), off, out=z)
    assert (y[:10] == 3).all() and (y[260:] == 3).all() and (z[:10] == 3).all() and (z[260:] == 3).all()
    xq, wq, xv = R4.round4(x.cpu()), [R4.round4(t) for t in w.cpu()], x.cpu().double()
    for lo, hi, g in ((10, 140, 1), (140, 260, 2)):
        for got, rows in ((y, xq), (z, xv)):
            want, mag = rows[lo:hi] @ wq[g].t(), rows[lo:hi].abs() @ wq[g].abs().t()
            sums = 96 * 2.0 ** -23 * mag
            assert ((got[lo:hi].cpu().double() - want).abs() <= sums + (want.abs() + sums) * 2.0 ** -8).all()
    dw = K.mx4_wgrad(K.mx4_quantize(z, "cols", off), K.mx4_quantize(x, "cols", off), off)
    assert (dw[0] == 0).all()
    for lo, hi, g in ((10, 140, 1), (140, 260, 2)):
        a, b = R4.round4(z[lo:hi].cpu().t()), R4.round4(x[lo:hi].cpu().t())
        want, mag = a @ b.t(), a.abs() @ b.abs().t()
        sums = 160 * 2.0 ** -23 * mag
        assert ((dw[g].cpu().double() - want).abs() <= sums + (want.abs() + sums) * 2.0 ** -8).all()


@pytest.mark.parametrize("counts", [[97, 96], [30, 0, 259], [96, 96], [1030, 1020], [2100, 1, 1000]])
def test_products_on_both_sides_of_the_group_sizes(counts):
    """Up to 96 rows a group (weights' gradients: 1024) take another kernel than more; each against float64."""
    rows, G, N, k = sum(counts), len(counts), 264, 200
    x, dy, w, off = rand(rows, k, seed=1), rand(rows, N, seed=2), rand(G, N, k, seed=3, std=0.1), offsets_of(counts)
    y = K.mx4_gemm(K.mx4_quantize(x), K.mx4_quantize(w), off)
    dw = K.mx4_wgrad(K.mx4_quantize(dy, "cols", off), K.mx4_quantize(x, "cols", off), off)
    act, hpre = K.mx4_gemm_act(K.mx4_quantize(x), K.mx4_quantize(w), off, "gelu")
    assert torch.equal(hpre, y)
    at = 0
    for g, n in enumerate(counts):
        rows_of, xt, dyt = x[at:at + n].cpu(), x[at:at + n].cpu().t(), dy[at:at + n].cpu().t()
        pairs = [(y[at:at + n], R4.round4(rows_of), R4.round4(w[g].cpu()))] if n else []
        pairs.append((dw[g], R4.round4(dyt), R4.round4(xt)) if n else (dw[g], torch.zeros(N, 1), torch.zeros(k, 1)))
        for got, a, b in pairs:
            a, b = a.double(), b.double()
            want, mag = a @ b.t(), a.abs() @ b.abs().t()
            sums = (a.shape[1] + 32) * 2.0 ** -23 * mag
            assert ((got.cpu().double() - want).abs() <= sums + (want.abs() + sums) * 2.0 ** -8).all(), (g, n)
        at += n


@pytest.mark.parametrize("counts", [[1, 0], [2, 3], [40, 7], [70, 64]])
@pytest.mark.parametrize("k", [8184, 8192, 8200, 8328])
def test_serving_products_with_long_reductions(counts, k):
    """From 8192 places on a reduction is shared by more waves; one place in seven of a row is not zero."""
    x, w, off = rand(sum(counts), k, seed=1), rand(2, 48, k, seed=2, std=0.1), offsets_of(counts)
    x[:, torch.arange(k, device=DEV) % 7 != 3] = 0
    got, at = K.mx4_rows_gemm(x, K.mx4_quantize(w), off), 0
    for g, n in enumerate(counts):
        a, b = x[at:at + n].cpu().double(), R4.round4(w[g].cpu())
        want, mag = a @ b.t(), a.abs() @ b.abs().t()
        sums = (k + 32) * 2.0 ** -23 * mag
        assert ((got[at:at + n].cpu().double() - want).abs() <= sums + (want.abs() + sums) * 2.0 ** -8).all()
        at += n


def test_same_expert_twice_counts_twice():
    logits = rand(6, 5, seed=1, dtype=torch.float64)
    topi = torch.full((6, 2), 3, dtype=torch.int32, device=DEV)
    balance, _, counts = L.router_loss(logits, topi)
    assert counts.tolist() == [[0, 0, 0, 12, 0]]
    want = 5 / (2 * 36) * 12 * logits.softmax(1)[:, 3].sum()
    assert abs(balance - want) <= 64 * 2.0 ** -53 * want


@pytest.mark.parametrize("bits", ["1", 4, object()])
def test_layer_refuses_other_values_of_mx4(bits):
    cfg = moe.MoEConfig(hidden=32, ffn=32, num_experts=2, top_k=1, dtype=BF16)
    with pytest.raises(ValueError, match="mx4 must be True or an Mx4Experts"):
        L.moe_layer(moe._layer_meta(cfg), rand(4, 32), rand(2, 32, dtype=torch.float32), None, [], [], mx4=bits)


def test_served_experts_refuse_rows_that_need_a_gradient():
    """There is no backward through weights in 4 bits that are only served: the call says so instead of cutting the graph."""
    experts = L.Mx4Experts(list(rand(2, 32, 64, seed=3)), list(rand(2, 64, 16, seed=4)))
    x, off = rand(20, 64, seed=5), offsets_of([7, 13])
    want = L.mx4_experts(x, off, experts)
    leaf = x.clone().requires_grad_(True)
    for rows in (leaf, leaf * 1):
        with pytest.raises(ValueError, match="without autograd"):
            L.mx4_experts(rows, off, experts)
        with torch.no_grad():
            assert torch.equal(L.mx4_experts(rows, off, experts), want)
        assert torch.equal(L.mx4_experts(rows.detach(), off, experts), want)
