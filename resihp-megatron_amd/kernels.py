"""Torch-facing wrappers of the gfx950 kernels.

Each function checks shapes, dtypes and devices (the C ABI sees raw pointers
only), allocates its outputs and workspace through PyTorch's caching
allocator, and enqueues the kernels on the current HIP stream of the tensors'
device.  Nothing here computes on the CPU; every entry point goes through
``libresihp_moe.so``.
"""

from __future__ import annotations

import array
import collections
import ctypes
import operator

from dataclasses import dataclass

import torch

from . import _capi as C

_DT = {torch.float64: C.F64, torch.float32: C.F32, torch.bfloat16: C.BF16}

# Optional per-entry-point timer: an object with start(name, stream) / stop(name, stream)
# that records HIP events around every C call (None = no events).
_timer = None


def set_timer(timer) -> None:
    """Installs (or with None removes) the event timer used around each C call."""
    global _timer
    _timer = timer


def _call(name: str, dev: torch.device, *args) -> None:
    """Calls entry point ``name`` with ``args`` and the current stream of ``dev``."""
    if _timer is None and torch.cuda.current_device() == dev.index:
        # The usual case, without the objects that the device guard and the stream wrapper make (about
        # 6 us a call, of some twenty calls a layer pass).
        C.call(name, *args, torch._C._cuda_getCurrentRawStream(dev.index))
        return
    stream = torch.cuda.current_stream(dev)
    with torch.cuda.device(dev):
        if _timer is not None:
            _timer.start(name, stream)
        C.call(name, *args, stream.cuda_stream)
        if _timer is not None:
            _timer.stop(name, stream)


def dtype_code(t: torch.Tensor) -> int:
    try:
        return _DT[t.dtype]
    except KeyError:
        raise KernelArgumentError(f"unsupported dtype {t.dtype}") from None


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


class Group:
    """The tensors of a list of groups, found to be of one 2-D shape, dtype and HIP device and contiguous,
    with their pointer array: what a call checks and converts per tensor, done once for the calls that one
    forward or backward makes with them.  Not kept beyond it."""

    __slots__ = ("ts", "arr", "dtype", "shape", "device")

    def __init__(self, ts):
        self.ts = ts
        self.arr = C.ptr_array([t.data_ptr() for t in ts])
        self.dtype, self.shape, self.device = ts[0].dtype, ts[0].shape, ts[0].device

    def __len__(self) -> int:
        return len(self.ts)

    def __getitem__(self, i):
        return self.ts[i]


def group(ts):
    """``ts`` as a Group where its tensors are alike (see there), else as it is, for the calls to judge."""
    ts = list(ts)
    if not ts:
        return ts
    t0 = ts[0]
    dt, shape, dev = t0.dtype, t0.shape, t0.get_device()
    if dev < 0 or len(shape) != 2:
        return ts
    for t in ts:
        if t.dtype is not dt or t.get_device() != dev or not t.is_contiguous() or t.shape != shape:
            return ts
    return Group(ts)


def _distinct(ts):
    """The tensors of a list that differ from the one before: one, where every group shares a buffer."""
    out, last = [], None
    for t in ts:
        if t is not last:
            out.append(t)
            last = t
    return out


def _each(ts):
    """The groups of a product for ``_need_cuda``: those of a stacked tensor one by one."""
    return ts.unbind() if isinstance(ts, torch.Tensor) else ts


def _need_cuda(*ts) -> torch.device:
    """The HIP device of tensors, sequences of tensors, Groups and Nones."""
    flat = []
    for t in ts:
        if isinstance(t, Group):
            flat.append(t.ts[0])   # the others are alike
        elif t is None or isinstance(t, torch.Tensor):
            flat.append(t)
        else:
            flat.extend(_distinct(t))
    dev = None
    for t in flat:
        if t is None:
            continue
        if not t.is_cuda:
            raise RuntimeError("MoE kernels need tensors on a HIP device (cuda:N); got a CPU tensor")
        if not t.is_contiguous():
            raise RuntimeError("MoE kernels need contiguous tensors")
        if dev is None:
            dev = t.device
        elif t.device != dev:
            raise RuntimeError(f"tensors on different devices: {dev} and {t.device}")
    return dev


def need_device(*ts: torch.Tensor | None) -> torch.device:
    """The HIP device all of ``ts`` are on; raises RuntimeError for host tensors or mixed devices."""
    return _need_cuda(*ts)


class KernelArgumentError(RuntimeError):
    """Arguments the kernels cannot take.  A RuntimeError, like every failure of the layer, so the
    resilient trainer (resihp/train/resilient_loop.py:28) treats it as it treats the reference's."""


def _expect(cond: bool, msg: str) -> None:
    if not cond:
        raise KernelArgumentError(msg)


def _rows_of(t: torch.Tensor, name: str, cols: int, dtype: torch.dtype) -> int:
    _expect(t.dim() == 2 and t.shape[1] == cols, f"{name} must be [rows, {cols}], got {tuple(t.shape)}")
    _expect(t.dtype == dtype, f"{name} has dtype {t.dtype}, expected {dtype}")
    return t.shape[0]


def _index(t: torch.Tensor, name: str, shape: tuple[int, ...]) -> None:
    _expect(t.dtype == torch.int32 and tuple(t.shape) == shape, f"{name} must be int32 {shape}")


def score_code(score: str) -> int:
    return {"softmax": C.SCORE_SOFTMAX, "sigmoid": C.SCORE_SIGMOID}[score]


def act_code(act: str) -> int:
    return {"gelu": C.ACT_GELU, "swiglu": C.ACT_SWIGLU}[act]


# ----------------------------------------------------------------------------- routing


def route(x: torch.Tensor, router_w: torch.Tensor, bias: torch.Tensor | None, k: int, score: str = "softmax",
          normalize: bool = True, scale: float = 1.0) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Router logits [T,E], top-k expert ids [T,k] (int32) and gates [T,k] (router dtype)."""
    dev = _need_cuda(x, router_w, bias)
    T, h = x.shape
    E = router_w.shape[0]
    _rows_of(router_w, "router_w", h, router_w.dtype)
    _expect(bias is None or (bias.dtype == router_w.dtype and tuple(bias.shape) == (E,)),
            "bias must match the router dtype and have one entry per expert")
    logits = torch.empty(T, E, dtype=router_w.dtype, device=dev)
    topi = torch.empty(T, k, dtype=torch.int32, device=dev)
    gates = torch.empty(T, k, dtype=router_w.dtype, device=dev)
    _call("rhp_route", dev, _ptr(x), dtype_code(x), _ptr(router_w), dtype_code(router_w), _ptr(bias), T, h, E, k,
          score_code(score), int(normalize), float(scale), _ptr(logits), _ptr(topi), _ptr(gates))
    return logits, topi, gates


@dataclass
class DispatchPlan:
    """Dispatch plan of the local experts [e0, e1) (all int32 device tensors)."""

    counts: torch.Tensor       # [E + 1]; counts[E] = ids outside [0, E)
    offsets: torch.Tensor      # [L + 1]
    src_counts: torch.Tensor   # [n_src, L]
    perm: torch.Tensor         # [T * k]; rows [0, offsets[L]) valid
    pair_row: torch.Tensor     # [T * k]; -1 for pairs of other experts
    e0: int
    e1: int


def dispatch(topi: torch.Tensor, E: int, e0: int = 0, e1: int | None = None, n_src: int = 1) -> DispatchPlan:
    dev = _need_cuda(topi)
    _expect(topi.dtype == torch.int32 and topi.dim() == 2, "topi must be int32 [T, k]")
    e1 = E if e1 is None else e1
    T, k = topi.shape
    L = e1 - e0
    counts = torch.empty(E + 1, dtype=torch.int32, device=dev)
    offsets = torch.empty(L + 1, dtype=torch.int32, device=dev)
    src_counts = torch.empty(n_src, L, dtype=torch.int32, device=dev)
    perm = torch.empty(max(1, T * k), dtype=torch.int32, device=dev)
    pair_row = torch.empty(max(1, T * k), dtype=torch.int32, device=dev)
    ws_bytes = C.lib().rhp_dispatch_workspace_bytes(T, k, E, n_src)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
    _call("rhp_dispatch", dev, _ptr(topi), T, k, E, e0, e1, n_src, _ptr(counts), _ptr(offsets), _ptr(src_counts),
          _ptr(perm), _ptr(pair_row), _ptr(ws), ws_bytes)
    return DispatchPlan(counts, offsets, src_counts, perm[: T * k], pair_row[: T * k], e0, e1)


def update_expert_bias(bias: torch.Tensor, counts: torch.Tensor, rate: float) -> None:
    """bias += rate * sign(mean(counts) - counts), in place (counts: int32 [E])."""
    dev = _need_cuda(bias, counts)
    _expect(counts.dtype == torch.int32 and counts.numel() >= bias.numel(), "counts must be int32, one per expert")
    _call("rhp_update_expert_bias", dev, _ptr(bias), dtype_code(bias), _ptr(counts), bias.shape[0], float(rate))


def route_bwd(dgates: torch.Tensor, gates: torch.Tensor, logits: torch.Tensor, topi: torch.Tensor, score: str,
              normalize: bool, scale: float) -> torch.Tensor:
    """Gradient of the selected logits [T,k] from the gate gradient."""
    dev = _need_cuda(dgates, gates, logits, topi)
    T, k = topi.shape
    _index(topi, "topi", (T, k))
    _expect(logits.shape[0] == T, "logits must have one row per token")
    for name, t in (("dgates", dgates), ("gates", gates)):
        _expect(t.dtype == logits.dtype and tuple(t.shape) == (T, k), f"{name} must be {logits.dtype} [T, k]")
    dl = torch.empty(T, k, dtype=logits.dtype, device=dev)
    _call("rhp_route_bwd", dev, _ptr(dgates), _ptr(gates), _ptr(logits), _ptr(topi), dtype_code(logits), T,
          logits.shape[1], k, score_code(score), int(normalize), float(scale), _ptr(dl))
    return dl


# ----------------------------------------------------------------------------- rows


def permute(x: torch.Tensor, pair_row: torch.Tensor, k: int, rows: int) -> torch.Tensor:
    """Expert-contiguous copy of the token rows: out[pair_row[t*k+j]] = x[t]."""
    dev = _need_cuda(x, pair_row)
    T, h = x.shape
    _index(pair_row, "pair_row", (T * k,))
    xp = torch.empty(rows, h, dtype=x.dtype, device=dev)
    if rows == 0:
        return xp
    _call("rhp_permute", dev, _ptr(x), dtype_code(x), T, h, k, _ptr(pair_row), _ptr(xp))
    return xp


def combine(y: torch.Tensor, x: torch.Tensor, gates: torch.Tensor, topi: torch.Tensor, pair_row: torch.Tensor,
            shared: list[torch.Tensor] = ()) -> torch.Tensor:
    """out = x + sum of gate-weighted expert rows (ascending expert id) + shared expert rows."""
    dev = _need_cuda(y, x, gates, topi, pair_row, *shared)
    T, h = x.shape
    k = topi.shape[1]
    _index(topi, "topi", (T, k))
    _index(pair_row, "pair_row", (T * k,))
    _rows_of(y, "y", h, x.dtype)
    _expect(tuple(gates.shape) == (T, k), "gates must be [T, k]")
    for i, t in enumerate(shared):
        _expect(_rows_of(t, f"shared[{i}]", h, x.dtype) == T, "shared outputs need one row per token")
    out = torch.empty_like(x)
    arr = C.ptr_array([s.data_ptr() for s in shared])
    _call("rhp_combine", dev, _ptr(y), _ptr(x), _ptr(gates), dtype_code(gates), _ptr(topi), _ptr(pair_row), arr,
          len(shared), dtype_code(x), T, h, k, _ptr(out))
    return out


def combine_bwd(dout: torch.Tensor, y: torch.Tensor, gates: torch.Tensor, pair_row: torch.Tensor,
                rows: int) -> tuple[torch.Tensor, torch.Tensor]:
    """(dy [rows,h] = gate * dout row, dgates [T,k] = <dout, y row>)."""
    dev = _need_cuda(dout, y, gates, pair_row)
    T, h = dout.shape
    k = gates.shape[1]
    _index(pair_row, "pair_row", (T * k,))
    _expect(_rows_of(y, "y", h, dout.dtype) >= rows, "y has fewer rows than the plan")
    dy = torch.empty(rows, h, dtype=dout.dtype, device=dev)
    dgates = torch.empty_like(gates)
    _call("rhp_combine_bwd", dev, _ptr(dout), _ptr(y), _ptr(gates), dtype_code(gates), _ptr(pair_row),
          dtype_code(dout), T, h, k, _ptr(dy), _ptr(dgates))
    return dy, dgates


def token_bwd(dout: torch.Tensor, dxp: torch.Tensor | None, pair_row: torch.Tensor, dl: torch.Tensor | None,
              topi: torch.Tensor, router_w: torch.Tensor, shared_dx: list[torch.Tensor] = (),
              residual: bool = True) -> torch.Tensor:
    """dx = dout + sum of the token's permuted-row gradients + router input gradient + shared gradients;
    without ``residual`` the term dout is left out (a residual that does not pass through here)."""
    dev = _need_cuda(dout, dxp, pair_row, dl, topi, router_w, *shared_dx)
    T, h = dout.shape
    k = topi.shape[1]
    _index(topi, "topi", (T, k))
    _index(pair_row, "pair_row", (T * k,))
    _rows_of(router_w, "router_w", h, router_w.dtype)
    if dxp is not None:
        _rows_of(dxp, "dxp", h, dout.dtype)
    _expect(dl is None or (dl.dtype == router_w.dtype and tuple(dl.shape) == (T, k)), "dl must be router dtype [T,k]")
    for i, t in enumerate(shared_dx):
        _expect(_rows_of(t, f"shared_dx[{i}]", h, dout.dtype) == T, "shared gradients need one row per token")
    dx = torch.empty_like(dout)
    arr = C.ptr_array([s.data_ptr() for s in shared_dx])
    args = (_ptr(dxp), _ptr(pair_row), _ptr(dl), _ptr(topi), _ptr(router_w), dtype_code(router_w), arr, len(shared_dx),
            dtype_code(dout), T, h, router_w.shape[0], k, _ptr(dx))
    if residual:
        _call("rhp_token_bwd", dev, _ptr(dout), *args)
    else:
        _call("rhp_token_bwd_no_residual", dev, *args)
    return dx


def router_wgrad(dl: torch.Tensor, perm: torch.Tensor, offsets: torch.Tensor, x: torch.Tensor, E: int,
                 r_dtype: torch.dtype) -> torch.Tensor:
    """dW[e] = sum over pairs routed to e of dl * x[token]; perm/offsets from a plan over all E experts."""
    dev = _need_cuda(dl, perm, offsets, x)
    T, h = x.shape
    k = dl.shape[1]
    _expect(dl.dtype == r_dtype and tuple(dl.shape) == (T, k), "dl must be router dtype [T, k]")
    _index(offsets, "offsets", (E + 1,))
    _expect(perm.dtype == torch.int32 and perm.numel() == T * k, "perm must be int32 [T * k] over all experts")
    dw = torch.empty(E, h, dtype=r_dtype, device=dev)
    rc = _DT[r_dtype]
    ws_bytes = C.lib().rhp_router_wgrad_workspace_bytes(T, h, E, k, rc)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
    _call("rhp_router_wgrad", dev, _ptr(dl), _ptr(perm), _ptr(offsets), _ptr(x), dtype_code(x), rc, T, h, E, k,
          _ptr(dw), _ptr(ws), ws_bytes)
    return dw


# ----------------------------------------------------------------------------- sending side


@dataclass
class SendTables:
    """One period of every expert's holder picks for one EP group (int32 device tensors), as
    ``placement.send_tables`` lays them out."""

    pick_off: torch.Tensor     # [E + 1]
    pick_dev: torch.Tensor     # [pick_off[E]]: device (index in the group's send order) of each pick
    pick_rank: torch.Tensor    # [pick_off[E]]: picks of the same device earlier in the period
    period_cnt: torch.Tensor   # [E * n_dev]: picks of each device in expert e's period
    n_dev: int

    @classmethod
    def from_lists(cls, off, dev, rank, cnt, n_dev: int, device) -> "SendTables":
        mk = lambda v: torch.tensor(v if len(v) else [0], dtype=torch.int32, device=device)  # noqa: E731
        return cls(mk(off), mk(dev), mk(rank), mk(cnt), n_dev)


@dataclass
class SendPlan:
    """A source's send order for its EP group (all int32 device tensors)."""

    counts: torch.Tensor       # [n_dev, E]: pairs of expert e sent to device d (moe.py:199-207)
    offsets: torch.Tensor      # [n_dev * E + 1]: chunk starts in send order
    perm: torch.Tensor         # [T * k]: send row -> flat pair t*k + j (rows < offsets[-1] valid)
    row: torch.Tensor          # [T * k]: flat pair -> send row, -1 for ids outside [0, E)
    dispatch: DispatchPlan     # the expert-major plan it was built from (window [0, E))


def ep_send_plan(topi: torch.Tensor, E: int, tables: SendTables) -> SendPlan:
    """Send order of one source's routed pairs over its EP group (resihp/runtime/moe.py:193-211)."""
    dev = _need_cuda(topi, tables.pick_off)
    _expect(topi.dtype == torch.int32 and topi.dim() == 2, "topi must be int32 [T, k]")
    _expect(tables.pick_off.numel() == E + 1 and tables.period_cnt.numel() == E * tables.n_dev,
            f"send tables must cover {E} experts and {tables.n_dev} devices")
    T, k = topi.shape
    plan = dispatch(topi, E)
    n = tables.n_dev
    counts = torch.empty(n, E, dtype=torch.int32, device=dev)
    offsets = torch.empty(n * E + 1, dtype=torch.int32, device=dev)
    perm = torch.empty(max(1, T * k), dtype=torch.int32, device=dev)
    row = torch.empty(max(1, T * k), dtype=torch.int32, device=dev)
    _call("rhp_ep_send_plan", dev, _ptr(topi), T, k, E, n, _ptr(plan.counts), _ptr(plan.offsets),
          _ptr(plan.pair_row), _ptr(tables.pick_off), _ptr(tables.pick_dev), _ptr(tables.pick_rank),
          _ptr(tables.period_cnt), _ptr(counts), _ptr(offsets), _ptr(perm), _ptr(row))
    return SendPlan(counts, offsets, perm[: T * k], row[: T * k], plan)


# ----------------------------------------------------------------------------- received rows


@dataclass
class RecvPlan:
    """Expert-major grouping of a source-major received buffer (all int32 device tensors)."""

    offsets: torch.Tensor      # [L + 1] group offsets of the expert-major rows
    sort_row: torch.Tensor     # [rows]: expert-major row r holds received row sort_row[r]
    unsort_row: torch.Tensor   # [rows]: received row q is expert-major row unsort_row[q]
    rows: int


def recv_plan(recv_counts: torch.Tensor, rows: int | None = None) -> RecvPlan:
    """Plan of a received buffer from its per-(source, local expert) counts ``[n_src, L]``.

    ``rows`` is the counts' sum.  Without it the counts are read on the host (as the reference reads
    its split sizes, resihp/runtime/moe.py:210-211) and checked; a caller that already holds the sum
    passes it and saves the synchronisation.  With the true sum the two row maps are exact inverses.
    """
    dev = _need_cuda(recv_counts)
    _expect(recv_counts.dtype == torch.int32 and recv_counts.dim() == 2, "recv_counts must be int32 [n_src, L]")
    n_src, L = recv_counts.shape
    if rows is None:
        _expect(bool((recv_counts >= 0).all()), "recv_counts must be non-negative")
        rows = int(recv_counts.sum().item())
    offsets = torch.empty(L + 1, dtype=torch.int32, device=dev)
    sort_row = torch.empty(max(1, rows), dtype=torch.int32, device=dev)
    unsort_row = torch.empty(max(1, rows), dtype=torch.int32, device=dev)
    _call("rhp_recv_plan", dev, _ptr(recv_counts), n_src, L, rows, _ptr(offsets), _ptr(sort_row), _ptr(unsort_row))
    return RecvPlan(offsets, sort_row[:rows], unsort_row[:rows], rows)


def gather_rows(src: torch.Tensor, idx: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """out[r] = src[idx[r]] (whole rows; an index outside src's rows gives a zero row)."""
    dev = _need_cuda(src, idx, out)
    _expect(src.dim() == 2 and idx.dtype == torch.int32 and idx.dim() == 1, "src must be [rows, h], idx int32 [n]")
    rows, h = idx.numel(), src.shape[1]
    if out is None:
        out = torch.empty(rows, h, dtype=src.dtype, device=dev)
    _expect(out.dtype == src.dtype and tuple(out.shape) == (rows, h), f"out must be {src.dtype} [{rows}, {h}]")
    if rows:
        _call("rhp_gather_rows", dev, _ptr(src), dtype_code(src), src.shape[0], h, _ptr(idx), rows, _ptr(out))
    return out


# ----------------------------------------------------------------------------- expert GEMMs


def _arr(ts) -> object:
    if isinstance(ts, Group):
        return ts.arr
    if len(ts) > 1 and all(t is ts[0] for t in ts):
        return C.ptr_array([ts[0].data_ptr()] * len(ts))
    return C.ptr_array([t.data_ptr() for t in ts])


def _check_groups(what: str, ts: list[torch.Tensor], G: int, dtype: torch.dtype, cols: int,
                  rows: int | None = None, exact_shape: tuple[int, int] | None = None) -> None:
    """Every group tensor must have the kernel's dtype and shape; the kernels cannot see either."""
    if len(ts) != G:
        raise KernelArgumentError(f"{what}: expected {G} tensors, got {len(ts)}")
    last = None
    for i, t in enumerate(ts.ts[:1] if isinstance(ts, Group) else ts):
        if t is last:
            continue
        last, shape = t, t.shape
        if (t.dtype is dtype and len(shape) == 2 and shape[1] == cols
                and (exact_shape is None or shape[0] == exact_shape[0]) and (rows is None or shape[0] >= rows)):
            continue
        _expect(t.dtype == dtype, f"{what}[{i}] has dtype {t.dtype}, expected {dtype}")
        _expect(t.dim() == 2, f"{what}[{i}] must be 2-D")
        _expect(exact_shape is None or tuple(t.shape) == exact_shape,
                f"{what}[{i}] has shape {tuple(t.shape)}, expected {exact_shape}")
        _expect(t.shape[1] == cols, f"{what}[{i}] has {t.shape[1]} columns, expected {cols}")
        _expect(rows is None or t.shape[0] >= rows, f"{what}[{i}] has {t.shape[0]} rows, fewer than {rows}")


def _check_offsets(offsets: torch.Tensor, G: int) -> None:
    _expect(offsets.dtype == torch.int32 and offsets.numel() == G + 1, f"offsets must be int32 with {G + 1} entries")


def _shared_rows(rows_from_offsets: bool, rows_cap: int) -> int:
    # Routed experts share one buffer indexed by the offsets, shared experts have a buffer each:
    # either way every buffer must hold rows_cap rows.
    return rows_cap


def gemm_kernel(dtype: torch.dtype, act: str, h: int, f: int) -> str:
    """Which kernel the expert GEMMs run for these operands: ``"mfma"`` or ``"generic"``."""
    code = C.lib().rhp_expert_gemm_kernel(dtype_code_of(dtype), act_code(act), h, f)
    return "mfma" if code == C.GEMM_KERNEL_MFMA else "generic"


def dtype_code_of(dtype: torch.dtype) -> int:
    try:
        return _DT[dtype]
    except KeyError:
        raise KernelArgumentError(f"unsupported dtype {dtype}") from None


# K-split workspaces, one per (device, stream): its arrival counters are shared by every launch that
# uses it, so launches on two streams must not share one.  At most _SPLIT_WS_PER_DEVICE streams per
# device keep one (the least recently used is dropped first), so callers that make a stream per
# request do not grow device memory without bound.  A workspace is allocated on its own stream, so
# the caching allocator hands a dropped one's memory only to later work on that stream.
_SPLIT_WS_PER_DEVICE = 4
_split_ws_cache: "collections.OrderedDict[tuple[int, int], torch.Tensor]" = collections.OrderedDict()


def split_workspace(dev: torch.device, stream: torch.cuda.Stream | None = None) -> torch.Tensor:
    """The K-split workspace of the expert GEMMs for ``stream`` (default: the current stream of ``dev``).

    Allocated and zeroed once per (device, stream), for the last few streams of a device.  Its arrival
    counters must be zero before a call; every call that completes leaves them zero, and a call that
    fails resets them.  Under HIP graph capture a workspace is never allocated: make one call outside
    the capture on the same stream first, or the call raises.
    """
    idx = dev.index if isinstance(dev, torch.device) else torch.device(dev).index
    if idx is None:
        idx = torch.cuda.current_device()
    key = (idx, torch._C._cuda_getCurrentRawStream(idx) if stream is None else stream.cuda_stream)
    ws = _split_ws_cache.get(key)
    if ws is not None:
        _split_ws_cache.move_to_end(key)
        return ws
    stream = stream if stream is not None else torch.cuda.current_stream(idx)
    if torch.cuda.is_current_stream_capturing():
        raise KernelArgumentError("the expert GEMMs' K-split workspace of this stream is not allocated: "
                                  "call them once on this stream before capturing a graph")
    with torch.cuda.stream(stream):
        ws = torch.zeros(C.lib().rhp_expert_split_workspace_bytes(), dtype=torch.uint8, device=f"cuda:{idx}")
    _split_ws_cache[key] = ws
    mine = [kk for kk in _split_ws_cache if kk[0] == idx]
    for kk in mine[:max(0, len(mine) - _SPLIT_WS_PER_DEVICE)]:
        del _split_ws_cache[kk]
    return ws


def reset_split_workspace(ws: torch.Tensor, stream: torch.cuda.Stream | None = None) -> None:
    """Zeroes a K-split workspace's arrival counters on ``stream`` (a fill kernel)."""
    stream = stream if stream is not None else torch.cuda.current_stream(ws.device)
    with torch.cuda.device(ws.device):
        C.call("rhp_expert_split_workspace_reset", _ptr(ws), ws.numel(), stream.cuda_stream)


def _split_call(name: str, dev: torch.device, split: bool, *args) -> None:
    """Calls a GEMM entry point with the K-split workspace of the current stream (or none)."""
    if not split:
        _call(name, dev, *args, None, 0)
        return
    ws = split_workspace(dev)
    try:
        _call(name, dev, *args, _ptr(ws), ws.numel())
    except RuntimeError:
        # A call that did not complete may have left arrival counters set.
        reset_split_workspace(ws)
        raise


def expert_fc1_fwd(xs: list[torch.Tensor], offsets: torch.Tensor, rows_from_offsets: bool, rows_cap: int,
                   w1: list[torch.Tensor], f: int, act: str, hpre: list[torch.Tensor],
                   act_out: list[torch.Tensor], split: bool = True) -> None:
    dev = _need_cuda(offsets, _each(xs), _each(w1), _each(hpre), _each(act_out))
    G, dt, h = len(w1), w1[0].dtype, w1[0].shape[1]
    F1 = 2 * f if act == "swiglu" else f
    rows = _shared_rows(rows_from_offsets, rows_cap)
    _check_offsets(offsets, G)
    _check_groups("w1", w1, G, dt, h, exact_shape=(F1, h))
    _check_groups("x", xs, G, dt, h, rows)
    _check_groups("hpre", hpre, G, dt, F1, rows)
    _check_groups("act", act_out, G, dt, f, rows)
    _split_call("rhp_expert_fc1_fwd", dev, split, G, _ptr(offsets), int(rows_from_offsets), rows_cap,
                dtype_code(w1[0]), act_code(act), h, f, _arr(xs), _arr(w1), _arr(hpre), _arr(act_out))


def expert_fc1_act(xs: list[torch.Tensor], offsets: torch.Tensor, rows_from_offsets: bool, rows_cap: int,
                   w1: list[torch.Tensor], f: int, act: str, act_out: list[torch.Tensor], split: bool = True) -> None:
    """expert_fc1_fwd where no backward follows: only the activation rows are written."""
    dev = _need_cuda(offsets, _each(xs), _each(w1), _each(act_out))
    G, dt, h = len(w1), w1[0].dtype, w1[0].shape[1]
    rows = _shared_rows(rows_from_offsets, rows_cap)
    _check_offsets(offsets, G)
    _check_groups("w1", w1, G, dt, h, exact_shape=(2 * f if act == "swiglu" else f, h))
    _check_groups("x", xs, G, dt, h, rows)
    _check_groups("act", act_out, G, dt, f, rows)
    _split_call("rhp_expert_fc1_act", dev, split, G, _ptr(offsets), int(rows_from_offsets), rows_cap,
                dtype_code(w1[0]), act_code(act), h, f, _arr(xs), _arr(w1), _arr(act_out))


def expert_fc2_fwd(acts: list[torch.Tensor], offsets: torch.Tensor, rows_from_offsets: bool, rows_cap: int,
                   w2: list[torch.Tensor], ys: list[torch.Tensor], split: bool = True) -> None:
    dev = _need_cuda(offsets, _each(acts), _each(w2), _each(ys))
    G, dt, (h, f) = len(w2), w2[0].dtype, tuple(w2[0].shape)
    rows = _shared_rows(rows_from_offsets, rows_cap)
    _check_offsets(offsets, G)
    _check_groups("w2", w2, G, dt, f, exact_shape=(h, f))
    _check_groups("act", acts, G, dt, f, rows)
    _check_groups("y", ys, G, dt, h, rows)
    _split_call("rhp_expert_fc2_fwd", dev, split, G, _ptr(offsets), int(rows_from_offsets), rows_cap,
                dtype_code(w2[0]), h, f, _arr(acts), _arr(w2), _arr(ys))


def expert_fc2_bwd(dys: list[torch.Tensor], acts: list[torch.Tensor], hpres: list[torch.Tensor],
                   offsets: torch.Tensor, rows_from_offsets: bool, rows_cap: int, w2: list[torch.Tensor], act: str,
                   dhpre: list[torch.Tensor] | None, dw2: list[torch.Tensor] | None, split: bool = True) -> None:
    """Input-gradient product into ``dhpre`` and weight gradient into ``dw2``; either may be None (not
    both), so the two independent products can run on two streams.  ``w2`` gives the shapes either way."""
    _expect(dhpre is not None or dw2 is not None, "expert_fc2_bwd: nothing to compute")
    dev = _need_cuda(offsets, *map(_each, (dys, acts, hpres, w2, dhpre, dw2)))
    G, dt, (h, f) = len(w2), w2[0].dtype, tuple(w2[0].shape)
    F1 = 2 * f if act == "swiglu" else f
    rows = _shared_rows(rows_from_offsets, rows_cap)
    _check_offsets(offsets, G)
    _check_groups("w2", w2, G, dt, f, exact_shape=(h, f))
    _check_groups("dy", dys, G, dt, h, rows)
    if dw2 is not None:
        _check_groups("dw2", dw2, G, dt, f, exact_shape=(h, f))
        _check_groups("act", acts, G, dt, f, rows)
    if dhpre is not None:
        _check_groups("hpre", hpres, G, dt, F1, rows)
        _check_groups("dhpre", dhpre, G, dt, F1, rows)
    _split_call("rhp_expert_fc2_bwd", dev, split, G, _ptr(offsets), int(rows_from_offsets), rows_cap,
                dtype_code(w2[0]), act_code(act), h, f, _arr(dys), _arr(acts) if dw2 is not None else None,
                _arr(hpres) if dhpre is not None else None, _arr(w2), _arr(dhpre) if dhpre is not None else None,
                _arr(dw2) if dw2 is not None else None)


def expert_fc1_bwd(dhpre: list[torch.Tensor], xs: list[torch.Tensor], offsets: torch.Tensor,
                   rows_from_offsets: bool, rows_cap: int, w1: list[torch.Tensor], f: int, act: str,
                   dxs: list[torch.Tensor] | None, dw1: list[torch.Tensor] | None, split: bool = True) -> None:
    """Input gradient into ``dxs`` and weight gradient into ``dw1``; either may be None (not both)."""
    _expect(bool(dxs) or dw1 is not None, "expert_fc1_bwd: nothing to compute")
    dev = _need_cuda(offsets, *map(_each, (dhpre, xs, w1, dxs, dw1)))
    G, dt, h = len(w1), w1[0].dtype, w1[0].shape[1]
    F1 = 2 * f if act == "swiglu" else f
    rows = _shared_rows(rows_from_offsets, rows_cap)
    _check_offsets(offsets, G)
    _check_groups("w1", w1, G, dt, h, exact_shape=(F1, h))
    _check_groups("dhpre", dhpre, G, dt, F1, rows)
    if dw1 is not None:
        _check_groups("dw1", dw1, G, dt, h, exact_shape=(F1, h))
        _check_groups("x", xs, G, dt, h, rows)
    if dxs:
        _check_groups("dx", dxs, G, dt, h, rows)
    _split_call("rhp_expert_fc1_bwd", dev, split, G, _ptr(offsets), int(rows_from_offsets), rows_cap,
                dtype_code(w1[0]), act_code(act), h, f, _arr(dhpre), _arr(xs) if dw1 is not None else None, _arr(w1),
                _arr(dxs) if dxs else None, _arr(dw1) if dw1 is not None else None)


def _check_map(what: str, idx: torch.Tensor, rows_cap: int) -> None:
    _expect(idx.dtype == torch.int32 and idx.dim() == 1 and idx.is_contiguous() and idx.numel() >= rows_cap,
            f"{what}: the row map must be a contiguous int32 vector of at least {rows_cap} entries")


def expert_fc1_fwd_gather(src: torch.Tensor, src_idx: torch.Tensor, offsets: torch.Tensor, rows_cap: int,
                          w1: list[torch.Tensor], f: int, act: str, hpre: torch.Tensor, act_out: torch.Tensor,
                          split: bool = True) -> None:
    """expert_fc1_fwd on rows gathered from ``src``: grouped row r is ``src[src_idx[r]]`` (no copy)."""
    dev = _need_cuda(offsets, src, src_idx, _each(w1), hpre, act_out)
    G, dt, h = len(w1), w1[0].dtype, w1[0].shape[1]
    F1 = 2 * f if act == "swiglu" else f
    _check_offsets(offsets, G)
    _check_map("src_idx", src_idx, rows_cap)
    _check_groups("w1", w1, G, dt, h, exact_shape=(F1, h))
    _check_groups("src", [src], 1, dt, h)
    _check_groups("hpre", [hpre], 1, dt, F1, rows_cap)
    _check_groups("act", [act_out], 1, dt, f, rows_cap)
    _split_call("rhp_expert_fc1_fwd_gather", dev, split, G, _ptr(offsets), rows_cap, dtype_code(w1[0]),
                act_code(act), h, f, _ptr(src), src.shape[0], _ptr(src_idx), _arr(w1), _ptr(hpre), _ptr(act_out))


def expert_fc2_fwd_scatter(act_in: torch.Tensor, offsets: torch.Tensor, rows_cap: int, w2: list[torch.Tensor],
                           y: torch.Tensor, y_idx: torch.Tensor, split: bool = True) -> None:
    """expert_fc2_fwd writing grouped row r to ``y[y_idx[r]]`` (no copy)."""
    dev = _need_cuda(offsets, act_in, y, y_idx, _each(w2))
    G, dt, (h, f) = len(w2), w2[0].dtype, tuple(w2[0].shape)
    _check_offsets(offsets, G)
    _check_map("y_idx", y_idx, rows_cap)
    _check_groups("w2", w2, G, dt, f, exact_shape=(h, f))
    _check_groups("act", [act_in], 1, dt, f, rows_cap)
    _check_groups("y", [y], 1, dt, h)
    _split_call("rhp_expert_fc2_fwd_scatter", dev, split, G, _ptr(offsets), rows_cap, dtype_code(w2[0]), h, f,
                _ptr(act_in), _arr(w2), _ptr(y), y.shape[0], _ptr(y_idx))


def expert_fc2_dgrad_gather(dy: torch.Tensor, dy_idx: torch.Tensor, offsets: torch.Tensor, rows_cap: int,
                            w2: list[torch.Tensor], act: str, hpre: torch.Tensor, dhpre: torch.Tensor,
                            split: bool = True) -> None:
    """The input-gradient product of expert_fc2_bwd on output-gradient rows ``dy[dy_idx[r]]`` (no copy)."""
    dev = _need_cuda(offsets, dy, dy_idx, hpre, dhpre, _each(w2))
    G, dt, (h, f) = len(w2), w2[0].dtype, tuple(w2[0].shape)
    F1 = 2 * f if act == "swiglu" else f
    _check_offsets(offsets, G)
    _check_map("dy_idx", dy_idx, rows_cap)
    _check_groups("w2", w2, G, dt, f, exact_shape=(h, f))
    _check_groups("dy", [dy], 1, dt, h)
    _check_groups("hpre", [hpre], 1, dt, F1, rows_cap)
    _check_groups("dhpre", [dhpre], 1, dt, F1, rows_cap)
    _split_call("rhp_expert_fc2_dgrad_gather", dev, split, G, _ptr(offsets), rows_cap, dtype_code(w2[0]),
                act_code(act), h, f, _ptr(dy), dy.shape[0], _ptr(dy_idx), _ptr(hpre), _arr(w2), _ptr(dhpre))


def expert_fc1_dgrad_scatter(dhpre: torch.Tensor, offsets: torch.Tensor, rows_cap: int, w1: list[torch.Tensor],
                             f: int, act: str, dx: torch.Tensor, dx_idx: torch.Tensor, split: bool = True) -> None:
    """The input-gradient product of expert_fc1_bwd writing grouped row r to ``dx[dx_idx[r]]`` (no copy)."""
    dev = _need_cuda(offsets, dhpre, dx, dx_idx, _each(w1))
    G, dt, h = len(w1), w1[0].dtype, w1[0].shape[1]
    F1 = 2 * f if act == "swiglu" else f
    _check_offsets(offsets, G)
    _check_map("dx_idx", dx_idx, rows_cap)
    _check_groups("w1", w1, G, dt, h, exact_shape=(F1, h))
    _check_groups("dhpre", [dhpre], 1, dt, F1, rows_cap)
    _check_groups("dx", [dx], 1, dt, h)
    _split_call("rhp_expert_fc1_dgrad_scatter", dev, split, G, _ptr(offsets), rows_cap, dtype_code(w1[0]),
                act_code(act), h, f, _ptr(dhpre), _arr(w1), _ptr(dx), dx.shape[0], _ptr(dx_idx))


def expert_fc1_dgrad_router(dhpre: list[torch.Tensor], offsets: torch.Tensor, rows_cap: int, w1: list[torch.Tensor],
                            f: int, act: str, router_w: torch.Tensor, e0: int, perm: torch.Tensor, dl: torch.Tensor,
                            dxs: list[torch.Tensor], split: bool = True) -> None:
    """fc1's input gradient with the router term added per row: ``dxs[r] = dhpre[r] @ w1 + dl[perm[r]] *
    router_w[e0 + g]`` (then token_bwd runs without ``dl``).  Every expert of the layer must be local."""
    dev = _need_cuda(offsets, router_w, perm, dl, _each(dhpre), _each(w1), _each(dxs))
    G, dt, h = len(w1), w1[0].dtype, w1[0].shape[1]
    F1 = 2 * f if act == "swiglu" else f
    _check_offsets(offsets, G)
    _check_groups("w1", w1, G, dt, h, exact_shape=(F1, h))
    _check_groups("dhpre", dhpre, G, dt, F1, rows_cap)
    _check_groups("dx", dxs, G, dt, h, rows_cap)
    _expect(router_w.dtype == torch.float32 and router_w.dim() == 2 and router_w.shape[1] == h
            and router_w.is_contiguous() and 0 <= e0 and e0 + G <= router_w.shape[0],
            "router_w must be a contiguous float32 [E, h] holding experts e0 .. e0 + G")
    _expect(dl.dtype == torch.float32 and dl.is_contiguous(), "dl must be contiguous float32 [T, k]")
    _check_map("perm", perm, rows_cap)
    _split_call("rhp_expert_fc1_dgrad_router", dev, split, G, _ptr(offsets), rows_cap, dtype_code(w1[0]),
                act_code(act), h, f, _arr(dhpre), _arr(w1), _ptr(router_w), e0, _ptr(perm), _ptr(dl), _arr(dxs))


# ----------------------------------------------------------------------------- optimizer


def adam_step(params: list[torch.Tensor], grads: list[torch.Tensor | None], exp_avg: list[torch.Tensor],
              exp_avg_sq: list[torch.Tensor], lr: float, betas: tuple[float, float], eps: float,
              weight_decay: float, step: int) -> None:
    """One fused Adam step (resihp/runtime/optim.py:32-46) over tensors of one dtype, in place.

    ``step`` is the step number after this update (from 1); a ``None`` gradient steps with zeros.
    """
    if not params:
        return
    dev = _need_cuda(*params, *[g for g in grads if g is not None], *exp_avg, *exp_avg_sq)
    dt = params[0].dtype
    _expect(len(grads) == len(params) == len(exp_avg) == len(exp_avg_sq), "one grad and two moments per parameter")
    for i, p in enumerate(params):
        for what, t in (("grad", grads[i]), ("exp_avg", exp_avg[i]), ("exp_avg_sq", exp_avg_sq[i]), ("param", p)):
            if t is None:
                continue
            _expect(t.dtype == dt, f"{what} {i} has dtype {t.dtype}, expected {dt}")
            _expect(t.shape == p.shape and t.is_contiguous(), f"{what} {i} must be contiguous with the param's shape")
    numel = (ctypes.c_int64 * len(params))(*[p.numel() for p in params])
    garr = C.ptr_array([0 if g is None else g.data_ptr() for g in grads])
    _call("rhp_adam_step", dev, len(params), _arr(params), garr, _arr(exp_avg), _arr(exp_avg_sq), numel,
          dtype_code(params[0]), float(lr), float(betas[0]), float(betas[1]), float(eps), float(weight_decay),
          int(step))


# ----------------------------------------------------------------------------- layer norm


def _norm_args(x: torch.Tensor, weight: torch.Tensor | None, bias: torch.Tensor | None) -> tuple[torch.device, int]:
    """Checks a norm's rows and parameters; their device and the code of the parameters' dtype."""
    dev = x.get_device()
    t = weight if weight is not None else bias
    if (dev >= 0 and x.dim() == 2 and x.shape[1] > 0 and x.is_contiguous() and t is not None
            and (t.dtype is x.dtype or (t.dtype is torch.float32 and x.dtype is torch.bfloat16)) and t.dtype in _DT
            and t.shape == x.shape[1:] and t.get_device() == dev and t.is_contiguous()
            and (t is bias or bias is None or (bias.dtype is t.dtype and bias.shape == t.shape
                                               and bias.get_device() == dev and bias.is_contiguous()))):
        return x.device, _DT[t.dtype]   # the usual case in one condition; what fails it is named below
    d = _need_cuda(x, weight, bias)
    _expect(x.dim() == 2 and x.shape[1] >= 1, f"x must be [rows, h], got {tuple(x.shape)}")
    dt = t.dtype if t is not None else x.dtype
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None:
            _expect(tuple(t.shape) == (x.shape[1],), f"{name} must be [{x.shape[1]}], got {tuple(t.shape)}")
            _expect(t.dtype == dt, "weight and bias must have one dtype")
    _expect(dt == x.dtype or (x.dtype == torch.bfloat16 and dt == torch.float32),
            f"weight and bias of {x.dtype} rows must be {x.dtype}" +
            (" or float32" if x.dtype == torch.bfloat16 else "") + f", got {dt}")
    dtype_code(x)
    return d, dtype_code_of(dt)


def _stat_dtype(x: torch.Tensor) -> torch.dtype:
    return torch.float64 if x.dtype == torch.float64 else torch.float32


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
               eps: float = 1e-5) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Layer norm of the rows of ``x`` [T, h]: (y, mean [T], rstd [T]), the statistics in float32 (float64
    for float64 rows), as ``layer_norm_bwd`` takes them.  ``weight`` and ``bias`` ([h]; x's dtype, or
    float32 with bfloat16 rows) may be None."""
    dev, wc = _norm_args(x, weight, bias)
    T, h = x.shape
    y = torch.empty_like(x)
    mean = torch.empty(T, dtype=_stat_dtype(x), device=dev)
    rstd = torch.empty_like(mean)
    _call("rhp_layer_norm_fwd", dev, x.data_ptr(), _DT[x.dtype], _ptr(weight), _ptr(bias), wc, T, h, float(eps),
          y.data_ptr(), mean.data_ptr(), rstd.data_ptr())
    return y, mean, rstd


def layer_norm_bwd(dy: torch.Tensor, x: torch.Tensor, weight: torch.Tensor | None, mean: torch.Tensor,
                   rstd: torch.Tensor, dres: torch.Tensor | None = None, need_x: bool = True,
                   need_weight: bool = True, need_bias: bool = True, dtype: torch.dtype | None = None
                   ) -> tuple[torch.Tensor | None, torch.Tensor | None, torch.Tensor | None]:
    """Gradients (dx, dweight, dbias) of ``layer_norm`` under ``dy``; ``dres`` is added to dx (the gradient
    that reaches x beside the norm).  What is not needed is not computed and comes back as None.  dweight
    and dbias have the weight's dtype (``dtype``, or x's, without a weight)."""
    dev, _ = _norm_args(x, weight, None)
    wd = weight.dtype if weight is not None else x.dtype if dtype is None else dtype
    T, h = x.shape
    st, i = _stat_dtype(x), dev.index
    for t in (dy, dres):
        if t is not None and not (t.dtype is x.dtype and t.shape == x.shape and t.get_device() == i
                                  and t.is_contiguous()):
            _need_cuda(x, dy, dres)
            raise KernelArgumentError(f"dy and dres must be {x.dtype} with x's shape, got {t.dtype} {tuple(t.shape)}")
    for t in (mean, rstd):
        if not (t.dtype is st and t.shape == x.shape[:1] and t.get_device() == i and t.is_contiguous()):
            _need_cuda(x, mean, rstd)
            raise KernelArgumentError(f"mean and rstd must be {st} [{T}], got {t.dtype} {tuple(t.shape)}")
    if wd is not x.dtype and not (x.dtype is torch.bfloat16 and wd is torch.float32):
        raise KernelArgumentError(f"no {wd} gradients of {x.dtype} rows")
    dx = torch.empty_like(x) if need_x else None
    dw = torch.empty(h, dtype=wd, device=dev) if need_weight else None
    db = torch.empty(h, dtype=wd, device=dev) if need_bias else None
    if not (need_x or need_weight or need_bias):
        return None, None, None
    xc, ws, ws_bytes = _DT[x.dtype], None, 0
    if need_weight or need_bias:
        ws_bytes = C.lib().rhp_layer_norm_bwd_workspace_bytes(T, h, xc)
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
    _call("rhp_layer_norm_bwd", dev, dy.data_ptr(), x.data_ptr(), xc, _ptr(weight), _DT[wd], mean.data_ptr(),
          rstd.data_ptr(), _ptr(dres) if need_x else None, T, h, _ptr(dx), _ptr(dw), _ptr(db), _ptr(ws), ws_bytes)
    return dx, dw, db


# ----------------------------------------------------------------------------- AdamW, gradient norm

MOMENT_BLOCK = 128   # neighbouring elements that share an exponent, for moments in 8 bits


_CODES = {ctypes.c_void_p: "Q", ctypes.c_int64: "q", ctypes.c_int: "i", ctypes.c_uint32: "I"}
_T = torch._C.TensorBase   # its methods, mapped over lists of tensors


def _host_array(kind, values) -> ctypes.Array:
    """A ctypes array by way of ``array`` (for 135 values 1 us instead of the 8 of ctypes' own constructor)."""
    return (kind * max(1, len(values))).from_buffer(array.array(_CODES[kind], values or (0,)))


class AdamWPlan:
    """What an AdamW step needs to know of its tensors, laid out once (rhp_adamw_plan): the image on the host
    and on the device, and the tensors themselves, which it keeps alive.

    ``params`` are bfloat16 or float32 weights (or all float64); ``exp_avg`` and ``exp_avg_sq`` their
    moments in float32 (float64), or, with ``scales`` (uint8 [ceil(numel / 128), 2] a tensor), in 8 bits
    (uint8); ``masters`` float32 copies of bfloat16 weights, or None entries; ``keys`` tell the tensors'
    random bits apart (8 bits); ``decay`` False exempts a tensor from weight decay."""

    def __init__(self, params, exp_avg, exp_avg_sq, scales=None, masters=None, keys=None, decay=None):
        n = len(params)
        _expect(n > 0, "an AdamW plan needs a parameter")
        if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
            raise KernelArgumentError("an AdamW plan cannot be made while a graph is captured: step once before")
        masters = [None] * n if masters is None else list(masters)
        keys = [0] * n if keys is None else [int(k) & 0xFFFFFFFF for k in keys]
        decay = [True] * n if decay is None else list(decay)
        eight = scales is not None
        scales = list(scales) if eight else [None] * n
        _expect(n == len(exp_avg) == len(exp_avg_sq) == len(scales) == len(masters) == len(keys) == len(decay),
                "one entry per parameter in every list")
        self.device = _need_cuda(*params, *exp_avg, *exp_avg_sq, *scales, *masters)
        for i, p in enumerate(params):
            _expect(p.dtype in _DT, f"param {i}: unsupported dtype {p.dtype}")
            st = torch.uint8 if eight else _stat_dtype(p)
            for what, t in (("exp_avg", exp_avg[i]), ("exp_avg_sq", exp_avg_sq[i])):
                _expect(t.dtype == st and t.shape == p.shape, f"{what} {i} must be {st} with the param's shape")
            if eight:
                want = (-(-p.numel() // MOMENT_BLOCK), 2)
                _expect(scales[i] is not None and scales[i].dtype == torch.uint8 and tuple(scales[i].shape) == want,
                        f"scales {i} must be uint8 {want}")
            if masters[i] is not None:
                _expect(masters[i].dtype == torch.float32 and masters[i].shape == p.shape,
                        f"master {i} must be float32 with the param's shape")
        self.params, self.tensors = list(params), (list(exp_avg), list(exp_avg_sq), scales, masters)
        self.shapes, self.strides = [p.shape for p in params], [p.stride() for p in params]
        self.dtypes = [p.dtype for p in params]
        self.ptrs = [p.data_ptr() for p in params]
        self.numel = numel = _host_array(ctypes.c_int64, [p.numel() for p in params])
        size = C.lib().rhp_adamw_plan_bytes(n, numel, 8 if eight else 32)
        self.image = torch.empty(size, dtype=torch.uint8)
        addr = lambda ts: C.ptr_array([0 if t is None else t.data_ptr() for t in ts])  # noqa: E731
        C.call("rhp_adamw_plan", n, addr(params), _host_array(ctypes.c_int, [_DT[p.dtype] for p in params]),
               addr(masters), addr(exp_avg), addr(exp_avg_sq), addr(scales) if eight else None, numel,
               _host_array(ctypes.c_uint32, keys), _host_array(ctypes.c_int, [int(bool(d)) for d in decay]),
               8 if eight else 32, self.image.data_ptr(), size)
        self.dev_image = self.image.to(self.device)
        self.stream = torch._C._cuda_getCurrentRawStream(self.device.index)
        self.captured = False   # whether a graph has a step of it, which reads the image at every replay

    def holds(self, params) -> bool:
        """Whether these are the plan's parameters, in its order."""
        return len(params) == len(self.params) and all(map(operator.is_, params, self.params))

    def moved(self) -> bool:
        """Whether a parameter is no longer where the plan has it, or no longer of that type or laid out so."""
        ps = self.params
        return (list(map(_T.data_ptr, ps)) != self.ptrs or list(map(_T.size, ps)) != self.shapes
                or list(map(_T.stride, ps)) != self.strides or list(map(_T.dtype.__get__, ps)) != self.dtypes)


_GRAD_DT = {torch.float32: C.F32, torch.bfloat16: C.BF16}


class PlanGrads:
    """A plan's gradients, checked, with the arrays that the calls of one step take.  Not kept beyond it.
    ``moved``: what plan.moved() has just said, where it was asked."""

    def __init__(self, plan: AdamWPlan, grads, moved: bool | None = None):
        _expect(len(grads) == len(plan.params), "one gradient (or None) per parameter")
        if plan.moved() if moved is None else moved:
            raise KernelArgumentError("a parameter's storage has moved since the AdamW plan was made")
        taken = {torch.float64: C.F64} if plan.dtypes[0] is torch.float64 else _GRAD_DT
        there = [g for g in grads if g is not None]
        codes = [0 if g is None else taken.get(g.dtype) for g in grads]
        if (None in codes or not set(map(_T.get_device, there)) <= {plan.device.index}
                or not all(map(_T.is_contiguous, there))
                or [shape if g is None else g.shape for g, shape in zip(grads, plan.shapes)] != plan.shapes):
            for i, (g, shape) in enumerate(zip(grads, plan.shapes)):
                if g is not None and (g.dtype not in taken or g.get_device() != plan.device.index or g.shape != shape
                                      or not g.is_contiguous()):
                    raise KernelArgumentError(
                        f"gradient {i} must be contiguous with its parameter's shape {tuple(shape)}, on {plan.device}, "
                        f"float32 or bfloat16 (float64 with float64 weights): got {g.dtype} {tuple(g.shape)} on "
                        f"{g.device}")
        self.plan, self.grads, self.any = plan, grads, bool(there)
        self.ptrs = _host_array(ctypes.c_void_p, [0 if g is None else g.data_ptr() for g in grads])
        self.codes = _host_array(ctypes.c_int, codes)


def adamw_step(plan: AdamWPlan, grads, lr: float, betas: tuple[float, float], eps: float, weight_decay: float,
               step: int, grad_scale: torch.Tensor | None = None, seed: int = 0) -> None:
    """One AdamW step over the plan's tensors, in place, in one launch (up to 448 tensors and 2^30
    elements, 2^32 with moments in 8 bits).

    ``grads``: float32 or bfloat16 whatever the weight's type (float64 for float64 weights), or the plan's
    ``PlanGrads``; None steps with zeros.  ``grad_scale``: float32 tensor of one element on the device (or float64
    with float64 weights) that every gradient is multiplied with.  ``step`` counts from 1.  ``seed``: of the
    random bits that round moments of 8 bits.  A graph that captures the step needs the plan for as long as it
    is replayed."""
    if not isinstance(grads, PlanGrads):
        grads = PlanGrads(plan, grads)
    if grads.plan is not plan:
        raise KernelArgumentError("the gradients are another AdamW plan's")
    double = grad_scale is not None and grad_scale.dtype == torch.float64
    if grad_scale is not None:
        _expect((grad_scale.dtype == torch.float32 or (double and plan.dtypes[0] is torch.float64))
                and grad_scale.numel() == 1 and grad_scale.device == plan.device,
                "grad_scale must be one float32 (or float64 with float64 weights) on the plan's device")
    if torch.cuda.is_current_stream_capturing():
        plan.captured = True
    elif torch._C._cuda_getCurrentRawStream(plan.device.index) != plan.stream:
        # Should the plan be dropped while this step runs, its memory waits for this stream too.
        plan.dev_image.record_stream(torch.cuda.current_stream(plan.device))
    args = (plan.device, plan.image.data_ptr(), plan.dev_image.data_ptr(), plan.image.numel(), grads.ptrs, grads.codes,
            float(lr), float(betas[0]), float(betas[1]), float(eps), float(weight_decay), int(step), _ptr(grad_scale))
    if double:
        _call("rhp_adamw_step64", *args)
    else:
        _call("rhp_adamw_step", *args, int(seed) & 0xFFFFFFFFFFFFFFFF)


def _check_moments(q_m, q_v, scales) -> int:
    n = q_m.numel()
    _expect(q_m.dtype == q_v.dtype == scales.dtype == torch.uint8 and q_v.shape == q_m.shape,
            "codes and scales must be uint8, both moments' codes of one shape")
    want = (-(-n // MOMENT_BLOCK), 2)
    _expect(tuple(scales.shape) == want, f"scales must be {want}, got {tuple(scales.shape)}")
    return n


def moments_decode(q_m: torch.Tensor, q_v: torch.Tensor, scales: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """The values (m, v) that moments in 8 bits stand for, as bfloat16, which holds each exactly."""
    dev = _need_cuda(q_m, q_v, scales)
    n = _check_moments(q_m, q_v, scales)
    m, v = (torch.empty(q_m.shape, dtype=torch.bfloat16, device=dev) for _ in range(2))
    _call("rhp_moments_decode", dev, _ptr(q_m), _ptr(q_v), _ptr(scales), n, _ptr(m), _ptr(v))
    return m, v


def moments_encode(m: torch.Tensor, v: torch.Tensor, q_m: torch.Tensor, q_v: torch.Tensor,
                   scales: torch.Tensor) -> None:
    """Writes the 8-bit codes nearest to float32 moments; a v below zero makes its block of 128 NaN."""
    dev = _need_cuda(m, v, q_m, q_v, scales)
    n = _check_moments(q_m, q_v, scales)
    _expect(m.dtype == v.dtype == torch.float32 and m.numel() == v.numel() == n,
            "m and v must be float32, one per code")
    _call("rhp_moments_encode", dev, _ptr(m), _ptr(v), n, _ptr(q_m), _ptr(q_v), _ptr(scales))


def grad_norm(grads, max_norm: float = float("inf"), dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """[2] in ``dtype`` (float32 or float64) on the device: the 2-norm over all elements of all gradients (summed
    in float64), and min(1, max_norm / (norm + 1e-6)), which clips them.  ``grads``: tensors of any of the three
    dtypes on one device, None entries skipped; or a plan's ``PlanGrads``."""
    grads = grads if isinstance(grads, PlanGrads) else list(grads)
    if isinstance(grads, PlanGrads):
        dev, n, ptrs, codes, numel = grads.plan.device, len(grads.grads), grads.ptrs, grads.codes, grads.plan.numel
        _expect(grads.any, "grad_norm needs a gradient")
    else:
        grads = [g for g in grads if g is not None]
        n = len(grads)
        _expect(n > 0, "grad_norm needs a gradient")
        codes = [_DT.get(g.dtype) for g in grads]
        devs = set(map(_T.get_device, grads))
        if len(devs) > 1 or -1 in devs or None in codes or not all(map(_T.is_contiguous, grads)):
            _need_cuda(*grads)
            for g in grads:
                dtype_code(g)
        dev = grads[0].device
        ptrs = _host_array(ctypes.c_void_p, list(map(_T.data_ptr, grads)))
        codes = _host_array(ctypes.c_int, codes)
        numel = _host_array(ctypes.c_int64, list(map(_T.numel, grads)))
    if not max_norm > 0:
        raise KernelArgumentError(f"max_norm must be positive, got {max_norm}")
    _expect(dtype in (torch.float32, torch.float64), f"the norm is float32 or float64, not {dtype}")
    out = torch.empty(2, dtype=dtype, device=dev)
    ws_bytes = C.lib().rhp_grad_norm_workspace_bytes(n)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
    _call("rhp_grad_norm" if dtype is torch.float32 else "rhp_grad_norm64", dev, n, ptrs, codes, numel,
          float(max_norm), out.data_ptr(), ws.data_ptr(), ws_bytes)
    return out


# ----------------------------------------------------------------------------- fp8 experts

FP8_FORMATS = {"e4m3": (C.E4M3, torch.float8_e4m3fn, 448.0), "e5m2": (C.E5M2, torch.float8_e5m2, 57344.0)}
FP8_ALIGN = 128   # rows of each expert in the transposed copies are padded to this (the fp8 K step)
EPI_CODES = {"store": 0, "swiglu_fwd": 1, "gelu_fwd": 2, "swiglu_bwd": 3, "gelu_bwd": 4}


def fp8_padded_offsets(offsets: torch.Tensor) -> torch.Tensor:
    """poff[g+1] = poff[g] + roundup(rows of expert g, 128): where each expert starts in a transposed copy."""
    dev = _need_cuda(offsets)
    _expect(offsets.dtype == torch.int32 and offsets.dim() == 1 and offsets.numel() >= 2, "offsets must be int32 [G+1]")
    G = offsets.numel() - 1
    poff = torch.empty(G + 1, dtype=torch.int32, device=dev)
    _call("rhp_fp8_padded_offsets", dev, _ptr(offsets), G, FP8_ALIGN, _ptr(poff))
    return poff


def fp8_transposed_numel(cols: int, rows_cap: int, G: int) -> int:
    """Elements of a buffer that holds every expert's transposed, row-padded copy."""
    return cols * (rows_cap + (FP8_ALIGN - 1) * G)


def fp8_cast(x: torch.Tensor, offsets: torch.Tensor, poff: torch.Tensor, rows_cap: int, history: torch.Tensor,
             fmt: str, amax_bits: torch.Tensor, scale_inv: torch.Tensor, q: torch.Tensor | None = None,
             qt: torch.Tensor | None = None, margin: int = 0) -> None:
    """Delayed-scaling cast of bf16 rows to fp8 (row-major ``q`` and/or per-expert transposed ``qt``).

    ``amax_bits`` (int32 holding float bits) is raised to max |x|; ``scale_inv`` (float32 [1]) receives 1/scale.
    """
    dev = _need_cuda(x, offsets, poff, history, amax_bits, scale_inv, q, qt)
    code, fdt, _ = FP8_FORMATS[fmt]
    G = offsets.numel() - 1
    _expect(x.dtype == torch.bfloat16 and x.dim() == 2, "x must be bf16 [rows, cols]")
    rows, cols = x.shape
    _expect(cols % 64 == 0, "cols must be a multiple of 64")
    _expect(rows_cap <= rows, "rows_cap exceeds the rows of x")
    _expect(poff.dtype == torch.int32 and poff.numel() == G + 1, "poff must be int32 [G+1]")
    _expect(history.dtype == torch.float32 and history.dim() == 1, "history must be float32 [L]")
    _expect(amax_bits.dtype == torch.int32 and amax_bits.numel() == 1, "amax_bits must be int32 [1]")
    _expect(scale_inv.dtype == torch.float32 and scale_inv.numel() == 1, "scale_inv must be float32 [1]")
    _expect(q is not None or qt is not None, "nothing to write")
    if q is not None:
        _expect(q.dtype == fdt and tuple(q.shape) == (rows, cols), f"q must be {fdt} [{rows}, {cols}]")
    if qt is not None:
        _expect(qt.dtype == fdt and qt.numel() >= fp8_transposed_numel(cols, rows_cap, G), "qt is too small")
    _call("rhp_fp8_cast", dev, _ptr(x), C.BF16, cols, cols, G, _ptr(offsets), _ptr(poff), rows_cap, _ptr(history),
          history.numel(), code, margin, _ptr(amax_bits), _ptr(scale_inv), _ptr(q), _ptr(qt))


def fp8_cast_many(xs: list[torch.Tensor], histories: list[torch.Tensor], fmt: str, amax_bits: list[torch.Tensor],
                  scale_invs: list[torch.Tensor], qs: list[torch.Tensor], margin: int = 0) -> None:
    """fp8_cast of whole tensors in one launch (row-major codes only), each with its own scale state."""
    n = len(xs)
    _expect(len(histories) == n and len(amax_bits) == n and len(scale_invs) == n and len(qs) == n,
            "one history, amax, scale and code buffer per tensor")
    if n == 0:
        return
    dev = _need_cuda(*xs, *histories, *amax_bits, *scale_invs, *qs)
    code, fdt, _ = FP8_FORMATS[fmt]
    L = histories[0].numel()
    for x, hst, a, si, q in zip(xs, histories, amax_bits, scale_invs, qs):
        _expect(x.dtype == torch.bfloat16 and x.dim() == 2 and x.is_contiguous() and x.shape[1] % 64 == 0,
                "tensors must be contiguous bf16 [rows, cols], cols a multiple of 64")
        _expect(q.dtype == fdt and tuple(q.shape) == tuple(x.shape) and q.is_contiguous(), f"codes must be {fdt} like x")
        _expect(hst.dtype == torch.float32 and hst.numel() == L, f"histories must be float32 [{L}]")
        _expect(a.dtype == torch.int32 and a.numel() == 1 and si.dtype == torch.float32 and si.numel() == 1,
                "amax int32 [1] and 1/scale float32 [1] per tensor")
    rows = (ctypes.c_int64 * n)(*[x.shape[0] for x in xs])
    cols = (ctypes.c_int64 * n)(*[x.shape[1] for x in xs])
    _call("rhp_fp8_cast_many", dev, n, _arr(xs), rows, cols, _arr(histories), L, code, margin, _arr(amax_bits),
          _arr(scale_invs), _arr(qs))


def _code_state(history, amax_bits, scale_inv):
    _expect(history.dtype == torch.float32 and history.dim() == 1, "history must be float32 [L]")
    _expect(amax_bits.dtype == torch.int32 and amax_bits.numel() == 1, "amax_bits must be int32 [1]")
    _expect(scale_inv.dtype == torch.float32 and scale_inv.numel() == 1, "scale_inv must be float32 [1]")


def permute_fp8(x: torch.Tensor, pair_row: torch.Tensor, k: int, rows: int, history: torch.Tensor, fmt: str,
                amax_bits: torch.Tensor, scale_inv: torch.Tensor, margin: int = 0) -> torch.Tensor:
    """fp8 codes of ``permute(x, pair_row, k, rows)``, cast with the delayed scale of ``history`` in one pass."""
    dev = _need_cuda(x, pair_row, history, amax_bits, scale_inv)
    code, fdt, _ = FP8_FORMATS[fmt]
    _expect(x.dtype == torch.bfloat16 and x.dim() == 2 and x.is_contiguous(), "x must be contiguous bf16 [T, h]")
    T, h = x.shape
    _index(pair_row, "pair_row", (T * k,))
    _code_state(history, amax_bits, scale_inv)
    q = torch.empty(max(rows, 1), h, dtype=fdt, device=dev)   # a valid address also without rows
    _call("rhp_permute_fp8", dev, _ptr(x), T, h, k, _ptr(pair_row), code, _ptr(history), history.numel(), margin,
          _ptr(amax_bits), _ptr(scale_inv), _ptr(q))
    return q[:rows]


def combine_bwd_fp8(dout: torch.Tensor, y: torch.Tensor, gates: torch.Tensor, pair_row: torch.Tensor, rows: int,
                    history: torch.Tensor, fmt: str, amax_bits: torch.Tensor, scale_inv: torch.Tensor,
                    margin: int = 0) -> tuple[torch.Tensor, torch.Tensor]:
    """``combine_bwd`` with dy leaving as fp8 codes (the cast of its bf16 rows): (dy codes, dgates)."""
    dev = _need_cuda(dout, y, gates, pair_row, history, amax_bits, scale_inv)
    code, fdt, _ = FP8_FORMATS[fmt]
    _expect(dout.dtype == torch.bfloat16 and gates.dtype == torch.float32, "bf16 rows and float32 gates")
    T, h = dout.shape
    k = gates.shape[1]
    _index(pair_row, "pair_row", (T * k,))
    _expect(_rows_of(y, "y", h, dout.dtype) >= rows, "y has fewer rows than the plan")
    _code_state(history, amax_bits, scale_inv)
    q = torch.empty(max(rows, 1), h, dtype=fdt, device=dev)
    dgates = torch.empty_like(gates)
    _call("rhp_combine_bwd_fp8", dev, _ptr(dout), _ptr(y), _ptr(gates), _ptr(pair_row), T, h, k, _ptr(dgates), code,
          _ptr(history), history.numel(), margin, _ptr(amax_bits), _ptr(scale_inv), _ptr(q))
    return q[:rows], dgates


def fp8_amax_roll(history: torch.Tensor, amax_bits: torch.Tensor) -> None:
    """End of iteration: every history gets its pending amax prepended (newest first); the amax resets."""
    dev = _need_cuda(history, amax_bits)
    _expect(history.dtype == torch.float32 and history.dim() == 2, "history must be float32 [n, L]")
    _expect(amax_bits.dtype == torch.int32 and amax_bits.numel() == history.shape[0], "amax_bits must be int32 [n]")
    _call("rhp_fp8_amax_roll", dev, _ptr(history), _ptr(amax_bits), history.shape[0], history.shape[1])


def fp8_gemm(mode: int | bool, epi: str, offsets: torch.Tensor, rows_cap: int, ys: list[torch.Tensor], y_fmt: str,
             xs: list[torch.Tensor], x_fmt: str, N: int, K: int, Mo: int, f: int, cs: list[torch.Tensor],
             y_scale_inv: torch.Tensor, x_scale_inv: torch.Tensor, c2s: list[torch.Tensor] | None = None,
             auxs: list[torch.Tensor] | None = None) -> None:
    """Grouped fp8 product with bf16 outputs (rhp_fp8_gemm).  ``mode``: 0 (or False) row-grouped on [N, K]
    operands, 1 (or True) K-grouped on transposed copies, 2 row-grouped with x held [K, N], 3 K-grouped on
    the row-major codes [rows, Mo] and [rows, N]."""
    mode = int(mode)
    _expect(mode in (0, 1, 2, 3), "mode must be 0 to 3")
    kgroups = mode in (1, 3)
    G = offsets.numel() - 1
    dev = _need_cuda(offsets, *ys, *xs, *cs, *(c2s or []), *(auxs or []), y_scale_inv, x_scale_inv)
    ycode, ydt, _ = FP8_FORMATS[y_fmt]
    xcode, xdt, _ = FP8_FORMATS[x_fmt]
    _expect(len(cs) == G, f"expected {G} outputs")
    for t in ys:
        _expect(t.dtype == ydt, f"y operands must be {ydt}")
    for t in xs:
        _expect(t.dtype == xdt, f"x operands must be {xdt}")
    for t in cs + (c2s or []) + (auxs or []):
        _expect(t.dtype == torch.bfloat16 and t.dim() == 2, "outputs and pre-activations must be bf16 matrices")
    _expect(x_scale_inv.dtype == torch.float32 and x_scale_inv.numel() in (1, G), "x_scale_inv must be float32 [1] or [G]")
    _expect(y_scale_inv.dtype == torch.float32 and y_scale_inv.numel() == 1, "y_scale_inv must be float32 [1]")
    if mode == 3:
        _expect(len(ys) == 1 and len(xs) == 1, "K-grouped products take one buffer per operand")
        _expect(ys[0].dim() == 2 and ys[0].shape[1] == Mo and ys[0].shape[0] >= rows_cap and ys[0].is_contiguous(),
                f"y must be [>= {rows_cap}, {Mo}]")
        _expect(xs[0].dim() == 2 and xs[0].shape[1] == N and xs[0].shape[0] >= rows_cap and xs[0].is_contiguous(),
                f"x must be [>= {rows_cap}, {N}]")
        for t in cs:
            _expect(tuple(t.shape) == (Mo, N), f"outputs must be [{Mo}, {N}]")
        ldy, ldx = Mo, N
    elif kgroups:
        _expect(len(ys) == 1 and len(xs) == 1, "K-grouped products take one transposed buffer per operand")
        _expect(ys[0].numel() >= fp8_transposed_numel(Mo, rows_cap, G), "y is too small")
        _expect(xs[0].numel() >= fp8_transposed_numel(N, rows_cap, G), "x is too small")
        for t in cs:
            _expect(tuple(t.shape) == (Mo, N), f"outputs must be [{Mo}, {N}]")
        ldy = ldx = 0
    elif mode == 2:
        _expect(len(ys) == G and len(xs) == G, f"expected {G} operands per side")
        for t in ys:
            _expect(t.dim() == 2 and t.shape[1] == K and t.shape[0] >= rows_cap, f"y must be [>= {rows_cap}, {K}]")
        for t in xs:
            _expect(tuple(t.shape) == (K, N) and t.is_contiguous(), f"x must be [{K}, {N}]")
        ldy, ldx = K, N
    else:
        _expect(len(ys) == G and len(xs) == G, f"expected {G} operands per side")
        for t in ys:
            _expect(t.dim() == 2 and t.shape[1] == K and t.shape[0] >= rows_cap, f"y must be [>= {rows_cap}, {K}]")
        xrows = 2 * f if epi == "swiglu_fwd" else N
        for t in xs:
            _expect(tuple(t.shape) == (xrows, K), f"x must be [{xrows}, {K}]")
        ldy = ldx = K
    c2p = _arr(c2s) if c2s else None
    auxp = _arr(auxs) if auxs else None
    _call("rhp_fp8_gemm", dev, mode, EPI_CODES[epi], G, _ptr(offsets), rows_cap, ycode, xcode, N, K, Mo, f,
          _arr(ys), ldy, _arr(xs), ldx, _arr(cs), cs[0].shape[1], c2p, c2s[0].shape[1] if c2s else 0, auxp,
          auxs[0].shape[1] if auxs else 0, _ptr(y_scale_inv), _ptr(x_scale_inv),
          0 if x_scale_inv.numel() == 1 else 1)


def fp8_gemm_cast(epi: str, offsets: torch.Tensor, poff: torch.Tensor, rows_cap: int, ys: list[torch.Tensor],
                  y_fmt: str, xs: list[torch.Tensor], x_fmt: str, N: int, K: int, f: int,
                  y_scale_inv: torch.Tensor, x_scale_inv: torch.Tensor, history: torch.Tensor, q_fmt: str,
                  amax_bits: torch.Tensor, scale_inv: torch.Tensor, q: torch.Tensor | None, qt: torch.Tensor | None,
                  cs: list[torch.Tensor] | None = None, auxs: list[torch.Tensor] | None = None,
                  margin: int = 0, x_kn: bool = False) -> None:
    """Row-grouped fp8 product whose epilogue casts its activation output to fp8 (rhp_fp8_gemm_cast).
    ``x_kn``: the weights are held [K, N] (row-major codes; backward epilogues only).

    Forward epilogues store the pre-activation in ``cs`` and cast the activation; backward epilogues read
    the pre-activation from ``auxs`` and cast the pre-activation gradient.  The codes equal those of
    ``fp8_gemm`` followed by ``fp8_cast`` of its bf16 output, bit for bit.
    """
    G = offsets.numel() - 1
    dev = _need_cuda(offsets, poff, *ys, *xs, *(cs or []), *(auxs or []), y_scale_inv, x_scale_inv, history,
                     amax_bits, scale_inv, q, qt)
    ycode, ydt, _ = FP8_FORMATS[y_fmt]
    xcode, xdt, _ = FP8_FORMATS[x_fmt]
    qcode, qdt, _ = FP8_FORMATS[q_fmt]
    fwd = epi in ("swiglu_fwd", "gelu_fwd")
    _expect(epi in ("swiglu_fwd", "gelu_fwd", "swiglu_bwd", "gelu_bwd"), f"no quantising form of epilogue {epi!r}")
    _expect(len(ys) == G and len(xs) == G, f"expected {G} operands per side")
    for t in ys:
        _expect(t.dtype == ydt and t.dim() == 2 and t.shape[1] == K and t.shape[0] >= rows_cap,
                f"y operands must be {ydt} [>= {rows_cap}, {K}]")
    xrows = 2 * f if epi == "swiglu_fwd" else N
    xshape = (K, N) if x_kn else (xrows, K)
    _expect(not (x_kn and fwd), "[K, N] weights only with the backward epilogues")
    for t in xs:
        _expect(t.dtype == xdt and tuple(t.shape) == xshape and t.is_contiguous(),
                f"x operands must be {xdt} {list(xshape)}")
    if fwd:
        _expect(cs is not None and len(cs) == G and auxs is None, "forward epilogues take G pre-activation outputs")
    else:
        _expect(cs is None and auxs is not None and len(auxs) == G, "backward epilogues take G pre-activation inputs")
    for t in (cs or []) + (auxs or []):
        _expect(t.dtype == torch.bfloat16 and t.dim() == 2, "pre-activations must be bf16 matrices")
    _expect(poff.dtype == torch.int32 and poff.numel() == G + 1, "poff must be int32 [G+1]")
    _expect(history.dtype == torch.float32 and history.dim() == 1, "history must be float32 [L]")
    _expect(amax_bits.dtype == torch.int32 and amax_bits.numel() == 1, "amax_bits must be int32 [1]")
    _expect(scale_inv.dtype == torch.float32 and scale_inv.numel() == 1, "scale_inv must be float32 [1]")
    _expect(x_scale_inv.dtype == torch.float32 and x_scale_inv.numel() in (1, G), "x_scale_inv must be float32 [1] or [G]")
    _expect(y_scale_inv.dtype == torch.float32 and y_scale_inv.numel() == 1, "y_scale_inv must be float32 [1]")
    cols = 2 * N if epi == "swiglu_bwd" else N
    _expect(q is not None or qt is not None, "nothing to write")
    if q is not None:
        _expect(q.dtype == qdt and q.dim() == 2 and q.shape[1] == cols and q.shape[0] >= rows_cap,
                f"q must be {qdt} [>= {rows_cap}, {cols}]")
    if qt is not None:
        _expect(qt.dtype == qdt and qt.numel() >= fp8_transposed_numel(cols, rows_cap, G), "qt is too small")
    _call("rhp_fp8_gemm_cast", dev, EPI_CODES[epi], G, _ptr(offsets), _ptr(poff), rows_cap, ycode, xcode, N, K, f,
          _arr(ys), K, _arr(xs), N if x_kn else K, int(x_kn), _arr(cs) if cs else None, cs[0].shape[1] if cs else 0,
          _arr(auxs) if auxs else None, auxs[0].shape[1] if auxs else 0, _ptr(y_scale_inv), _ptr(x_scale_inv),
          0 if x_scale_inv.numel() == 1 else 1, _ptr(history), history.numel(), qcode, margin, _ptr(amax_bits),
          _ptr(scale_inv), _ptr(q), _ptr(qt))
