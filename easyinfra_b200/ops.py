"""Torch-facing wrappers of the C-ABI entry points.

Each wrapper validates devices/dtypes, allocates its outputs with PyTorch on the
input's device, and launches on the current CUDA stream.  Nothing here computes on
the CPU: a missing library or a non-CUDA tensor raises.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional

import torch

from . import _lib

_DT = {torch.bfloat16: _lib.DTYPE_BF16, torch.float32: _lib.DTYPE_F32}

# Kernel launches issued through this module (for launch accounting in benchmarks).
LAUNCHES = {"count": 0}


def _count(n: int) -> None:
    LAUNCHES["count"] += n


# Optional callable(name, "start" | "end") invoked around kernel launches on the
# launching stream; benchmarks use it to record CUDA events around one kernel.
EVENT_HOOK = {"fn": None}


def _hook(name: str, phase: str) -> None:
    fn = EVENT_HOOK["fn"]
    if fn is not None:
        fn(name, phase)


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


def _need_cuda(*ts: Optional[torch.Tensor]) -> None:
    for t in ts:
        if t is not None and not t.is_cuda:
            raise ValueError("easyinfra_b200 ops take CUDA tensors only (no CPU path)")


def _dtype_code(t: torch.Tensor) -> int:
    if t.dtype not in _DT:
        raise TypeError(f"unsupported dtype {t.dtype}; expected bfloat16 or float32")
    return _DT[t.dtype]


def _rows_contig(t: torch.Tensor) -> torch.Tensor:
    if t.dim() != 2 or t.stride(1) != 1:
        t = t.contiguous()
    return t


@dataclass
class RouterOutput:
    topk_ids: torch.Tensor      # [T, K] int32 logical expert ids
    topk_weights: torch.Tensor  # [T, K] fp32, rounded to the activation dtype
    phys_ids: torch.Tensor      # [T, K] int32 physical slots
    slot_counts: torch.Tensor   # [num_slots] int32
    slot_offsets: torch.Tensor  # [num_slots + 1] int32
    shared_gate: Optional[torch.Tensor]  # [T] fp32 or None
    logits: Optional[torch.Tensor]       # [T, E1] fp32 or None
    workspace: torch.Tensor     # router workspace (needed by permute)


class Workspace:
    """Reusable router/permute workspace; zeroed once at allocation (the completion
    counter in its first bytes must start at zero and every call leaves it at zero).
    A buffer that was outgrown stays allocated: a graph captured with it replays on its
    address.  Every one is at least twice the last, so all of them together are less than
    twice the newest."""

    def __init__(self, device: torch.device):
        self.device = device
        self.buf = torch.zeros(0, dtype=torch.uint8, device=device)
        self.outgrown = []

    def get(self, nbytes: int) -> torch.Tensor:
        if self.buf.numel() < nbytes:
            self.outgrown.append(self.buf)
            self.buf = torch.zeros(max(nbytes, 2 * self.buf.numel()), dtype=torch.uint8,
                                   device=self.device)
        return self.buf


def router_workspace_bytes(T: int, E1: int, num_slots: int) -> int:
    return int(_lib.load().b200moe_router_workspace_bytes(T, E1, num_slots))


def _router_outputs(T, H, x_dtype, dev, gate_w, top_k, gate_bias, has_shared_gate, log2phy, rep_count,
                    num_slots, keep_logits, workspace):
    """Validated inputs and freshly allocated outputs of one softmax-router call."""
    E1 = gate_w.shape[0]
    E = E1 - (1 if has_shared_gate else 0)
    if gate_w.dtype != x_dtype or gate_w.shape[1] != H:
        raise ValueError("gate_w must be [E(+1), H] with x's dtype")
    gate_w = gate_w.contiguous()
    if num_slots is None:
        num_slots = E
    out = dict(
        E=E, E1=E1, gate_w=gate_w, num_slots=num_slots,
        topk_ids=torch.empty(T, top_k, dtype=torch.int32, device=dev),
        topk_w=torch.empty(T, top_k, dtype=torch.float32, device=dev),
        phys=torch.empty(T, top_k, dtype=torch.int32, device=dev),
        counts=torch.empty(num_slots, dtype=torch.int32, device=dev),
        offsets=torch.empty(num_slots + 1, dtype=torch.int32, device=dev),
        sg=torch.empty(T, dtype=torch.float32, device=dev) if has_shared_gate else None,
        logits=torch.empty(T, E1, dtype=torch.float32, device=dev) if keep_logits else None)
    out["ws"] = (workspace or Workspace(dev)).get(router_workspace_bytes(T, E1, num_slots))
    if gate_bias is not None:
        # one fp32 bias per router column; the shared-expert gate column has none
        gate_bias = gate_bias.to(torch.float32).reshape(-1)
        if has_shared_gate and gate_bias.numel() == E:
            gate_bias = torch.cat([gate_bias, gate_bias.new_zeros(1)])
        if gate_bias.numel() != E1:
            raise ValueError(f"gate_bias has {gate_bias.numel()} entries, router has {E1} columns")
        gate_bias = gate_bias.contiguous()
    out["gate_bias"] = gate_bias
    out["max_rep"] = 0
    if log2phy is not None:
        log2phy = log2phy.to(torch.int32).contiguous()
        rep_count = rep_count.to(torch.int32).contiguous()
        out["max_rep"] = log2phy.shape[1]
    out["log2phy"], out["rep_count"] = log2phy, rep_count
    return out


def _router_result(o) -> "RouterOutput":
    return RouterOutput(o["topk_ids"], o["topk_w"], o["phys"], o["counts"], o["offsets"], o["sg"], o["logits"],
                        o["ws"])


def _router_tail(o, T, H, top_k, renorm, scale, has_shared_gate, status):
    """The router arguments after x (shared by b200moe_router and b200moe_add_rmsnorm_router)."""
    return (o["gate_w"].data_ptr(), _ptr(o["gate_bias"]), int(has_shared_gate), T, H, o["E"], top_k, int(renorm),
            float(scale), _ptr(o["log2phy"]), _ptr(o["rep_count"]), o["max_rep"], o["num_slots"],
            o["topk_ids"].data_ptr(), o["topk_w"].data_ptr(), o["phys"].data_ptr(), _ptr(o["sg"]),
            o["counts"].data_ptr(), o["offsets"].data_ptr(), _ptr(o["logits"]), o["ws"].data_ptr(),
            o["ws"].numel(), _ptr(status), _stream())


def _router_launches(T: int) -> int:
    # batches of up to 8 tokens run as one fused launch (logits + selection)
    return 0 if T == 0 else (1 if T <= 8 else 2)


def _in_place(residual: torch.Tensor, hidden: Optional[torch.Tensor], ro: torch.Tensor) -> bool:
    # the C-ABI runs the separate kernels when residual_out overlaps residual under an add
    if hidden is None or residual.shape[0] == 0:
        return False
    span = ((residual.shape[0] - 1) * residual.stride(0) + residual.shape[1]) * residual.element_size()
    r0, o0 = residual.data_ptr(), ro.data_ptr()
    return o0 < r0 + span and r0 < o0 + span


def _prologue_router_launches(T: int, in_place: bool) -> int:
    if T == 0:
        return 0
    return 1 if T <= 8 and not in_place else 1 + _router_launches(T)


def router(x: torch.Tensor, gate_w: torch.Tensor, top_k: int, *, renorm: bool,
           gate_bias: Optional[torch.Tensor] = None, scale: float = 1.0,
           has_shared_gate: bool = False, log2phy: Optional[torch.Tensor] = None,
           rep_count: Optional[torch.Tensor] = None, num_slots: Optional[int] = None,
           keep_logits: bool = False, workspace: Optional[Workspace] = None,
           status: Optional[torch.Tensor] = None) -> RouterOutput:
    """softmax top-k routing + replica pick + slot histogram (one call; two kernels, or
    one for batches of up to 8 tokens)."""
    _need_cuda(x, gate_w, gate_bias, log2phy, rep_count, status)
    x = _rows_contig(x)
    T, H = x.shape
    o = _router_outputs(T, H, x.dtype, x.device, gate_w, top_k, gate_bias, has_shared_gate, log2phy, rep_count,
                        num_slots, keep_logits, workspace)
    _lib.call("b200moe_router", x.data_ptr(), x.stride(0), _dtype_code(x),
              *_router_tail(o, T, H, top_k, renorm, scale, has_shared_gate, status))
    _count(_router_launches(T))
    return _router_result(o)


def add_rmsnorm_router(residual: torch.Tensor, hidden: Optional[torch.Tensor], norm_weight: torch.Tensor,
                       eps: float, gate_w: torch.Tensor, top_k: int, *, renorm: bool,
                       residual_out: Optional[torch.Tensor] = None, normed: Optional[torch.Tensor] = None,
                       gate_bias: Optional[torch.Tensor] = None, scale: float = 1.0,
                       has_shared_gate: bool = False, log2phy: Optional[torch.Tensor] = None,
                       rep_count: Optional[torch.Tensor] = None, num_slots: Optional[int] = None,
                       workspace: Optional[Workspace] = None, status: Optional[torch.Tensor] = None,
                       permute: bool = False, send: Optional[torch.Tensor] = None):
    """The block prologue (residual += hidden; normed = RMSNorm) and the router in one
    call: one launch for batches of up to 8 tokens.  Returns (residual_out, normed,
    RouterOutput); bit-identical to add_rmsnorm followed by router.  With permute=True
    the routed rows are permuted too (in the same launch up to 8 tokens; `send` is the
    optional [>= T*K, H] send buffer) and a PermuteOutput is returned fourth,
    bit-identical to calling permute afterwards.  An in-place add (residual_out
    overlapping residual) runs the separate kernels."""
    _need_cuda(residual, hidden, norm_weight, gate_w, gate_bias, log2phy, rep_count, status)
    residual = _rows_contig(residual)
    T, H = residual.shape
    if hidden is not None:
        hidden = _rows_contig(hidden)
        if hidden.stride(0) != residual.stride(0):
            raise ValueError("residual and hidden must share a row stride")
    ro = residual_out if residual_out is not None else torch.empty_like(residual)
    nm = normed if normed is not None else torch.empty_like(residual)
    if ro.stride(0) != residual.stride(0):
        raise ValueError("residual_out must have residual's row stride")
    o = _router_outputs(T, H, residual.dtype, residual.device, gate_w, top_k, gate_bias, has_shared_gate, log2phy,
                        rep_count, num_slots, False, workspace)
    head = (residual.data_ptr(), _ptr(hidden), norm_weight.contiguous().data_ptr(), float(eps), residual.stride(0),
            ro.data_ptr(), nm.data_ptr(), nm.stride(0), _dtype_code(residual))
    if not permute:
        _lib.call("b200moe_add_rmsnorm_router", *head, *_router_tail(o, T, H, top_k, renorm, scale,
                                                                     has_shared_gate, status))
        _count(_prologue_router_launches(T, _in_place(residual, hidden, ro)))
        return ro, nm, _router_result(o)
    if nm.stride(0) != H:
        raise ValueError("the permute reads normed rows with row stride H")
    sb = send if send is not None else torch.empty(T * top_k, H, dtype=residual.dtype, device=residual.device)
    if sb.shape[0] < T * top_k or sb.shape[1] != H or not sb.is_contiguous():
        raise ValueError("send buffer must be contiguous [>= T*K, H]")
    pos_of = torch.empty(T, top_k, dtype=torch.int32, device=residual.device)
    tail = list(_router_tail(o, T, H, top_k, renorm, scale, has_shared_gate, status))
    # the router tail ends (..., logits_out, workspace, workspace_bytes, status, stream):
    # send and pos_of go after logits_out
    tail[-4:-4] = [sb.data_ptr(), pos_of.data_ptr()]
    _lib.call("b200moe_add_rmsnorm_router_permute", *head, *tail)
    in_place = _in_place(residual, hidden, ro)
    _count(_prologue_router_launches(T, in_place) + (1 if T > 8 or in_place else 0))
    return ro, nm, _router_result(o), PermuteOutput(sb, pos_of, None, None)


def router_sigmoid_grouped(x: torch.Tensor, gate_w: torch.Tensor, correction_bias: torch.Tensor,
                           top_k: int, *, n_group: int, topk_group: int, renorm: bool, scale: float,
                           log2phy: Optional[torch.Tensor] = None, rep_count: Optional[torch.Tensor] = None,
                           num_slots: Optional[int] = None, keep_logits: bool = False,
                           workspace: Optional[Workspace] = None,
                           status: Optional[torch.Tensor] = None) -> RouterOutput:
    """DeepSeek-V3 router: sigmoid scores + correction bias, group-limited top-k."""
    _need_cuda(x, gate_w, correction_bias, log2phy, rep_count, status)
    x = _rows_contig(x)
    T, H = x.shape
    E = gate_w.shape[0]
    if gate_w.dtype != x.dtype or gate_w.shape[1] != H:
        raise ValueError("gate_w must be [E, H] with x's dtype")
    gate_w = gate_w.contiguous()
    correction_bias = correction_bias.to(torch.float32).contiguous()
    if num_slots is None:
        num_slots = E
    dev = x.device
    topk_ids = torch.empty(T, top_k, dtype=torch.int32, device=dev)
    topk_w = torch.empty(T, top_k, dtype=torch.float32, device=dev)
    phys = torch.empty(T, top_k, dtype=torch.int32, device=dev)
    counts = torch.empty(num_slots, dtype=torch.int32, device=dev)
    offsets = torch.empty(num_slots + 1, dtype=torch.int32, device=dev)
    logits = torch.empty(T, E, dtype=torch.float32, device=dev) if keep_logits else None
    ws = (workspace or Workspace(dev)).get(router_workspace_bytes(T, E, num_slots))
    max_rep = 0
    if log2phy is not None:
        log2phy = log2phy.to(torch.int32).contiguous()
        rep_count = rep_count.to(torch.int32).contiguous()
        max_rep = log2phy.shape[1]
    _lib.call("b200moe_router_sigmoid_grouped", x.data_ptr(), x.stride(0), _dtype_code(x),
              gate_w.data_ptr(), correction_bias.data_ptr(), T, H, E, top_k, n_group, topk_group,
              int(renorm), float(scale), _ptr(log2phy), _ptr(rep_count), max_rep, num_slots,
              topk_ids.data_ptr(), topk_w.data_ptr(), phys.data_ptr(), counts.data_ptr(),
              offsets.data_ptr(), _ptr(logits), ws.data_ptr(), ws.numel(), _ptr(status), _stream())
    _count(_router_launches(T))
    return RouterOutput(topk_ids, topk_w, phys, counts, offsets, None, logits, ws)


def router_from_logits(logits: torch.Tensor, top_k: int, *, renorm: bool, round_bf16: bool,
                       scale: float = 1.0, has_shared_gate: bool = False,
                       log2phy: Optional[torch.Tensor] = None,
                       rep_count: Optional[torch.Tensor] = None,
                       num_slots: Optional[int] = None,
                       workspace: Optional[Workspace] = None,
                       status: Optional[torch.Tensor] = None) -> RouterOutput:
    """Selection half of the router on given fp32 logits [T, E(+1)]."""
    _need_cuda(logits, log2phy, rep_count, status)
    logits = logits.to(torch.float32).contiguous()
    T, E1 = logits.shape
    E = E1 - (1 if has_shared_gate else 0)
    if num_slots is None:
        num_slots = E
    dev = logits.device
    topk_ids = torch.empty(T, top_k, dtype=torch.int32, device=dev)
    topk_w = torch.empty(T, top_k, dtype=torch.float32, device=dev)
    phys = torch.empty(T, top_k, dtype=torch.int32, device=dev)
    counts = torch.empty(num_slots, dtype=torch.int32, device=dev)
    offsets = torch.empty(num_slots + 1, dtype=torch.int32, device=dev)
    sg = torch.empty(T, dtype=torch.float32, device=dev) if has_shared_gate else None
    ws = (workspace or Workspace(dev)).get(router_workspace_bytes(T, E1, num_slots))
    max_rep = 0
    if log2phy is not None:
        log2phy = log2phy.to(torch.int32).contiguous()
        rep_count = rep_count.to(torch.int32).contiguous()
        max_rep = log2phy.shape[1]
    _lib.call("b200moe_router_from_logits", logits.data_ptr(), int(has_shared_gate), T, E, top_k,
              int(renorm), float(scale), int(round_bf16), _ptr(log2phy), _ptr(rep_count),
              max_rep, num_slots, topk_ids.data_ptr(), topk_w.data_ptr(), phys.data_ptr(),
              _ptr(sg), counts.data_ptr(), offsets.data_ptr(), ws.data_ptr(), ws.numel(),
              _ptr(status), _stream())
    _count(1 if T else 0)
    return RouterOutput(topk_ids, topk_w, phys, counts, offsets, sg, logits, ws)


@dataclass
class PermuteOutput:
    send: torch.Tensor        # [T*K, H] rows in (physical slot, t*K+k) order
    pos_of: torch.Tensor      # [T, K] int32 send row of (t, k)
    send_token: Optional[torch.Tensor]  # [T*K] int64 (reference send_indices)
    send_slot: Optional[torch.Tensor]   # [T*K] int64 (reference send_weight_top_k)


def permute(x: torch.Tensor, r: RouterOutput, *, num_slots: int, E1: int,
            with_indices: bool = False, out: Optional[torch.Tensor] = None) -> PermuteOutput:
    _need_cuda(x)
    x = _rows_contig(x)
    T, H = x.shape
    K = r.phys_ids.shape[1]
    send = out if out is not None else torch.empty(T * K, H, dtype=x.dtype, device=x.device)
    if send.shape[0] < T * K or send.shape[1] != H or not send.is_contiguous():
        raise ValueError("send buffer must be contiguous [>= T*K, H]")
    pos_of = torch.empty(T, K, dtype=torch.int32, device=x.device)
    st = sl = None
    if with_indices:
        st = torch.empty(T * K, dtype=torch.int64, device=x.device)
        sl = torch.empty(T * K, dtype=torch.int64, device=x.device)
    _lib.call("b200moe_permute", x.data_ptr(), x.stride(0), _dtype_code(x), T, H, K, E1,
              r.phys_ids.data_ptr(), num_slots, send.data_ptr(), pos_of.data_ptr(), _ptr(st),
              _ptr(sl), r.workspace.data_ptr(), r.workspace.numel(), _stream())
    _count(1 if T else 0)
    return PermuteOutput(send, pos_of, st, sl)


def grouped_swiglu(x: torch.Tensor, expert_offsets: torch.Tensor, w_gate_up: torch.Tensor,
                   *, out: Optional[torch.Tensor] = None,
                   status: Optional[torch.Tensor] = None, rows_hint: int = 0,
                   hook_name: str = "grouped_swiglu") -> torch.Tensor:
    """act = silu(x Wg^T) * (x Wu^T) per expert segment; x [rows, H] bf16 expert-major.
    rows_hint: expected rows when x is a worst-case buffer (picks the kernel);
    hook_name: the name EVENT_HOOK sees (the shared expert reports itself apart)."""
    _need_cuda(x, expert_offsets, w_gate_up, status)
    if x.dtype != w_gate_up.dtype or x.dtype not in (torch.bfloat16, torch.float32):
        raise TypeError("grouped GEMMs take bfloat16 (tensor cores) or float32 activations and weights")
    x = _rows_contig(x)
    P, twoI, H = w_gate_up.shape
    I = twoI // 2
    w_gate_up = w_gate_up.contiguous()
    offs = expert_offsets.to(torch.int32).contiguous()
    if offs.numel() != P + 1:
        raise ValueError(f"expert_offsets must have P+1={P + 1} entries")
    act = out if out is not None else torch.empty(x.shape[0], I, dtype=x.dtype, device=x.device)
    if x.dtype == torch.float32:
        _lib.call("b200moe_grouped_swiglu_f32", x.data_ptr(), x.stride(0), x.shape[0], offs.data_ptr(),
                  P, H, I, w_gate_up.data_ptr(), act.data_ptr(), act.stride(0), _stream())
        _count(1 if x.shape[0] else 0)
        return act
    _hook(hook_name, "start")
    _lib.call("b200moe_grouped_swiglu_ex", x.data_ptr(), x.stride(0), x.shape[0], rows_hint,
              offs.data_ptr(), P, H, I, w_gate_up.data_ptr(), act.data_ptr(), act.stride(0),
              _ptr(status), _stream())
    _hook(hook_name, "end")
    _count(1 if x.shape[0] else 0)
    return act


def grouped_down(act: torch.Tensor, expert_offsets: torch.Tensor, w_down: torch.Tensor, *,
                 out: Optional[torch.Tensor] = None,
                 out_row_map: Optional[torch.Tensor] = None,
                 status: Optional[torch.Tensor] = None, rows_hint: int = 0) -> torch.Tensor:
    """y = act Wd^T per expert segment (optionally scattering rows through out_row_map).
    rows_hint: expected rows when act is a worst-case buffer (picks the kernel)."""
    _need_cuda(act, expert_offsets, w_down, out_row_map, status)
    if act.dtype != w_down.dtype or act.dtype not in (torch.bfloat16, torch.float32):
        raise TypeError("grouped GEMMs take bfloat16 (tensor cores) or float32 activations and weights")
    act = _rows_contig(act)
    P, H, I = w_down.shape
    w_down = w_down.contiguous()
    offs = expert_offsets.to(torch.int32).contiguous()
    y = out if out is not None else torch.empty(act.shape[0], H, dtype=act.dtype, device=act.device)
    if out_row_map is not None:
        out_row_map = out_row_map.to(torch.int32).contiguous()
    if act.dtype == torch.float32:
        _lib.call("b200moe_grouped_down_f32", act.data_ptr(), act.stride(0), act.shape[0],
                  offs.data_ptr(), P, H, I, w_down.data_ptr(), y.data_ptr(), y.stride(0),
                  _ptr(out_row_map), _stream())
        _count(1 if act.shape[0] else 0)
        return y
    _hook("grouped_down", "start")
    _lib.call("b200moe_grouped_down_ex", act.data_ptr(), act.stride(0), act.shape[0], rows_hint,
              offs.data_ptr(), P, H, I, w_down.data_ptr(), y.data_ptr(), y.stride(0),
              _ptr(out_row_map), _ptr(status), _stream())
    _hook("grouped_down", "end")
    _count(1 if act.shape[0] else 0)
    return y


def combine(y: torch.Tensor, pos_of: torch.Tensor, topk_weights: torch.Tensor, *,
            shared: Optional[torch.Tensor] = None, shared_gate: Optional[torch.Tensor] = None,
            out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """out[t] = sum_k w[t,k] y[pos_of[t,k]] (+ gate[t] * shared[t])."""
    _need_cuda(y, pos_of, topk_weights, shared, shared_gate)
    y = _rows_contig(y)
    T, K = pos_of.shape
    H = y.shape[1]
    o = out if out is not None else torch.empty(T, H, dtype=y.dtype, device=y.device)
    if shared is not None:
        shared = _rows_contig(shared)
        if shared.dtype != y.dtype:
            raise TypeError("shared must have y's dtype")
    if shared_gate is not None:
        shared_gate = shared_gate.to(torch.float32).contiguous()
    pos_of = pos_of.to(torch.int32).contiguous()
    topk_weights = topk_weights.to(torch.float32).contiguous()
    _lib.call("b200moe_combine", y.data_ptr(), y.stride(0), _dtype_code(y), pos_of.data_ptr(),
              topk_weights.data_ptr(), T, K, H, _ptr(shared),
              shared.stride(0) if shared is not None else 0, _ptr(shared_gate), o.data_ptr(),
              o.stride(0), _stream())
    _count(1 if T else 0)
    return o


def gather_segments(src: torch.Tensor, dst: torch.Tensor, src_start: torch.Tensor,
                    dst_start: torch.Tensor, length: torch.Tensor, max_rows: int,
                    inverse_map: Optional[torch.Tensor] = None) -> None:
    """dst[dst_start[i] + r] = src[src_start[i] + r] for r < length[i] (row copies);
    inverse_map[dst row] = src row when given (int32)."""
    _need_cuda(src, dst, src_start, dst_start, length, inverse_map)
    if inverse_map is not None and (inverse_map.dtype != torch.int32 or not inverse_map.is_contiguous()):
        raise ValueError("inverse_map must be a contiguous int32 tensor")
    if src.dtype != dst.dtype or src.shape[1:] != dst.shape[1:]:
        raise ValueError("src/dst row format mismatch")
    row_bytes = (src.numel() // max(src.shape[0], 1)) * src.element_size()
    src_start = src_start.to(torch.int32).contiguous()
    dst_start = dst_start.to(torch.int32).contiguous()
    length = length.to(torch.int32).contiguous()
    _lib.call("b200moe_gather_segments", src.data_ptr(), dst.data_ptr(), row_bytes,
              src_start.data_ptr(), dst_start.data_ptr(), length.data_ptr(), length.numel(),
              int(max_rows), _ptr(inverse_map), _stream())
    _count(1 if (length.numel() and max_rows) else 0)


def add_rmsnorm(residual: torch.Tensor, hidden: Optional[torch.Tensor], weight: Optional[torch.Tensor],
                eps: float = 1e-6, *, residual_out: Optional[torch.Tensor] = None,
                normed: Optional[torch.Tensor] = None, norm: bool = True):
    """(residual + hidden, weight * rmsnorm(residual + hidden)) in one pass; returns
    (residual_out, normed or None)."""
    _need_cuda(residual, hidden, weight, residual_out, normed)
    residual = _rows_contig(residual)
    T, H = residual.shape
    if hidden is not None:
        hidden = hidden.contiguous()
        if hidden.shape != residual.shape or hidden.dtype != residual.dtype:
            raise ValueError("hidden must match residual")
    ro = residual_out if residual_out is not None else torch.empty_like(residual)
    nm = None
    if norm:
        if weight is None or weight.dtype != residual.dtype or weight.numel() != H:
            raise ValueError("norm weight must be [H] in the activation dtype")
        weight = weight.contiguous()
        nm = normed if normed is not None else torch.empty_like(residual)
    _lib.call("b200moe_add_rmsnorm", residual.data_ptr(), _ptr(hidden), _ptr(weight) if norm else None,
              float(eps), T, H, _dtype_code(residual), residual.stride(0), ro.data_ptr(), _ptr(nm),
              nm.stride(0) if nm is not None else 0, _stream())
    _count(1 if T else 0)
    return ro, nm


# ------------------------------------------------------------------ microscaled (MX) formats
# Blocks of 32 elements share one power-of-two scale, held as its biased exponent
# (2^(byte - 127), 255 = NaN): the smallest one, 2^-127 at least, with which the block's
# largest magnitude does not pass the element type's largest value.  Elements are
# rounded to the nearest, ties to even; a block with a NaN or an infinity is all NaN.  (The
# OCP specification's conversion rounds the scale down and saturates: same format, other codes
# and scales where it does.)
#
# These wrappers run on the tensors' own device, whichever is current; an output may not
# overlap an input unless its operator says so.  Decode calls last
# a few microseconds on the GPU, so their host side is kept short: one pass over the
# arguments, the raw stream handle, no temporaries.
MX_BLOCK = 32

_current_device = torch._C._cuda_getDevice if hasattr(torch._C, "_cuda_getDevice") else torch.cuda.current_device
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


# torch's allocation without its argument parser, on the current device: 0.6 us instead of
# the 1.3 to 2.4 us of the public functions (the same caching allocator).  Both names are
# torch's own: the function is taken only if it gives what it is asked for, and it passes by
# dispatch modes and the deterministic fill, under which the public one allocates.
_private_empty = getattr(getattr(getattr(torch._C, "_dynamo", None), "guards", None), "_empty_strided_cuda", None)
_modes = getattr(torch._C, "_len_torch_dispatch_stack", None)
_FAST_EMPTY = {}  # "fn": the function or None, from the first allocation on


def _checked_empty(fn, modes):
    """fn, if it allocates the asked-for matrix on the current device and modes counts."""
    try:
        t = fn((2, 3), (3, 1), torch.uint8)
        if (tuple(t.shape), t.stride(), t.dtype) == ((2, 3), (3, 1), torch.uint8) and modes() >= 0 \
                and t.is_cuda and t.get_device() == _current_device():
            return fn
    except Exception:
        pass
    return None


def _empty_2d(rows: int, cols: int, dtype: torch.dtype, dev: torch.device) -> torch.Tensor:
    """Contiguous [rows, cols] on a CUDA device."""
    if "fn" not in _FAST_EMPTY:
        _FAST_EMPTY["fn"] = _checked_empty(_private_empty, _modes)
    fn = _FAST_EMPTY["fn"]
    if fn is not None and dev.index == _current_device() and not _modes() \
            and not torch.are_deterministic_algorithms_enabled():
        return fn((rows, cols), (cols, 1), dtype)
    return torch.empty_strided((rows, cols), (cols, 1), dtype=dtype, device=dev)


def _call_on(dev: torch.device, name: str, *args) -> None:
    """The entry point on dev's current stream, with dev current."""
    index = dev.index
    if index == _current_device():
        if _lib.CALL_HOOK["fn"] is None:
            rc = getattr(_lib.load(), name)(*args, _raw_stream(index))
            if rc:
                _lib.raise_error(name, rc)
        else:
            _lib.call(name, *args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            _lib.call(name, *args, _raw_stream(index))


def _mx_device(*ts: Optional[torch.Tensor]) -> torch.device:
    """The CUDA device all tensors share (the first one is given)."""
    index = ts[0].get_device()  # -1 on the CPU
    for t in ts:
        if t is not None and t.get_device() != index:
            _need_cuda(*ts)
            raise ValueError(f"tensors on {ts[0].device} and {t.device}")
    if index < 0:
        _need_cuda(ts[0])
    return ts[0].device


def _need_int32(n: int, what: str) -> None:
    # the C entry points take these as int, and ctypes would pass the low 32 bits on
    if n > 0x7fffffff:
        raise ValueError(f"{what} = {n} is above 2^31 - 1")


def mx8_row_bytes(K: int) -> int:
    """Bytes of one MX8 row: K elements, K/32 scales, padding to 16 bytes."""
    return K + (K // MX_BLOCK + 15) // 16 * 16


@dataclass
class MX8Rows:
    """Rows of e4m3 elements with their scales behind them, as one uint8 matrix
    [rows, >= mx8_row_bytes(K)]: a row moves as one piece."""
    buf: torch.Tensor
    K: int

    @property
    def rows(self) -> int:
        return self.buf.shape[0]

    @property
    def data(self) -> torch.Tensor:
        """[rows, K] float8_e4m3fn view of the elements."""
        b = self.buf
        return torch.as_strided(b.view(torch.float8_e4m3fn), (b.shape[0], self.K), b.stride())

    @property
    def scales(self) -> torch.Tensor:
        """[rows, K/32] float8_e8m0fnu view of the scales."""
        b = self.buf
        return torch.as_strided(b.view(torch.float8_e8m0fnu), (b.shape[0], self.K // MX_BLOCK), b.stride(),
                                b.storage_offset() + self.K)


@dataclass
class MX4Weights:
    """Expert weights in the layout the MX4 products read (pack_mx4_weights)."""
    data: torch.Tensor     # [P, rows/64, K/128, 64, 64] uint8, gate and up rows interleaved by 32 for swiglu
    scales: torch.Tensor   # [P, K/128, rows/128, 512] uint8
    swiglu: bool

    def __post_init__(self):
        d, s = self.data, self.scales
        if (d.dtype != torch.uint8 or s.dtype != torch.uint8 or d.dim() != 5 or d.shape[1] % 2
                or tuple(d.shape[3:]) != (64, 64) or tuple(s.shape) != (d.shape[0], d.shape[2], d.shape[1] // 2, 512)
                or not d.is_contiguous() or not s.is_contiguous() or s.device != d.device):
            raise ValueError("not the product layout of MX4 weights (pack_mx4_weights)")
        #: (P, rows, K) of the matrix it stands for ([P, 2I, H] or [P, H, I])
        self.shape = (d.shape[0], 64 * d.shape[1], 128 * d.shape[2])

    @property
    def device(self) -> torch.device:
        return self.data.device


def _row_matrix(t: torch.Tensor) -> torch.Tensor:
    """t as a 2D matrix of whole rows a kernel can walk: unit inner stride and rows that
    do not overlap (an expanded tensor is copied)."""
    if t.dim() != 2 or t.stride(1) != 1 or (t.shape[0] > 1 and t.stride(0) < t.shape[1]):
        t = t.contiguous()
    return t


def _ld(t: torch.Tensor) -> int:
    # the row stride of a one-row matrix is arbitrary
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _mx8_ld(b: torch.Tensor, K: int, what: str) -> int:
    """Row stride in bytes of MX8 rows of K elements."""
    if b.dtype != torch.uint8 or b.dim() != 2 or b.shape[1] < mx8_row_bytes(K) or b.stride(1) != 1:
        raise ValueError(f"{what} must be a uint8 matrix with rows of at least {mx8_row_bytes(K)} bytes (K={K})")
    return b.stride(0) if b.shape[0] > 1 else b.shape[1] // 16 * 16


def _new_mx8(rows: int, K: int, dev: torch.device) -> MX8Rows:
    return MX8Rows(_empty_2d(rows, mx8_row_bytes(K), torch.uint8, dev), K)


def _mx8_out(like: torch.Tensor, rows: int, K: int, out: Optional[MX8Rows]):
    """(MX8 rows to write, their row stride in bytes): the caller's, or new ones."""
    if out is None:
        n = mx8_row_bytes(K)
        return MX8Rows(_empty_2d(rows, n, torch.uint8, like.device), K), n
    if out.K != K or out.rows != rows:
        raise ValueError(f"out must hold {rows} rows of {K}")
    return out, _mx8_ld(out.buf, K, "out")


def quantize_mx8(x: torch.Tensor, *, out: Optional[MX8Rows] = None) -> MX8Rows:
    """[rows, K] bf16 or fp32 to MX8 rows (K a multiple of 32); the padding is zeroed."""
    if x.dim() != 2 or x.shape[1] % MX_BLOCK:
        raise ValueError("quantize_mx8 takes [rows, K] with K a multiple of 32")
    _need_int32(x.shape[1], "K")
    dev = _mx_device(x, None if out is None else out.buf)
    code = _dtype_code(x)
    x = _row_matrix(x)
    rows, K = x.shape
    q, ldq = _mx8_out(x, rows, K, out)
    _call_on(dev, "b200moe_quantize_mx8", x.data_ptr(), _ld(x), code, rows, K, q.buf.data_ptr(), ldq)
    _count(1 if x.numel() else 0)
    return q


def dequantize_mx8(q: MX8Rows, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values of MX8 rows, [rows, K] in bf16 or fp32."""
    _need_int32(q.K, "K")
    dev = _mx_device(q.buf)
    out = _empty_2d(q.rows, q.K, dtype, dev)
    _call_on(dev, "b200moe_dequantize_mx8", q.buf.data_ptr(), _mx8_ld(q.buf, q.K, "q"), q.rows, q.K, out.data_ptr(),
             q.K, _dtype_code(out))
    _count(1 if out.numel() else 0)
    return out


def quantize_mx4(x: torch.Tensor):
    """[..., K] bf16 or fp32 to 4-bit MX: (elements [..., K/2] uint8, two e2m1 a byte with
    the even one in the low half; scale bytes [..., K/32] uint8).  K a multiple of 32."""
    shape = x.shape
    if not shape or shape[-1] % MX_BLOCK:
        raise ValueError("quantize_mx4 takes [..., K] with K a multiple of 32")
    _need_int32(shape[-1], "K")
    dev = _mx_device(x)
    code = _dtype_code(x)
    K, n, ld = shape[-1], x.numel(), shape[-1]
    if not x.is_contiguous():
        x = _row_matrix(x)
        if len(shape) == 2:
            ld = _ld(x)
    if len(shape) == 2:
        data = _empty_2d(shape[0], K // 2, torch.uint8, dev)
        scales = _empty_2d(shape[0], K // MX_BLOCK, torch.uint8, dev)
    else:
        data = x.new_empty((*shape[:-1], K // 2), dtype=torch.uint8)
        scales = x.new_empty((*shape[:-1], K // MX_BLOCK), dtype=torch.uint8)
    _call_on(dev, "b200moe_quantize_mx4", x.data_ptr(), ld, code, n // K if K else 0, K, data.data_ptr(),
             scales.data_ptr())
    _count(1 if n else 0)
    return data, scales


def dequantize_mx4(data: torch.Tensor, scales: torch.Tensor, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values of quantize_mx4's result, [..., K] in bf16 or fp32."""
    _check_mx4(data, scales)
    _need_int32(2 * data.shape[-1], "K")
    dev = _mx_device(data, scales)
    data, scales = data.contiguous(), scales.contiguous()
    shape = data.shape
    K = 2 * shape[-1]
    out = _empty_2d(shape[0], K, dtype, dev) if len(shape) == 2 else data.new_empty((*shape[:-1], K), dtype=dtype)
    n = 2 * data.numel()
    _call_on(dev, "b200moe_dequantize_mx4", data.data_ptr(), scales.data_ptr(), n // K if K else 0, K, out.data_ptr(),
             K, _dtype_code(out))
    _count(1 if n else 0)
    return out


def _check_mx4(data: torch.Tensor, scales: torch.Tensor) -> None:
    if data.dtype != torch.uint8 or scales.dtype != torch.uint8:
        raise TypeError("MX4 elements and scales are uint8")
    a, b = data.shape, scales.shape
    if not a or a[:-1] != b[:-1] or 2 * a[-1] != MX_BLOCK * b[-1]:
        raise ValueError("MX4 elements [..., K/2] need scales [..., K/32]")


def pack_mx4_weights(data: torch.Tensor, scales: torch.Tensor, *, swiglu: bool) -> MX4Weights:
    """MX4 weights [P, rows, K/2] and their scales [P, rows, K/32] in the order the
    products read them; done once, when the weights are loaded (it only moves bytes, on
    the device where the weights are).  swiglu: the rows are [gate 0..I-1, up 0..I-1] and
    are interleaved by 32.  rows (swiglu: I) and K must be multiples of 128."""
    _check_mx4(data, scales)
    if data.dim() != 3:
        raise ValueError("expert weights are [P, rows, K/2]")
    P, N, K = data.shape[0], data.shape[1], 2 * data.shape[2]
    if N % (256 if swiglu else 128) or K % 128 or not N or not K:
        raise ValueError(f"the MX4 products need {'I' if swiglu else 'rows'} and K to be multiples of 128 "
                         f"(rows={N}, K={K})")
    if swiglu:
        data, scales = (t.reshape(P, 2, N // 64, 32, -1).transpose(1, 2).reshape(P, N, -1) for t in (data, scales))
    # clone: with one k-block the order is the caller's already, and the memory must not be
    data = data.reshape(P, N // 64, 64, K // 128, 64).transpose(2, 3).clone(memory_format=torch.contiguous_format)
    # [P, n-tile, row / 32, row % 32, k-block, block of 32] -> 512 bytes per (k-block, n-tile)
    scales = scales.reshape(P, N // 128, 4, 32, K // 128, 4).permute(0, 4, 1, 3, 2, 5)
    scales = scales.clone(memory_format=torch.contiguous_format)
    return MX4Weights(data, scales.view(P, K // 128, N // 128, 512), swiglu)


def add_rmsnorm_mx8(residual: torch.Tensor, hidden: Optional[torch.Tensor], weight: torch.Tensor, eps: float = 1e-6,
                    *, residual_out: Optional[torch.Tensor] = None, normed: Optional[torch.Tensor] = None,
                    norm: bool = True, out: Optional[MX8Rows] = None):
    """The block prologue with 8-bit rows for the experts, in one pass: returns
    (residual + hidden, normed = weight * rmsnorm of it or None, MX8Rows of normed).
    Rounding points as in add_rmsnorm, with the mean of the squares summed in 64 bits; the
    MX8 rows are quantize_mx8(normed), bit for bit.  norm=False leaves the bf16/fp32
    normed rows out.  residual_out may be residual or hidden itself."""
    shape, dtype = residual.shape, residual.dtype
    if len(shape) != 2 or shape[1] % MX_BLOCK or shape[1] == 0:
        raise ValueError("add_rmsnorm_mx8 takes [T, H] with H a multiple of 32")
    T, H = shape
    _need_int32(T, "T")
    _need_int32(H, "H")
    dev = _mx_device(residual, hidden, weight, residual_out, normed, None if out is None else out.buf)
    code = _DT.get(dtype)
    if code is None:
        _dtype_code(residual)
    if weight.dtype != dtype or weight.numel() != H:
        raise ValueError("norm weight must be [H] in the activation dtype")
    if not weight.is_contiguous():
        weight = weight.contiguous()
    if hidden is not None and (hidden.shape != shape or hidden.dtype != dtype):
        raise ValueError("hidden must match residual")
    if residual_out is None:
        # one stride serves residual, hidden and residual_out
        if not residual.is_contiguous():
            residual = residual.contiguous()
        if hidden is not None and not hidden.is_contiguous():
            hidden = hidden.contiguous()
        ld, residual_out = H, _empty_2d(T, H, dtype, dev)
    else:
        residual, hidden, ld = _strided_residual(residual, hidden, residual_out)
    ld_normed = H
    if normed is not None:
        if not norm or normed.shape != shape or normed.dtype != dtype or normed.stride(1) != 1:
            raise ValueError("normed must match residual")
        ld_normed = _ld(normed)
    elif norm:
        normed = _empty_2d(T, H, dtype, dev)
    out, ldq = _mx8_out(residual, T, H, out)
    _call_on(dev, "b200moe_add_rmsnorm_mx8", residual.data_ptr(), None if hidden is None else hidden.data_ptr(),
             weight.data_ptr(), float(eps), T, H, code, ld, residual_out.data_ptr(), normed.data_ptr() if norm else None,
             ld_normed, out.buf.data_ptr(), ldq)
    if T:
        _count(1)
    return residual_out, normed, out


def _strided_residual(residual: torch.Tensor, hidden: Optional[torch.Tensor], ro: torch.Tensor):
    """(residual, hidden, row stride) for a caller's residual_out, whose stride decides."""
    if ro.shape != residual.shape or ro.dtype != residual.dtype or ro.stride(1) != 1 or _ld(ro) < ro.shape[1]:
        raise ValueError("residual_out must match residual")
    ld = _ld(ro)
    same = ro.data_ptr() == residual.data_ptr() and _ld(residual) == ld and residual.stride(1) == 1
    if not same and _overlap(ro, residual):
        raise ValueError("residual_out overlaps residual without being it")

    def with_stride(t):
        if t.stride(1) == 1 and _ld(t) == ld:
            return t
        c = torch.empty_strided(t.shape, (ld, 1), dtype=t.dtype, device=t.device)
        return c.copy_(t)

    if not same:
        residual = with_stride(residual)
    if hidden is not None:
        if _overlap(ro, hidden) and not (ro.data_ptr() == hidden.data_ptr() and _ld(hidden) == ld):
            raise ValueError("residual_out overlaps hidden without being it")
        hidden = with_stride(hidden)
    return residual, hidden, ld


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    def span(t):
        last = sum((n - 1) * st for n, st in zip(t.shape, t.stride()))
        return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()

    if a.numel() == 0 or b.numel() == 0:
        return False
    (a0, a1), (b0, b1) = span(a), span(b)
    return a0 < b1 and b0 < a1


def _mx_product_args(x: MX8Rows, expert_offsets: torch.Tensor, w: MX4Weights, swiglu: bool):
    """(rows, their stride in bytes, offsets, P, N, K) of a product, checked."""
    if not isinstance(x, MX8Rows) or not isinstance(w, MX4Weights):
        raise TypeError("the MX4 products take MX8Rows and MX4Weights")
    if w.swiglu != swiglu:
        raise ValueError("weights packed for the " + ("gate/up" if w.swiglu else "down") + " product")
    P, N, K = w.shape
    if x.K != K:
        raise ValueError(f"activation rows of {x.K}, weights of {K}")
    if expert_offsets.numel() != P + 1:
        raise ValueError(f"expert_offsets must have P+1={P + 1} entries")
    if expert_offsets.dtype != torch.int32 or not expert_offsets.is_contiguous():
        expert_offsets = expert_offsets.to(torch.int32).contiguous()
    return x.buf, _mx8_ld(x.buf, K, "activations"), expert_offsets, P, N, K


def _check_status(status: Optional[torch.Tensor]) -> Optional[int]:
    if status is None:
        return None
    if status.dtype != torch.int32 or status.numel() < 1:
        raise ValueError("status must be an int32 tensor")
    return status.data_ptr()


def grouped_swiglu_mx4(x: MX8Rows, expert_offsets: torch.Tensor, w_gate_up: MX4Weights, *,
                       out: Optional[MX8Rows] = None, status: Optional[torch.Tensor] = None, rows_hint: int = 0,
                       hook_name: str = "grouped_swiglu") -> MX8Rows:
    """grouped_swiglu on MX8 rows and MX4 weights: MX8(silu(x Wg^T) * (x Wu^T)) per expert
    segment, accumulated in fp32 and rounded once.  Rows past expert_offsets[P] are left
    as they were, and so is what a row of out holds behind its scales."""
    b, ldx, offs, P, N, K = _mx_product_args(x, expert_offsets, w_gate_up, True)
    dev = _mx_device(b, offs, w_gate_up.data, status, None if out is None else out.buf)
    rows, I = b.shape[0], N // 2
    if out is None:
        # rows at multiples of 32 bytes: the epilogue then stores a block at once
        ld = (mx8_row_bytes(I) + 31) // 32 * 32
        out = MX8Rows(_empty_2d(rows, ld, torch.uint8, dev), I)
    elif out.K != I or out.rows < rows:
        raise ValueError(f"out must hold {rows} rows of {I}")
    else:
        ld = _mx8_ld(out.buf, I, "out")
    _hook(hook_name, "start")
    _call_on(dev, "b200moe_grouped_swiglu_mx4", b.data_ptr(), ldx, rows, rows_hint, offs.data_ptr(), P, K, I,
             w_gate_up.data.data_ptr(), w_gate_up.scales.data_ptr(), out.buf.data_ptr(), ld, _check_status(status))
    _hook(hook_name, "end")
    if rows:
        _count(1)
    return out


def grouped_down_mx4(act: MX8Rows, expert_offsets: torch.Tensor, w_down: MX4Weights, *,
                     out: Optional[torch.Tensor] = None, out_row_map: Optional[torch.Tensor] = None,
                     status: Optional[torch.Tensor] = None, rows_hint: int = 0) -> torch.Tensor:
    """grouped_down on MX8 rows and MX4 weights: y = act Wd^T per expert segment in bf16,
    optionally scattering rows through out_row_map (entries outside out are skipped and
    recorded in status; a row that two entries name holds parts of either).  Rows that no
    segment names are left as they were."""
    b, lda, offs, P, H, I = _mx_product_args(act, expert_offsets, w_down, False)
    dev = _mx_device(b, offs, w_down.data, out, out_row_map, status)
    rows = b.shape[0]
    if out is None:
        out = _empty_2d(rows, H, torch.bfloat16, dev)
        ldo = H
    else:
        if out.dtype != torch.bfloat16 or out.dim() != 2 or out.shape[1] != H or out.stride(1) != 1:
            raise ValueError(f"out must be [rows, {H}] bf16")
        ldo = _ld(out)
    if out_row_map is None:
        if out.shape[0] < rows:
            raise ValueError(f"out must have {rows} rows")
    else:
        if out_row_map.numel() < rows:
            raise ValueError(f"out_row_map must have {rows} entries")
        out_row_map = out_row_map.to(torch.int32).contiguous()
    _hook("grouped_down", "start")
    _call_on(dev, "b200moe_grouped_down_mx4", b.data_ptr(), lda, rows, rows_hint, offs.data_ptr(), P, H, I,
             w_down.data.data_ptr(), w_down.scales.data_ptr(), out.data_ptr(), ldo, out.shape[0], _ptr(out_row_map),
             _check_status(status))
    _hook("grouped_down", "end")
    if rows:
        _count(1)
    return out


def permute_mx8(x: MX8Rows, r: RouterOutput, *, num_slots: int, E1: int, with_indices: bool = False,
                out: Optional[MX8Rows] = None) -> PermuteOutput:
    """permute on MX8 rows, elements and scales together; send is MX8Rows."""
    dev = _mx_device(x.buf, None if out is None else out.buf)
    ldx = _mx8_ld(x.buf, x.K, "x")
    n = mx8_row_bytes(x.K)
    T, K = r.phys_ids.shape
    if x.rows != T:
        raise ValueError(f"{x.rows} rows, routing of {T}")
    q = out if out is not None else _new_mx8(T * K, x.K, dev)
    if q.K != x.K or q.rows < T * K:
        raise ValueError(f"out must hold {T * K} rows of {x.K}")
    if q.buf.dtype != torch.uint8 or q.buf.dim() != 2 or q.buf.shape[1] != n or not q.buf.is_contiguous():
        raise ValueError(f"out must be contiguous rows of {n} bytes")
    if ldx % 16 or x.buf.data_ptr() % 16 or q.buf.data_ptr() % 16:
        raise ValueError("MX8 rows must be 16-byte aligned")
    rows = torch.as_strided(x.buf, (T, n), (ldx, 1))  # a single row may have any stride of its own
    with torch.cuda.device(dev):
        perm = permute(rows.view(torch.bfloat16), r, num_slots=num_slots, E1=E1, with_indices=with_indices,
                       out=q.buf.view(torch.bfloat16))
    perm.send = q
    return perm
