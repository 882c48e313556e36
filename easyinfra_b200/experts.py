"""Drop-in expert implementations for EasyInfra's MoE plugin points.

B200MoE follows the expert-module contract that `get_moe_impl()`
(easyinfra/generation/modules/moe/config.py:4-15) hands to the MoE block:

  * constructor (layer_idx, hidden_size, moe_intermediate_size, activation_key,
    gate_up_bias, down_bias, num_logical_experts, ep_group, moe_tp_group,
    phy2log_expert_map[G, P], **kwargs)                       native_moe.py:18-31
  * forward(hidden_states[M, H] in [source rank][local slot] order,
            expert_count: list[int] of length G*P or tensor [G, P])
    -> [M, H] in the same order, not yet weighted           moe_all2all.py:262
  * stacked weights experts_gate_up_weight [P, 2I, H] and experts_down_weight
    [P, H, I] with FusedMoE's loader contract                 fused_moe.py:46-57, 77-104

`cutlass_grouped_gemm_single` re-implements the external op that
`MOE_IMPL=cutlass` loads (easyinfra/__init__.py:6-20; called at
single_group_gemm_moe.py:81,90) on the same kernels.
"""
from __future__ import annotations

from typing import List, Sequence, Union

import numpy as np
import torch
from torch import nn
from torch.nn.parameter import Parameter

from . import ops
from .layer import regroup_tables, upload_tables


def _counts_matrix(expert_count, G: int, P: int) -> np.ndarray:
    if isinstance(expert_count, torch.Tensor):
        c = expert_count.detach().to("cpu").numpy()
    else:
        c = np.asarray(list(expert_count))
    if c.size == G * P:
        return c.reshape(G, P).astype(np.int64)
    raise ValueError(f"expert_count list length is {c.size} while ep={G} with {P} physical experts each.")


class B200MoE(nn.Module):
    def __init__(self, layer_idx: int, hidden_size: int, moe_intermediate_size: int,
                 activation_key: str, gate_up_bias: bool, down_bias: bool,
                 num_logical_experts: int, ep_group, moe_tp_group, phy2log_expert_map: torch.Tensor,
                 dtype: torch.dtype = torch.bfloat16, device=None, **kwargs):
        super().__init__()
        if activation_key != "silu":
            raise NotImplementedError(f"activation {activation_key!r}: the fused epilogue implements SwiGLU")
        if gate_up_bias or down_bias:
            raise NotImplementedError("expert biases are not supported (the reference kernels ignore them too)")
        self.layer_idx = layer_idx
        self.num_logical_experts = num_logical_experts
        self.ep_group = ep_group
        self.moe_tp_group = moe_tp_group
        self.ep_size = ep_group.group_size
        self.ep_rank = ep_group.local_rank
        self.moe_tp_size = moe_tp_group.group_size
        self.moe_tp_intermediate_size = moe_intermediate_size // self.moe_tp_size
        if self.moe_tp_intermediate_size * self.moe_tp_size != moe_intermediate_size:
            raise ValueError(f"MoE intermediate size {moe_intermediate_size} cannot divide moe_tp size "
                             f"{self.moe_tp_size}")
        if self.moe_tp_size != 1:
            raise NotImplementedError("MoE-TP > 1 (the reference forces a 1-rank MoE-TP group under EP)")
        self.num_physical_experts = phy2log_expert_map.shape[-1]
        self.num_global_experts = self.num_physical_experts * self.ep_size
        self.hidden_size = hidden_size
        I, H, P = self.moe_tp_intermediate_size, hidden_size, self.num_physical_experts
        self.experts_gate_up_weight = Parameter(self._unfilled(P, 2 * I, H, dtype, device), requires_grad=False)
        self.experts_down_weight = Parameter(self._unfilled(P, H, I, dtype, device), requires_grad=False)
        self.experts_gate_up_mx4 = self.experts_down_mx4 = None  # after quantize_mx4()
        self.experts_gate_up_bias = None
        self.experts_down_bias = None
        self._loaded = {"gate_up": [None] * (2 * P), "down": [None] * P}
        self.forward = self.forward_ep

    # -------------------------------------------------------------- weights
    @staticmethod
    def _unfilled(P, rows, K, dtype, device) -> torch.Tensor:
        """Uninitialised weights whose slots each end in a NaN, by which quantize_mx4 knows the
        ones that nothing was loaded into, however the others were filled."""
        w = torch.empty(P, rows, K, dtype=dtype, device=device)
        w[:, -1, -1] = float("nan")
        return w

    _PROJ = {"gate": ("gate_up", 0), "up": ("gate_up", 1), "down": ("down", 0)}
    _BLOCK = {"gate_up": 2, "down": 1}

    def weight_loader(self, module_name: str, value: torch.Tensor, dtype: torch.dtype, param_name: str,
                      **kwargs):
        """param_name "<physical id>.<gate|up|down>_proj.weight" (fused_moe.py:77-104):
        stacks per-slot projections into the [P, 2I, H] / [P, H, I] parameters once
        every slot of a projection has arrived."""
        parts = param_name.split(".")
        slot = int(parts[0])
        proj, off = self._PROJ[parts[1][:-5]]
        if proj not in self._loaded:
            raise ValueError(f"projection {proj} already loaded")
        dev = self.experts_gate_up_weight.device
        self._loaded[proj][self._BLOCK[proj] * slot + off] = value.to(dev)
        if all(v is not None for v in self._loaded[proj]):
            name = "experts_" + proj + "_weight"
            old = getattr(self, name)
            stacked = torch.stack(self._loaded[proj], 0).view(old.shape).to(dtype)
            setattr(self, name, Parameter(stacked, requires_grad=False))
            del self._loaded[proj]

    def quantize_mx4(self) -> None:
        """Turn the loaded bf16 weights into 4-bit MX (ops.MX4Weights, a quarter of the bytes)
        and drop them; forward then takes bf16 rows and quantises them to MX8.  hidden and
        intermediate size must be multiples of 128.  Whole-layer users bind
        experts_gate_up_mx4 / experts_down_mx4 as LayerParams weights.  These are made where
        the bf16 weights are and stay there.  The state dict holds them (in the products'
        layout) instead of the bf16 ones; loading such a state dict quantises the module."""
        if self.experts_gate_up_mx4 is not None:
            raise ValueError("the experts are MX4 already")
        # none left (all loaded), or both untouched (the caller filled the parameters)
        if len(self._loaded) == 1 or any(v is not None for parts in self._loaded.values() for v in parts):
            raise ValueError("projections still to load: " + ", ".join(sorted(self._loaded)))
        if any(w.dtype != torch.bfloat16 for w in (self.experts_gate_up_weight, self.experts_down_weight)):
            raise ValueError("quantize_mx4 takes bfloat16 experts (the MX4 products write bfloat16)")
        for name in ("experts_gate_up_weight", "experts_down_weight"):
            empty = torch.isnan(getattr(self, name)[:, -1, -1]).nonzero().flatten().tolist()
            if empty:
                raise ValueError(f"{name}: no weights in slots {empty} (their last element is a NaN)")
        gate_up = ops.pack_mx4_weights(*ops.quantize_mx4(self.experts_gate_up_weight), swiglu=True)
        down = ops.pack_mx4_weights(*ops.quantize_mx4(self.experts_down_weight), swiglu=False)
        self.experts_gate_up_mx4, self.experts_down_mx4 = gate_up, down
        self._drop_bf16()

    def _drop_bf16(self) -> None:
        self._loaded = {}
        for name in ("experts_gate_up_weight", "experts_down_weight"):
            old = getattr(self, name)
            setattr(self, name, Parameter(old.new_empty(0), requires_grad=False))

    _MX4 = ("experts_gate_up_mx4", "experts_down_mx4")

    def _save_to_state_dict(self, destination, prefix, keep_vars):
        super()._save_to_state_dict(destination, prefix, keep_vars)
        for name in self._MX4:
            w = getattr(self, name)
            if w is not None:
                destination[f"{prefix}{name}.data"], destination[f"{prefix}{name}.scales"] = w.data, w.scales

    def _load_from_state_dict(self, state_dict, prefix, local_metadata, strict, missing_keys, unexpected_keys,
                              error_msgs):
        keys = [f"{prefix}{name}.{part}" for name in self._MX4 for part in ("data", "scales")]
        there = [k for k in keys if k in state_dict]
        if len(there) == len(keys):
            self._load_mx4(*(state_dict[k] for k in keys), prefix, error_msgs)
        elif there or self.experts_gate_up_mx4 is not None:
            missing_keys += [k for k in keys if k not in there]
        super()._load_from_state_dict(state_dict, prefix, local_metadata, strict, missing_keys, unexpected_keys,
                                      error_msgs)
        unexpected_keys[:] = [k for k in unexpected_keys if k not in there]

    def _load_mx4(self, gu_data, gu_scales, down_data, down_scales, prefix, error_msgs) -> None:
        P, H, I = self.num_physical_experts, self.hidden_size, self.moe_tp_intermediate_size
        try:
            new = (ops.MX4Weights(gu_data, gu_scales, True), ops.MX4Weights(down_data, down_scales, False))
        except ValueError as e:
            error_msgs.append(f"{prefix}{self._MX4[0]}: {e}")
            return
        if (new[0].shape, new[1].shape) != ((P, 2 * I, H), (P, H, I)):
            error_msgs.append(f"size mismatch for the MX4 experts of {prefix or 'the module'}: {new[0].shape} and "
                              f"{new[1].shape} in the state dict, {(P, 2 * I, H)} and {(P, H, I)} here")
            return
        dev = self.experts_down_weight.device
        for name, w in zip(self._MX4, new):
            mine = getattr(self, name)
            if mine is None:
                d, s = ((t if dev.type == "meta" else t.to(dev, copy=True)) for t in (w.data, w.scales))
                setattr(self, name, ops.MX4Weights(d, s, w.swiglu))
            else:  # in place, as parameters are loaded: layers and graphs hold these
                mine.data.copy_(w.data)
                mine.scales.copy_(w.scales)
        self._drop_bf16()

    # -------------------------------------------------------------- forward
    def forward_ep(self, hidden_states: torch.Tensor, expert_count: Union[List[int], torch.Tensor]):
        M = hidden_states.shape[0]
        if self.experts_gate_up_mx4 is not None and hidden_states.dtype != torch.bfloat16:
            raise ValueError("MX4 experts need bfloat16 activations")
        if M == 0:
            return torch.empty_like(hidden_states)
        G, P = self.ep_size, self.num_physical_experts
        mine = _counts_matrix(expert_count, G, P)
        if int(mine.sum()) != M:
            raise ValueError(f"expert_count sums to {int(mine.sum())} but hidden_states has {M} rows")
        offs, src, dst, ln, max_seg = regroup_tables(mine)
        d_offs, d_src, d_dst, d_len = upload_tables(hidden_states.device, offs, src, dst, ln)
        if self.experts_gate_up_mx4 is not None:
            q, row_map = ops.quantize_mx8(hidden_states), None
            if G > 1:
                xe = torch.empty_like(q.buf)
                row_map = torch.empty(M, dtype=torch.int32, device=hidden_states.device)
                ops.gather_segments(q.buf, xe, d_src, d_dst, d_len, max_seg, inverse_map=row_map)
                q = ops.MX8Rows(xe, q.K)
            act = ops.grouped_swiglu_mx4(q, d_offs, self.experts_gate_up_mx4)
            return ops.grouped_down_mx4(act, d_offs, self.experts_down_mx4, out_row_map=row_map)
        if G == 1:
            act = ops.grouped_swiglu(hidden_states, d_offs, self.experts_gate_up_weight)
            return ops.grouped_down(act, d_offs, self.experts_down_weight)
        xe = torch.empty_like(hidden_states)
        row_map = torch.empty(M, dtype=torch.int32, device=hidden_states.device)
        ops.gather_segments(hidden_states, xe, d_src, d_dst, d_len, max_seg, inverse_map=row_map)
        act = ops.grouped_swiglu(xe, d_offs, self.experts_gate_up_weight)
        return ops.grouped_down(act, d_offs, self.experts_down_weight, out_row_map=row_map)

    forward_noep = forward_ep


def grouped_linear(A: torch.Tensor, weights: Sequence[torch.Tensor], block_sizes: Sequence[int]):
    """C[M, N] = A[M, K] . concat_i(B_i^T) row-blocked by block_sizes: rows of block i
    use B_i [N, K].  Blocks that share one weight tensor (the reference repeats the
    per-slot weight list once per source rank) are computed together."""
    if len(weights) != len(block_sizes):
        raise ValueError("one weight per block")
    M = int(sum(block_sizes))
    if M != A.shape[0]:
        raise ValueError(f"block_sizes sum to {M}, A has {A.shape[0]} rows")
    N, K = weights[0].shape
    C = torch.empty(M, N, dtype=A.dtype, device=A.device)
    if M == 0:
        return C
    # distinct weights in first-seen order
    key = {}
    uniq = []
    wid = []
    for w in weights:
        k = (w.data_ptr(), tuple(w.shape), tuple(w.stride()))
        if k not in key:
            key[k] = len(uniq)
            uniq.append(w)
        wid.append(key[k])
    P = len(uniq)
    base = uniq[0]
    step = base.numel()
    views = all(u.is_contiguous() and u.untyped_storage().data_ptr() == base.untyped_storage().data_ptr()
                and u.data_ptr() == base.data_ptr() + i * step * base.element_size()
                for i, u in enumerate(uniq))
    W = base.as_strided((P, N, K), (step, K, 1)) if views else torch.stack(uniq, 0)
    # regroup blocks by weight: segment (w, j) = j-th block that uses weight w
    starts = np.cumsum([0] + list(block_sizes))[:-1]
    per_w: List[List[int]] = [[] for _ in range(P)]
    for b, w in enumerate(wid):
        per_w[w].append(b)
    offs = np.zeros(P + 1, dtype=np.int64)
    src, dst, ln = [], [], []
    row = 0
    for w in range(P):
        for b in per_w[w]:
            src.append(starts[b])
            dst.append(row)
            ln.append(block_sizes[b])
            row += block_sizes[b]
        offs[w + 1] = row
    d_offs, d_src, d_dst, d_len = upload_tables(A.device, offs, np.array(src), np.array(dst), np.array(ln))
    Ae = torch.empty_like(A)
    row_map = torch.empty(M, dtype=torch.int32, device=A.device)
    ops.gather_segments(A.contiguous(), Ae, d_src, d_dst, d_len, int(max(ln)), inverse_map=row_map)
    return ops.grouped_down(Ae, d_offs, W, out=C, out_row_map=row_map)


_REGISTERED = {"done": False}


def register_torch_ops() -> None:
    """Define torch.ops.ops.cutlass_grouped_gemm_single(A, B_list, block_sizes) (and the
    aten_ variant) on the B200 kernels, unless another library already defined them."""
    if _REGISTERED["done"]:
        return
    import torch.library

    lib = torch.library.Library("ops", "FRAGMENT")
    for name in ("cutlass_grouped_gemm_single", "aten_grouped_gemm_single"):
        if hasattr(torch.ops.ops, name):
            continue
        lib.define(f"{name}(Tensor A, Tensor[] B, int[] block_sizes) -> Tensor")
        lib.impl(name, lambda A, B, block_sizes: grouped_linear(A, B, block_sizes), "CUDA")
    _REGISTERED["done"] = True
    _REGISTERED["lib"] = lib
