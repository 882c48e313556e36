"""B200MoE.quantize_mx4 without a GPU: what it refuses, before any kernel."""
from __future__ import annotations

from types import SimpleNamespace as NS

import pytest
import torch

from easyinfra_b200.experts import B200MoE

bf = torch.bfloat16
P, H, I = 2, 128, 128


def experts(dtype=bf):
    one = NS(group_size=1, local_rank=0)
    return B200MoE(0, H, I, "silu", False, False, P, one, one, torch.arange(P).view(1, P), dtype=dtype)


def fill(m):
    with torch.no_grad():
        m.experts_gate_up_weight.zero_()
        m.experts_down_weight.zero_()
    return m


def test_fp32_experts_are_refused():
    """Their forward would return bf16 rows for fp32 ones."""
    m = fill(experts(torch.float32))
    with pytest.raises(ValueError, match="bfloat16 experts"):
        m.quantize_mx4()
    assert m.experts_gate_up_mx4 is None and m.experts_gate_up_weight.shape == (P, 2 * I, H)


@pytest.mark.parametrize("rows", [0, 3])
def test_quantised_experts_refuse_fp32_rows(rows):
    """The empty batch too, which used to come back as it was."""
    m = experts()
    m.experts_gate_up_mx4 = m.experts_down_mx4 = object()
    with pytest.raises(ValueError, match="bfloat16 activations"):
        m.forward(torch.zeros(rows, H), [rows, 0])
    assert m.forward(torch.zeros(0, H, dtype=bf), [0, 0]).shape == (0, H)


def test_experts_without_weights_are_refused():
    """Nothing was loaded, or one slot was left out: the memory holds whatever it held."""
    with pytest.raises(ValueError, match=r"experts_gate_up_weight: no weights in slots \[0, 1\]"):
        experts().quantize_mx4()
    m = fill(experts())
    m.experts_down_weight[1] = experts().experts_down_weight[1]
    with pytest.raises(ValueError, match=r"experts_down_weight: no weights in slots \[1\]"):
        m.quantize_mx4()


@pytest.mark.parametrize("how", ["copy", "data", "state dict", "loader", "attribute"])
def test_experts_with_weights_get_to_the_kernels(how):
    """Whichever way they came: without a GPU the first kernel call is what refuses."""
    m = experts()
    gu, down = torch.zeros(P, 2 * I, H, dtype=bf), torch.zeros(P, H, I, dtype=bf)
    if how == "copy":
        fill(m)
    elif how == "data":
        m.experts_gate_up_weight.data.copy_(gu)
        m.experts_down_weight.data.copy_(down)
    elif how == "state dict":
        m.load_state_dict({"experts_gate_up_weight": gu, "experts_down_weight": down})
    elif how == "loader":
        for p in range(P):
            m.weight_loader("experts", gu[p, :I], bf, f"{p}.gate_proj.weight")
            m.weight_loader("experts", gu[p, I:], bf, f"{p}.up_proj.weight")
            m.weight_loader("experts", down[p], bf, f"{p}.down_proj.weight")
    else:
        m.experts_gate_up_weight = torch.nn.Parameter(gu, requires_grad=False)
        m.experts_down_weight = torch.nn.Parameter(down, requires_grad=False)
    with pytest.raises(ValueError, match="CUDA tensors only"):
        m.quantize_mx4()
