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
