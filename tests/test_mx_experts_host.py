"""B200MoE.quantize_mx4 without a GPU: what it refuses, before any kernel, and checkpoints of
quantised experts."""
from __future__ import annotations

import io
from types import SimpleNamespace as NS

import pytest
import torch

from easyinfra_b200 import ops
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


# ------------------------------------------------------------------ checkpoints
def quantised(seed):
    """A module as quantize_mx4 leaves it, with random codes."""
    g = torch.Generator().manual_seed(seed)

    def packed(rows, K, swiglu):
        return ops.pack_mx4_weights(torch.randint(0, 256, (P, rows, K // 2), generator=g, dtype=torch.uint8),
                                    torch.randint(0, 256, (P, rows, K // 32), generator=g, dtype=torch.uint8),
                                    swiglu=swiglu)

    m = experts()
    m.experts_gate_up_mx4, m.experts_down_mx4 = packed(2 * I, H, True), packed(H, I, False)
    m._drop_bf16()
    return m


def same(a, b):
    return all(torch.equal(getattr(u, part), getattr(v, part)) for u, v in (
        (a.experts_gate_up_mx4, b.experts_gate_up_mx4), (a.experts_down_mx4, b.experts_down_mx4))
        for part in ("data", "scales"))


def test_state_dict_holds_the_quantised_weights():
    """Into a new module and into a quantised one, which keeps its memory; alone and as part of
    another module; through a file."""
    m = quantised(1)
    buf = io.BytesIO()
    torch.save(m.state_dict(), buf)
    buf.seek(0)
    sd = torch.load(buf)
    fresh = experts()
    assert not fresh.load_state_dict(sd).missing_keys
    assert same(m, fresh) and fresh.experts_gate_up_weight.numel() == fresh.experts_down_weight.numel() == 0
    sd["experts_down_mx4.data"].fill_(0)                       # a copy, not the checkpoint's memory
    assert same(m, fresh)
    with pytest.raises(ValueError, match="MX4 already"):
        fresh.quantize_mx4()
    other = quantised(2)
    at = other.experts_down_mx4.data.data_ptr()
    assert not same(m, other)
    other.load_state_dict(m.state_dict())
    assert same(m, other) and other.experts_down_mx4.data.data_ptr() == at
    outer = torch.nn.ModuleDict({"experts": experts()})
    outer.load_state_dict(torch.nn.ModuleDict({"experts": m}).state_dict())
    assert same(m, outer["experts"])


def test_state_dict_of_other_experts_is_refused():
    m = quantised(1)
    sd = m.state_dict()
    for key in sd:
        part = {k: v for k, v in sd.items() if k != key}
        for into in (experts(), quantised(3)):
            with pytest.raises(RuntimeError, match="Missing key|size mismatch"):
                into.load_state_dict(part)
    with pytest.raises(RuntimeError, match="Unexpected key"):
        experts().load_state_dict(dict(sd, **{"experts_down_mx4.more": torch.zeros(1)}))
    with pytest.raises(RuntimeError, match="size mismatch"):    # bf16 weights into quantised experts
        quantised(1).load_state_dict(fill(experts()).state_dict())
    wide = dict(sd)
    wide["experts_down_mx4.data"] = sd["experts_down_mx4.data"].repeat(2, 1, 1, 1, 1)
    with pytest.raises(RuntimeError, match="product layout"):
        experts().load_state_dict(wide)
    wide["experts_down_mx4.scales"] = sd["experts_down_mx4.scales"].repeat(2, 1, 1, 1)
    with pytest.raises(RuntimeError, match="size mismatch"):
        experts().load_state_dict(wide)
    bf16 = fill(experts()).state_dict()
    assert sorted(bf16) == ["experts_down_weight", "experts_gate_up_weight"]
