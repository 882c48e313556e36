"""Captured stacks whose MoEStack object is gone, on a B200: the memory that they replay on is
still theirs after the allocator gave back whatever nobody holds."""
from __future__ import annotations

import gc

import pytest
import torch

from easyinfra_b200 import configs as C
from easyinfra_b200 import ops
from easyinfra_b200.layer import LayerParams, MoELayer
from easyinfra_b200.placement import Placement
from easyinfra_b200.stack import MoEStack

pytestmark = pytest.mark.gpu
SHAPE = C.small(C.CONFIGS["qwen3"], hidden=1024, intermediate=128, num_experts=16, top_k=4, placement=None)


def make_layers(device, mx):
    E, out = SHAPE.num_experts, []
    for l in range(2):
        wgu, wd = C.expert_weights(SHAPE, l, list(range(E)), device=device, fast=True)
        if mx:
            wgu = ops.pack_mx4_weights(*ops.quantize_mx4(wgu), swiglu=True)
            wd = ops.pack_mx4_weights(*ops.quantize_mx4(wd), swiglu=False)
        out.append(MoELayer(LayerParams(C.router_weight(SHAPE, l, device), wgu, wd), Placement.default(E, 1),
                            SHAPE.top_k, SHAPE.norm_topk_prob))
    return out


def check_captures(device, mx, sizes):
    """One graph per batch size over the same layers, each from a stack that nobody keeps."""
    layers = make_layers(device, mx)
    caps = []
    for T in sizes:
        caps.append((T, MoEStack(layers).capture(T)))
        gc.collect()
        torch.cuda.empty_cache()
    hogs = [torch.full((1 << 20,), 255, dtype=torch.uint8, device=device) for _ in range(64)]  # what was free is taken
    eager = MoEStack(layers)
    for seed in range(2):
        for T, cap in caps:
            x = C.hidden_states(SHAPE, T, device=device, seed_offset=seed)
            want = eager.forward(x).clone()
            assert torch.equal(cap(x), want)
    assert all(bool((h == 255).all()) for h in hogs)


@pytest.mark.parametrize("mx", [False, True])
def test_captures_outlive_their_stacks(cuda_device, mx):
    check_captures(cuda_device, mx, (700, 256, 64, 1))


@pytest.mark.parametrize("mx", [False, True])
def test_captures_outlive_a_larger_workspace(cuda_device, mx):
    """Growing sizes: each capture's layers have outgrown the workspace of the one before."""
    check_captures(cuda_device, mx, (1, 64, 700, 3000))
