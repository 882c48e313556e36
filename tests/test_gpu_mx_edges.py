"""Calls of the MX operators at the edge of what they document, on a B200."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from easyinfra_b200 import ops

pytestmark = pytest.mark.gpu
bf = torch.bfloat16


def gen(device, seed):
    return torch.Generator(device=device).manual_seed(seed)


def test_permute_of_one_row_in_a_wider_buffer(cuda_device):
    """MX8Rows takes rows of at least mx8_row_bytes(K) bytes; with one row their distance is
    nobody's business, an odd one too."""
    d, H, E = cuda_device, 96, 4
    x = torch.randn(1, H, generator=gen(d, 1), device=d).to(bf)
    r = ops.router(x, torch.randn(E, H, generator=gen(d, 2), device=d).to(bf), 2, renorm=True)
    q = ops.quantize_mx8(x)
    n = q.buf.shape[1]
    want = ops.permute_mx8(q, r, num_slots=E, E1=E).send.buf
    for width in (n, n + 1, n + 7, n + 16):
        buf = torch.full((1, width), 255, dtype=torch.uint8, device=d)
        buf[:, :n] = q.buf
        got = ops.permute_mx8(ops.MX8Rows(buf, H), r, num_slots=E, E1=E).send.buf
        assert torch.equal(got, want) and torch.equal(got, q.buf.expand(2, n))


def test_outputs_are_seen_by_modes(cuda_device):
    """Allocations go through torch's dispatcher while a mode listens, and are filled in
    deterministic mode; without either the results are the same."""
    from torch.utils._python_dispatch import TorchDispatchMode

    d = cuda_device
    x = torch.randn(4, 96, generator=gen(d, 3), device=d).to(bf)
    want = ops.quantize_mx8(x).buf

    class Log(TorchDispatchMode):
        def __init__(self):
            super().__init__()
            self.names = []

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            self.names.append(str(func))
            return func(*args, **(kwargs or {}))

    with Log() as log:
        got = ops.quantize_mx8(x).buf
    assert any("empty" in n for n in log.names) and torch.equal(got, want)
    before = torch.are_deterministic_algorithms_enabled()
    torch.use_deterministic_algorithms(True)
    try:
        assert (ops._empty_2d(3, 5, torch.uint8, x.device) == 255).all()
        assert torch.equal(ops.quantize_mx8(x).buf, want)
    finally:
        torch.use_deterministic_algorithms(before)


def test_eps_of_any_number_type(cuda_device):
    """As add_rmsnorm takes it: configurations hold it as whatever they were read into."""
    d = cuda_device
    x = torch.randn(3, 96, generator=gen(d, 4), device=d).to(bf)
    w = torch.ones(96, device=d, dtype=bf)
    want = ops.add_rmsnorm_mx8(x, None, w, 0.5)[1]
    for eps in (np.float32(0.5), np.float64(0.5), torch.tensor(0.5)):
        assert torch.equal(ops.add_rmsnorm_mx8(x, None, w, eps)[1], want)
    assert torch.equal(ops.add_rmsnorm_mx8(x, None, w, 1)[1], ops.add_rmsnorm_mx8(x, None, w, 1.0)[1])
