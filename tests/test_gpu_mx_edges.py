"""Calls of the MX operators at the edge of what they document, on a B200."""
from __future__ import annotations

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
