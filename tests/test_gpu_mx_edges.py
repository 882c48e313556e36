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


@pytest.mark.parametrize("dtype", [bf, torch.float32])
@pytest.mark.parametrize("T", [1, 6, 1500])
def test_prologue_outputs_in_place_of_inputs(cuda_device, T, dtype):
    """residual_out may be residual or hidden; rows of any stride, and normed rows of another."""
    d, H = cuda_device, 160
    g = gen(d, T)
    wide = torch.randn(2, T, 2 * H, generator=g, device=d).to(dtype)
    w = (1 + 0.2 * torch.randn(H, generator=g, device=d)).to(dtype)
    want = ops.add_rmsnorm_mx8(wide[0, :, :H].contiguous(), wide[1, :, :H].contiguous(), w)
    for target in (0, 1):
        buf = wide.clone()
        res, hid = buf[0, :, :H], buf[1, :, :H]
        nbuf = torch.full((T, 3 * H), 7.0, dtype=dtype, device=d)
        ro, nm, q = ops.add_rmsnorm_mx8(res, hid, w, residual_out=(res, hid)[target], normed=nbuf[:, H:2 * H])
        assert ro.data_ptr() == buf[target].data_ptr()
        for got, exp in zip((ro, nm, q.buf), (want[0], want[1], want[2].buf)):
            assert torch.equal(got, exp)
        assert torch.equal(buf[1 - target], wide[1 - target]) and torch.equal(buf[target, :, H:], wide[target, :, H:])
        assert (nbuf[:, :H] == 7).all() and (nbuf[:, 2 * H:] == 7).all()
    buf = wide.clone()  # hidden alone contiguous, the residual not
    ro, nm, q = ops.add_rmsnorm_mx8(buf[0, :, :H], buf[1, :, :H].contiguous(), w, residual_out=buf[0, :, :H])
    assert torch.equal(ro, want[0]) and torch.equal(nm, want[1]) and torch.equal(q.buf, want[2].buf)
    if T > 1:
        with pytest.raises(ValueError, match="overlaps"):
            flat = torch.zeros(T * H + 8, dtype=dtype, device=d)
            ops.add_rmsnorm_mx8(flat[:T * H].view(T, H), None, w, residual_out=flat[8:].view(T, H))


def product_problem(d, counts, H, I):
    g = gen(d, sum(counts) + H)
    P, rows = len(counts), sum(counts)
    wgu = ops.pack_mx4_weights(*ops.quantize_mx4(0.1 * torch.randn(P, 2 * I, H, generator=g, device=d)), swiglu=True)
    wd = ops.pack_mx4_weights(*ops.quantize_mx4(0.1 * torch.randn(P, H, I, generator=g, device=d)), swiglu=False)
    q = ops.quantize_mx8(torch.randn(rows, H, generator=g, device=d))
    offs = torch.tensor([0] + counts, device=d).cumsum(0)
    return q, offs, wgu, wd


def test_products_take_tables_of_other_types(cuda_device):
    """Offsets and row maps in 64 bits, and offsets that are a strided column."""
    d = cuda_device
    q, offs, wgu, wd = product_problem(d, [5, 0, 61, 2], 256, 128)
    want = ops.grouped_swiglu_mx4(q, offs.int(), wgu)
    y = ops.grouped_down_mx4(want, offs.int(), wd)
    column = torch.stack([offs.int(), offs.int() + 1], 1)[:, 0]
    assert not column.is_contiguous()
    perm = torch.randperm(68, generator=gen(d, 1), device=d)
    for table in (offs, column):
        act = ops.grouped_swiglu_mx4(q, table, wgu)
        assert torch.equal(act.data.view(torch.uint8), want.data.view(torch.uint8))
        assert torch.equal(act.scales.view(torch.uint8), want.scales.view(torch.uint8))
        assert torch.equal(ops.grouped_down_mx4(act, table, wd), y)
        assert torch.equal(ops.grouped_down_mx4(act, table, wd, out_row_map=perm)[perm], y)


@pytest.mark.parametrize("hint", [1, 100, 10000])
def test_products_on_a_stream_of_their_own(cuda_device, hint):
    """Inputs made on one stream, products on another that waits for it, results on a third;
    memory of the first ones is given back meanwhile."""
    d = cuda_device
    q, offs, wgu, wd = product_problem(d, [70, 1, 33], 512, 256)
    want = ops.grouped_down_mx4(ops.grouped_swiglu_mx4(q, offs, wgu, rows_hint=3 * hint), offs, wd, rows_hint=3 * hint)
    x = ops.dequantize_mx8(q, torch.float32)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(4):
        a.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(a):
            q2 = ops.quantize_mx8(x)
            act = ops.grouped_swiglu_mx4(q2, offs, wgu, rows_hint=3 * hint)
            del q2
            ops.quantize_mx8(torch.zeros_like(x))                # may take q2's memory, after the product
        b.wait_stream(a)
        with torch.cuda.stream(b):
            act.buf.record_stream(b)
            y = ops.grouped_down_mx4(act, offs, wd, rows_hint=3 * hint)
        torch.cuda.current_stream().wait_stream(b)
        y.record_stream(torch.cuda.current_stream())
        assert torch.equal(y, want)


@pytest.mark.parametrize("hint", [1, 100, 10000])
def test_products_repeat_themselves(cuda_device, hint):
    """The same bits from call to call, between calls on other inputs, in each kernel."""
    d = cuda_device
    counts = [300, 1, 0, 513, 130]
    q, offs, wgu, wd = product_problem(d, counts, 1024, 512)
    other = ops.quantize_mx8(torch.randn(sum(counts), 1024, generator=gen(d, 2), device=d))
    hint *= len(counts)

    def run(x):
        act = ops.grouped_swiglu_mx4(x, offs, wgu, rows_hint=hint)
        return act.data.view(torch.uint8), act.scales.view(torch.uint8), ops.grouped_down_mx4(act, offs, wd, rows_hint=hint)

    want = [[t.clone() for t in run(x)] for x in (q, other)]
    for i in range(40):
        assert all(torch.equal(a, b) for a, b in zip(run((q, other)[i % 2]), want[i % 2]))


def test_rows_beyond_32_bits(cuda_device):
    """Activation rows whose bytes, and dense rows whose elements, pass 2^32: the last rows are
    those of a call on them alone, in every kernel."""
    d, rows, K, tail = cuda_device, 2_100_000, 2048, 300
    if torch.cuda.mem_get_info(d)[0] < 40 << 30:
        pytest.skip("needs 40 GB")
    x = torch.randn(rows, K, generator=gen(d, 1), device=d, dtype=bf)
    w = torch.ones(K, dtype=bf, device=d)
    q = ops.quantize_mx8(x)
    assert rows * q.buf.stride(0) > 2 ** 32 and x.numel() > 2 ** 32
    small = ops.quantize_mx8(x[-tail:])
    assert torch.equal(q.buf[-tail:], small.buf) and torch.equal(ops.dequantize_mx8(q)[-tail:], ops.dequantize_mx8(small))
    for a, b in zip(ops.quantize_mx4(x), ops.quantize_mx4(x[-tail:])):
        assert torch.equal(a[-tail:], b)
    ro, nm, qn = ops.add_rmsnorm_mx8(x, None, w)
    ro2, nm2, qn2 = ops.add_rmsnorm_mx8(x[-tail:], None, w)
    assert torch.equal(ro[-tail:], ro2) and torch.equal(nm[-tail:], nm2) and torch.equal(qn.buf[-tail:], qn2.buf)
    del x, ro, nm, qn
    g = gen(d, 2)
    wgu = ops.pack_mx4_weights(*ops.quantize_mx4(0.1 * torch.randn(2, 256, K, generator=g, device=d)), swiglu=True)
    wd = ops.pack_mx4_weights(*ops.quantize_mx4(0.1 * torch.randn(2, 256, K, generator=g, device=d)), swiglu=False)
    offs = torch.tensor([0, rows - tail, rows], dtype=torch.int32, device=d)
    alone = torch.tensor([0, 0, tail], dtype=torch.int32, device=d)
    act2, y2 = ops.grouped_swiglu_mx4(small, alone, wgu), ops.grouped_down_mx4(small, alone, wd)
    for hint in (2, 200, 20000):
        act = ops.grouped_swiglu_mx4(q, offs, wgu, rows_hint=hint)
        assert torch.equal(act.data[-tail:].view(torch.uint8), act2.data.view(torch.uint8))
        assert torch.equal(act.scales[-tail:].view(torch.uint8), act2.scales.view(torch.uint8))
        assert torch.equal(ops.grouped_down_mx4(q, offs, wd, rows_hint=hint)[-tail:], y2)
    del q, act
    torch.cuda.empty_cache()
