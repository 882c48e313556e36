"""Microscaled operators without a GPU: the oracle's formats, the weights' product layout,
argument checks of the wrappers and of the C entry points."""
from __future__ import annotations

import pytest
import torch

from easyinfra_b200 import _lib, ops
from easyinfra_b200.experts import B200MoE
from oracle import mx_oracle as M

bf = torch.bfloat16


def test_oracle_grids_are_the_types():
    codes = torch.arange(127, dtype=torch.uint8)
    assert torch.equal(codes.view(torch.float8_e4m3fn).double(), M.E4M3)
    assert M.E2M1[-1] == 6 and M.E4M3[-1] == 448


@pytest.mark.parametrize("four_bit", [True, False])
def test_oracle_quantisation_is_the_nearest_value(four_bit):
    """Against a search over the whole grid, for values at, next to and between its points."""
    grid = M.E2M1 if four_bit else M.E4M3
    mid = (grid[1:] + grid[:-1]) / 2
    pts = torch.cat([grid, mid, mid * (1 + 2 ** -20), mid * (1 - 2 ** -20)])
    pts = torch.cat([pts, -pts])
    pts = torch.cat([pts, torch.zeros(-len(pts) % 31)])
    blocks = torch.cat([pts.view(-1, 31), torch.full((pts.numel() // 31, 1), float(grid[-1]), dtype=torch.float64)], 1)
    codes, byte = M.quantize(blocks, four_bit)
    assert (byte == 127).all()
    got = M.values(codes, byte, four_bit)
    dist = (blocks.abs()[..., None] - grid).abs()
    assert torch.equal((got - blocks).abs(), dist.min(-1).values)
    tie = (dist == dist.min(-1, keepdim=True).values).sum(-1) == 2
    assert tie.any() and (codes[tie] % 2 == 0).all()


@pytest.mark.parametrize("four_bit", [True, False])
def test_oracle_scale_is_the_smallest(four_bit):
    top = 6.0 if four_bit else 448.0
    g = torch.Generator().manual_seed(3)
    x = torch.randn(500, 32, generator=g, dtype=torch.float64) * torch.exp2(torch.randint(-60, 60, (500, 1), generator=g))
    x[0] = 0
    x[1, 0], x[1, 1:] = top * 2.0 ** 5, 0          # exactly at the border
    x[2, 0], x[2, 1:] = top * 2.0 ** 5 * (1 + 2 ** -30), 0
    x[3] = 2.0 ** -140
    _, byte = M.quantize(x, four_bit)
    s, amax = M.scale_values(byte), x.abs().amax(-1, keepdim=True)
    assert (amax <= top * s).all()
    assert ((amax > top * s / 2) | (byte == 0)).all()
    assert byte[0] == 0 and byte[3] == 0 and byte[1] == 132 and byte[2] == 133


def test_pack4_roundtrip():
    codes = torch.arange(16, dtype=torch.uint8).repeat(4).view(2, 32)
    assert torch.equal(M.unpack4(M.pack4(codes)), codes)
    assert M.pack4(codes)[0, 0] == 0x10


@pytest.mark.parametrize("P,N,K", [(1, 128, 128), (2, 256, 128), (1, 128, 256)])
def test_packed_weights_are_a_copy(P, N, K):
    """Also where the product layout is the order that the elements have already."""
    data = torch.zeros(P, N, K // 2, dtype=torch.uint8)
    scales = torch.zeros(P, N, K // 32, dtype=torch.uint8)
    w = ops.pack_mx4_weights(data, scales, swiglu=False)
    data.fill_(1)
    scales.fill_(1)
    assert not w.data.any() and not w.scales.any()


def test_quantize_experts_half_loaded():
    """One projection through the loader, the other not at all: refused before any work."""
    moe = B200MoE.__new__(B200MoE)
    torch.nn.Module.__init__(moe)
    moe.experts_gate_up_mx4, moe._loaded = None, {"down": [None] * 2}
    with pytest.raises(ValueError, match="still to load: down"):
        moe.quantize_mx4()


@pytest.mark.parametrize("P,N,K,swiglu", [(1, 128, 128, False), (2, 256, 128, True), (3, 384, 256, False),
                                          (2, 512, 384, True)])
def test_product_layout_of_weights(P, N, K, swiglu):
    """Every element row and every scale byte is where the header says."""
    g = torch.Generator().manual_seed(N + K)
    data = torch.randint(0, 256, (P, N, K // 2), generator=g, dtype=torch.uint8)
    scales = torch.randint(0, 256, (P, N, K // 32), generator=g, dtype=torch.uint8)
    w = ops.pack_mx4_weights(data, scales, swiglu=swiglu)
    assert w.shape == (P, N, K) and w.scales.shape == (P, K // 128, N // 128, 512)
    half = N // 2
    for row in range(N):
        src = row
        if swiglu:  # gate 0..31, up 0..31, gate 32..63, ...
            src = (row // 64) * 32 + row % 32 + (half if row % 64 >= 32 else 0)
        assert torch.equal(w.data[:, row // 64, :, row % 64].reshape(P, -1), data[:, src])
        for b in range(K // 32):
            r = row % 128
            byte = w.scales[:, b // 4, row // 128, (r % 32) * 16 + (r // 32) * 4 + b % 4]
            assert torch.equal(byte, scales[:, src, b])


def test_pack_refuses():
    d, s = torch.zeros(2, 128, 64, dtype=torch.uint8), torch.zeros(2, 128, 4, dtype=torch.uint8)
    ops.pack_mx4_weights(d, s, swiglu=False)
    for bad in (lambda: ops.pack_mx4_weights(d, s, swiglu=True),                      # I = 64
                lambda: ops.pack_mx4_weights(d[:, :96], s[:, :96], swiglu=False),     # rows
                lambda: ops.pack_mx4_weights(d[..., :32], s[..., :2], swiglu=False),  # K = 64
                lambda: ops.pack_mx4_weights(d, s[..., :3], swiglu=False),
                lambda: ops.pack_mx4_weights(d[0], s[0], swiglu=False)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        ops.pack_mx4_weights(d.int(), s, swiglu=False)


def test_mx8_row_bytes():
    lib = _lib.load()
    for K in (0, 32, 128, 480, 512, 544, 768, 1408, 2048, 14336):
        want = K + -(-(K // 32) // 16) * 16
        assert ops.mx8_row_bytes(K) == want == lib.b200moe_mx8_row_bytes(K)


def _rows(T, K):
    return ops.MX8Rows(torch.zeros(T, ops.mx8_row_bytes(K), dtype=torch.uint8), K)


def _weights(P, N, K, swiglu):
    return ops.pack_mx4_weights(torch.zeros(P, N, K // 2, dtype=torch.uint8),
                                torch.zeros(P, N, K // 32, dtype=torch.uint8), swiglu=swiglu)


HOST_CALLS = {
    "quantize_mx8": lambda: ops.quantize_mx8(torch.zeros(2, 128, dtype=bf)),
    "dequantize_mx8": lambda: ops.dequantize_mx8(_rows(2, 128)),
    "quantize_mx4": lambda: ops.quantize_mx4(torch.zeros(2, 128, dtype=bf)),
    "dequantize_mx4": lambda: ops.dequantize_mx4(torch.zeros(2, 64, dtype=torch.uint8),
                                                 torch.zeros(2, 4, dtype=torch.uint8)),
    "add_rmsnorm_mx8": lambda: ops.add_rmsnorm_mx8(torch.zeros(2, 128, dtype=bf), None, torch.ones(128, dtype=bf)),
    "grouped_swiglu_mx4": lambda: ops.grouped_swiglu_mx4(_rows(2, 128), torch.zeros(2, dtype=torch.int32),
                                                         _weights(1, 256, 128, True)),
    "grouped_down_mx4": lambda: ops.grouped_down_mx4(_rows(2, 128), torch.zeros(2, dtype=torch.int32),
                                                     _weights(1, 128, 128, False)),
    "permute_mx8": lambda: ops.permute_mx8(_rows(2, 128), None, num_slots=1, E1=1),
}


@pytest.mark.parametrize("name", sorted(HOST_CALLS))
def test_mx_ops_refuse_host_tensors(name):
    with pytest.raises(ValueError, match="CUDA tensors only"):
        HOST_CALLS[name]()


def test_c_entry_points_refuse_bad_arguments():
    """Without a device every entry point reports an error code and a message; nothing is
    dereferenced.  (With one, the same calls fail their argument checks.)"""
    lib = _lib.load()
    calls = [
        lambda: lib.b200moe_quantize_mx8(None, 33, 0, 1, 33, None, 64, None),
        lambda: lib.b200moe_dequantize_mx8(None, 48, 1, 32, None, 32, 7, None),
        lambda: lib.b200moe_quantize_mx4(None, 32, 0, -1, 32, None, None, None),
        lambda: lib.b200moe_dequantize_mx4(None, None, 1, 32, None, 32, 0, None),
        lambda: lib.b200moe_add_rmsnorm_mx8(None, None, None, 1e-6, 1, 100, 0, 100, None, None, 0, None, 128, None),
        lambda: lib.b200moe_grouped_swiglu_mx4(None, 144, 1, 0, None, 1, 100, 128, None, None, None, 144, None, None),
        lambda: lib.b200moe_grouped_down_mx4(None, 144, 1, 0, None, 0, 128, 128, None, None, None, 128, 1, None, None,
                                             None),
    ]
    for c in calls:
        assert c() < 0
        assert lib.b200moe_last_error()


def _layer_params(**kw):
    from easyinfra_b200.layer import LayerParams

    E, H, I = 4, 128, 128
    base = dict(gate_w=torch.zeros(E, H, dtype=bf), w_gate_up=_weights(E, 2 * I, H, True), w_down=_weights(E, H, I, False))
    return LayerParams(**dict(base, **kw))


def test_layer_refuses_mixed_weights():
    from easyinfra_b200.layer import MoELayer
    from easyinfra_b200.placement import Placement

    pl = Placement(torch.arange(4).view(1, 4), 4)
    lay = MoELayer(_layer_params(), pl, 2, True)
    assert lay.mx and (lay.H, lay.I) == (128, 128)
    bad = [(_layer_params(w_down=torch.zeros(4, 128, 128, dtype=bf)), {}),
           (_layer_params(gate_w=torch.zeros(4, 128)), {}),
           (_layer_params(), dict(exchange=object())),
           (_layer_params(shared_gate_up=_weights(1, 256, 128, True)), {}),
           (_layer_params(shared_gate_up=_weights(1, 256, 128, True), shared_down=torch.zeros(128, 128, dtype=bf)), {})]
    for p, kw in bad:
        with pytest.raises(ValueError):
            MoELayer(p, pl, 2, True, **kw)


def test_weights_refuse_another_layout():
    w = _weights(2, 256, 128, True)
    for d, s in ((w.data.view(2, 256, 64), w.scales), (w.data, w.scales[:, :, :1]), (w.data.int(), w.scales),
                 (w.data.transpose(1, 2), w.scales), (w.data, w.scales.transpose(0, 1))):
        with pytest.raises(ValueError):
            ops.MX4Weights(d, s, True)


def test_layer_refuses_an_exchange_that_comes_later():
    """The NVLink transport is often attached after the layer was made."""
    from easyinfra_b200.layer import LayerParams, MoELayer
    from easyinfra_b200.placement import Placement

    pl = Placement(torch.arange(4).view(1, 4), 4)
    lay = MoELayer(_layer_params(), pl, 2, True)
    with pytest.raises(ValueError, match="NVLink exchange"):
        lay.exchange = object()
    assert lay.exchange is None
    plain = MoELayer(LayerParams(torch.zeros(4, 128, dtype=bf), torch.zeros(4, 256, 128, dtype=bf),
                                 torch.zeros(4, 128, 128, dtype=bf)), pl, 2, True)
    mark = object()
    plain.exchange = mark
    assert plain.exchange is mark
    plain.exchange = None


LONG = 2 ** 32 + 128  # as an int of 32 bits: 128
LONG_CALLS = {
    "quantize_mx8": lambda: ops.quantize_mx8(torch.zeros(1, 1, dtype=bf).expand(1, LONG)),
    "dequantize_mx8": lambda: ops.dequantize_mx8(ops.MX8Rows(torch.zeros(1, 1, dtype=torch.uint8).expand(
        1, ops.mx8_row_bytes(LONG)), LONG)),
    "quantize_mx4": lambda: ops.quantize_mx4(torch.zeros(1, dtype=bf).expand(LONG)),
    "dequantize_mx4": lambda: ops.dequantize_mx4(torch.zeros(1, dtype=torch.uint8).expand(LONG // 2),
                                                 torch.zeros(1, dtype=torch.uint8).expand(LONG // 32)),
    "add_rmsnorm_mx8 H": lambda: ops.add_rmsnorm_mx8(torch.zeros(1, 1, dtype=bf).expand(1, LONG), None,
                                                     torch.zeros(1, dtype=bf).expand(LONG)),
    "add_rmsnorm_mx8 T": lambda: ops.add_rmsnorm_mx8(torch.zeros(1, 1, dtype=bf).expand(LONG, 128), None,
                                                     torch.zeros(128, dtype=bf)),
}


@pytest.mark.parametrize("name", sorted(LONG_CALLS))
def test_lengths_beyond_31_bits_are_refused(name):
    """They went to the entry points with their low 32 bits: a first part was computed, the rest
    of the output left as it was allocated."""
    with pytest.raises(ValueError, match="above 2.31 - 1"):
        LONG_CALLS[name]()


def test_private_allocation_is_checked_before_use(monkeypatch):
    """Another signature, another result or no such function: the public one is used."""
    on_gpu = type("T", (), dict(shape=(2, 3), dtype=torch.uint8, is_cuda=True, stride=lambda self: (3, 1),
                                get_device=lambda self: 5))
    monkeypatch.setattr(ops, "_current_device", lambda: 5)

    def made(**kw):
        t = type("U", (on_gpu,), kw)()
        return lambda size, stride, dtype: t

    none = lambda: 0  # noqa: E731
    good = made()
    assert ops._checked_empty(good, none) is good
    for bad in (None, lambda size: on_gpu(), lambda size, stride, dtype: torch.empty(size, dtype=dtype), made(shape=(3, 2)),
                made(dtype=torch.int8), made(is_cuda=False), made(stride=lambda self: (1, 2)),
                made(get_device=lambda self: 0)):
        assert ops._checked_empty(bad, none) is None
    for modes in (None, lambda x: 0, lambda: "none"):
        assert ops._checked_empty(good, modes) is None
