"""MX4 experts in the framework's own paths on a B200: the layer (one rank, shared expert,
replicas, emulated expert parallelism), captured stacks, the expert module and the block."""
from __future__ import annotations

import pytest
import torch

from easyinfra_b200 import configs as C
from easyinfra_b200 import ops
from easyinfra_b200.layer import LayerParams, MoELayer, forward_ep_single_device
from easyinfra_b200.placement import Placement
from easyinfra_b200.stack import MoEStack
from oracle import mx_oracle as M

pytestmark = pytest.mark.gpu
bf = torch.bfloat16

QWEN3 = C.small(C.CONFIGS["qwen3"], hidden=256, intermediate=128, num_experts=16, top_k=4, num_layers=1, placement=None)
QWEN15 = C.small(C.CONFIGS["qwen15"], hidden=256, intermediate=128, shared_intermediate=512, num_layers=1)
MIXTRAL = C.small(C.CONFIGS["mixtral"], hidden=512, intermediate=1024, num_layers=1)


def mx4(w, swiglu):
    return ops.pack_mx4_weights(*ops.quantize_mx4(w), swiglu=swiglu)


def make_layer(shape, device, layer=0, shared="bf16", placement=None, rank=0):
    """(MX4 layer, its bf16 weights) of one rank."""
    E = shape.num_experts
    placement = placement or Placement(torch.arange(E).view(1, E), E)
    ids = placement.phy2log[rank].tolist()
    gw = C.router_weight(shape, layer, device)
    gb = C.gate_bias(shape, layer)
    sgu, sd = C.shared_weights(shape, layer, device)
    wgu, wd = C.expert_weights(shape, layer, ids, device)
    if shared == "mx4" and sgu is not None:
        sgu, sd = mx4(sgu[None], True), mx4(sd[None], False)
    g = torch.Generator(device=device)
    g.manual_seed(91 + layer)
    norm = (1 + 0.1 * torch.randn(shape.hidden, generator=g, device=device)).to(bf)
    p = LayerParams(gw, mx4(wgu, True), mx4(wd, False), None if gb is None else gb.to(bf).float().to(device),
                    sgu, sd, norm_weight=norm)
    return MoELayer(p, placement, shape.top_k, shape.norm_topk_prob, rank=rank, shared_gate=shape.shared_gate), (wgu, wd)


def by_hand(lay, residual, hidden):
    """The layer's block view as the separate calls a user would make."""
    p = lay.p
    ro, nm, q = ops.add_rmsnorm_mx8(residual, hidden, p.norm_weight, p.norm_eps)
    r = ops.router(nm, p.gate_w, lay.top_k, renorm=lay.norm_topk_prob, gate_bias=p.gate_bias,
                   has_shared_gate=lay.shared_gate, log2phy=lay.log2phy if lay.use_map else None,
                   rep_count=lay.rep_count if lay.use_map else None, num_slots=lay.G * lay.P)
    perm = ops.permute_mx8(q, r, num_slots=lay.G * lay.P, E1=p.gate_w.shape[0])
    act = ops.grouped_swiglu_mx4(perm.send, r.slot_offsets, p.w_gate_up)
    y = ops.grouped_down_mx4(act, r.slot_offsets, p.w_down)
    shared = None
    if p.shared_gate_up is not None:
        offs = torch.tensor([0, residual.shape[0]], dtype=torch.int32, device=residual.device)
        if isinstance(p.shared_gate_up, ops.MX4Weights):
            shared = ops.grouped_down_mx4(ops.grouped_swiglu_mx4(q, offs, p.shared_gate_up), offs, p.shared_down)
        else:
            shared = ops.grouped_down(ops.grouped_swiglu(nm, offs, p.shared_gate_up[None]), offs, p.shared_down[None])
    out = ops.combine(y, perm.pos_of, r.topk_weights, shared=shared, shared_gate=r.shared_gate)
    return ro, out, dict(r=r, perm=perm, q=q, act=act, y=y, nm=nm)


@pytest.mark.parametrize("T", [1, 5, 8, 9, 64, 333])
@pytest.mark.parametrize("shape,shared", [(QWEN3, "bf16"), (QWEN15, "bf16"), (QWEN15, "mx4"), (MIXTRAL, "bf16")])
def test_layer_is_its_operators(cuda_device, shape, shared, T):
    """forward_block has the bits of the separate calls, and its permuted rows, expert outputs
    and combination are what the routing says."""
    d = cuda_device
    lay, _ = make_layer(shape, d, shared=shared)
    status = torch.zeros(1, dtype=torch.int32, device=d)
    lay.status = status
    res = 2 * C.hidden_states(shape, T, device=d)
    hid = C.hidden_states(shape, T, device=d, seed_offset=1)
    ro, out, v = by_hand(lay, res, hid)
    ro2, out2 = lay.forward_block(res, hid)
    assert torch.equal(ro, ro2) and torch.equal(out, out2)
    assert torch.equal(lay.forward(v["nm"]), out)             # quantises the rows itself
    torch.cuda.synchronize()
    assert int(status.item()) == 0
    # rows moved whole
    K = lay.top_k
    n = ops.mx8_row_bytes(shape.hidden)
    pos = v["perm"].pos_of.long()
    for k in range(K):
        assert torch.equal(v["perm"].send.buf[pos[:, k]], v["q"].buf[:, :n])
    # every routed row against its expert in 64 bits, from the kernel's own activations
    slot = v["r"].phys_ids.long()
    _, byte = v["act"].buf, v["act"].buf[:, v["act"].K:v["act"].K + v["act"].K // 32]
    act = M.values(v["act"].buf[:, :v["act"].K].contiguous(), byte.contiguous(), False)
    wd = ops.dequantize_mx4(*unpack(lay.p.w_down), torch.float32).double()
    for k in range(K):
        a = act[pos[:, k]]
        ref = torch.einsum("ti,thi->th", a, wd[slot[:, k]])
        tot = torch.einsum("ti,thi->th", a.abs(), wd[slot[:, k]].abs())
        err = (v["y"][pos[:, k]].double() - ref).abs()
        assert (err <= 2.0 ** -8 * ref.abs() + 1.04 * a.shape[1] * 2.0 ** -23 * tot).all()


def unpack(w: ops.MX4Weights):
    """(elements [P, rows, K/2], scales [P, rows, K/32]) of weights packed without swiglu."""
    P, N, K = w.shape
    data = w.data.transpose(2, 3).reshape(P, N, K // 2)
    sc = w.scales.view(P, K // 128, N // 128, 32, 4, 4).permute(0, 2, 4, 3, 1, 5).reshape(P, N, K // 32)
    return data, sc.contiguous()


def test_layer_against_the_bf16_layer(cuda_device):
    """The quantised layer's distance from the bf16 one is what the formats allow.  Per
    element, relative: weights 2^-2 of the value at most (e2m1 rounds by half a step of at
    most 2^-1 relative in its normal range, more only below a sixth of the block's largest),
    rows 2^-4 at most.  Rounding errors of different elements are independent, so their sum over H
    and I terms averages out to the root mean square of one element, which is below
    0.15 for normally distributed weights of a block (a step of 2^-1 to 2^-2 of the value,
    uniformly hit: 2^-1.5 / sqrt(12) = 0.10, and the small elements) and 0.03 for the rows: three
    products of such factors, silu's slope at most 1.1: sqrt(3) * 1.1 * 0.16 < 0.31."""
    d = cuda_device
    lay, (wgu, wd) = make_layer(MIXTRAL, d)
    ref = MoELayer(LayerParams(lay.p.gate_w, wgu, wd, lay.p.gate_bias, norm_weight=lay.p.norm_weight), lay.placement,
                   lay.top_k, lay.norm_topk_prob)
    x = C.hidden_states(MIXTRAL, 256, device=d)
    a, b = lay.forward(x).double(), ref.forward(x).double()
    rel = float((a - b).norm() / b.norm())
    print(f"relative distance {rel:.3f}")
    assert 0 < rel < 0.31


def test_replicas_and_emulated_ranks(cuda_device):
    """A placement with replicated experts, as one rank and as four emulated ranks that
    exchange MX8 rows: the same bits, whatever kernel each rank's row count picks."""
    d = cuda_device
    E, G = QWEN3.num_experts, 4
    phy = torch.cat([torch.arange(E), torch.tensor([3, 3, 7, 0])]).view(G, -1)
    whole = Placement(phy.view(1, -1), E)
    split = Placement(phy, E)
    one, _ = make_layer(QWEN3, d, placement=whole)
    ranks = [make_layer(QWEN3, d, placement=split, rank=r)[0] for r in range(G)]
    for T in (3, 40, 700):
        xs = [C.hidden_states(QWEN3, T if r != 2 else 0, rank=r, device=d) for r in range(G)]
        outs = forward_ep_single_device(ranks, xs)
        for x, o in zip(xs, outs):
            assert torch.equal(o, one.forward(x)) and o.shape == x.shape


def test_empty_batch(cuda_device):
    lay, _ = make_layer(QWEN15, cuda_device, shared="mx4")
    x = torch.zeros(0, QWEN15.hidden, dtype=bf, device=cuda_device)
    ro, out = lay.forward_block(x, x)
    assert ro.shape == out.shape == (0, QWEN15.hidden) and lay.forward(x).shape == (0, QWEN15.hidden)


@pytest.mark.parametrize("T", [1, 8, 64])
def test_captured_stacks(cuda_device, T):
    """Two captured stacks replayed in turn, on changing inputs, have the eager bits."""
    d = cuda_device
    stacks = [MoEStack([make_layer(QWEN15, d, layer=i + 10 * j, shared=s)[0] for i in range(3)])
              for j, s in enumerate(("bf16", "mx4"))]
    caps = [s.capture(T) for s in stacks]
    for seed in range(3):
        x = C.hidden_states(QWEN15, T, device=d, seed_offset=seed)
        want = [s.forward(x).clone() for s in stacks]
        got = [c(x).clone() for c in caps]
        for a, b in zip(want, got):
            assert torch.equal(a, b)


def test_products_on_two_streams(cuda_device):
    """Calls of the same weights on two streams at once, each on its own rows."""
    d = cuda_device
    lay, _ = make_layer(MIXTRAL, d)
    E = MIXTRAL.num_experts
    offs = torch.arange(0, 33 * E, 33, dtype=torch.int32, device=d)[:E + 1]
    offs = torch.cat([offs, offs[-1:] + 33])[:E + 1]
    qs = [ops.quantize_mx8(C.hidden_states(MIXTRAL, int(offs[-1]), device=d, seed_offset=i)) for i in range(2)]

    def run(q):
        return ops.grouped_down_mx4(ops.grouped_swiglu_mx4(q, offs, lay.p.w_gate_up), offs, lay.p.w_down)

    want = [run(q) for q in qs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = run(qs[i])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))


@pytest.mark.parametrize("hint", [1, 100, 1000])
def test_operators_in_a_graph(cuda_device, hint):
    """Norm, both quantisations and both products recorded on a side stream and replayed on
    new inputs, against the same calls outside; two graphs of the same weights.  I = 256
    and H = 256 let the hint pick each of the three kernels."""
    d, T, H, I = cuda_device, 130, 256, 256
    g = torch.Generator(device=d).manual_seed(hint)
    wgu = ops.pack_mx4_weights(*ops.quantize_mx4(torch.randn(2, 2 * I, H, generator=g, device=d)), swiglu=True)
    wd = ops.pack_mx4_weights(*ops.quantize_mx4(torch.randn(2, H, I, generator=g, device=d)), swiglu=False)
    weight = torch.ones(H, dtype=bf, device=d)
    offs = torch.tensor([0, 60, T], dtype=torch.int32, device=d)

    def run(res, hid):
        ro, normed, q = ops.add_rmsnorm_mx8(res, hid, weight)
        act = ops.grouped_swiglu_mx4(q, offs, wgu, rows_hint=2 * hint)
        y = ops.grouped_down_mx4(act, offs, wd, rows_hint=2 * hint)
        return ro, normed, y, ops.dequantize_mx8(ops.quantize_mx8(y)), ops.dequantize_mx4(*ops.quantize_mx4(y))

    side, graphs = torch.cuda.Stream(), []
    for _ in range(2):
        ins = [torch.zeros(T, H, dtype=bf, device=d) for _ in range(2)]
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            run(*ins)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs = run(*ins)
        graphs.append((graph, ins, outs))
    for _ in range(2):
        xs = [[torch.randn(T, H, generator=g, device=d).to(bf) for _ in range(2)] for _ in graphs]
        want = [run(*x) for x in xs]
        for (graph, ins, _), x in zip(graphs, xs):
            for a, b in zip(ins, x):
                a.copy_(b)
            graph.replay()
        torch.cuda.synchronize()
        for (_, _, outs), w in zip(graphs, want):
            assert all(torch.equal(a, b) for a, b in zip(outs, w))


def test_permute_refuses_bad_rows(cuda_device):
    d = cuda_device
    lay, _ = make_layer(MIXTRAL, d)
    q = ops.quantize_mx8(C.hidden_states(MIXTRAL, 4, device=d))
    r = lay.route(C.hidden_states(MIXTRAL, 4, device=d))
    E1, n = lay.p.gate_w.shape[0], q.buf.shape[1]
    kw = dict(num_slots=lay.P, E1=E1)
    odd = torch.empty(4, n + 1, dtype=torch.uint8, device=d)
    K = r.phys_ids.shape[1]
    with pytest.raises(ValueError, match="aligned"):
        ops.permute_mx8(ops.MX8Rows(odd, q.K), r, **kw)
    with pytest.raises(ValueError, match="contiguous"):
        ops.permute_mx8(q, r, out=ops.MX8Rows(torch.empty(4 * K, n + 16, dtype=torch.uint8, device=d), q.K), **kw)
    with pytest.raises(ValueError, match="rows"):
        ops.permute_mx8(ops.MX8Rows(q.buf[:3], q.K), r, **kw)


class _Group:
    def __init__(self, size, rank=0):
        self.group_size, self.local_rank = size, rank


def test_expert_module(cuda_device):
    """B200MoE.quantize_mx4: forward is the MX4 products of the quantised weights, rows in
    [source][slot] order; weights are taken once."""
    from easyinfra_b200.experts import B200MoE

    d = cuda_device
    shape, E = MIXTRAL, MIXTRAL.num_experts
    wgu, wd = C.expert_weights(shape, 0, list(range(E)), d)
    for G in (1, 2):
        P = E // G
        m = B200MoE(0, shape.hidden, shape.intermediate, "silu", False, False, E, _Group(G), _Group(1),
                    torch.arange(E).view(G, P), dtype=bf, device=d)
        m.experts_gate_up_weight.copy_(wgu[:P])
        m.experts_down_weight.copy_(wd[:P])
        counts = [(5 * i) % 7 for i in range(G * P)]
        x = C.hidden_states(shape, sum(counts), device=d)
        m.quantize_mx4()
        assert m.experts_gate_up_weight.numel() == 0
        got = m.forward(x, counts)
        gu, dn = mx4(wgu[:P], True), mx4(wd[:P], False)
        row = 0
        for i, c in enumerate(counts):  # each block on its own, as one expert
            offs = torch.tensor([0, c], dtype=torch.int32, device=d)
            e = i % P
            one = [ops.MX4Weights(w.data[e:e + 1], w.scales[e:e + 1], w.swiglu) for w in (gu, dn)]
            if c:
                act = ops.grouped_swiglu_mx4(ops.quantize_mx8(x[row:row + c]), offs, one[0])
                assert torch.equal(got[row:row + c], ops.grouped_down_mx4(act, offs, one[1]))
            row += c
        with pytest.raises(ValueError):
            m.quantize_mx4()
        with pytest.raises(ValueError):
            m.weight_loader("experts", wd[0], bf, "0.down_proj.weight")


def test_block_binds_quantised_experts(cuda_device):
    """The block's stages run on MX4 experts after experts.quantize_mx4(), also when its layer
    was bound before."""
    from types import SimpleNamespace

    from easyinfra_b200.block import B200MoeAll2AllBlock

    d = cuda_device
    shape, E = MIXTRAL, MIXTRAL.num_experts
    blk = B200MoeAll2AllBlock(0, shape.hidden, shape.intermediate, "silu", False, False, E, shape.top_k, True, False,
                              None, _Group(1), _Group(1), False, dtype=bf, device=d)
    wgu, wd = C.expert_weights(shape, 0, list(range(E)), d)
    blk.gate.weight.copy_(C.router_weight(shape, 0, d))
    blk.experts.experts_gate_up_weight.copy_(wgu)
    blk.experts.experts_down_weight.copy_(wd)
    assert not blk.layer().mx
    blk.experts.quantize_mx4()
    lay = blk.layer()
    assert lay.mx
    res, hid = C.hidden_states(shape, 50, device=d), C.hidden_states(shape, 50, device=d, seed_offset=3)
    chunk = SimpleNamespace(active_variables=(res, hid))
    for _, compute, communicate in blk.get_stages():
        compute(chunk)
        communicate(chunk)
    torch.cuda.synchronize()
    residual, out = chunk.active_variables
    lay.p.norm_weight = blk.post_attention_layernorm.weight
    ro, want = lay.forward_block(res, hid)
    assert torch.equal(residual, ro) and torch.equal(out, want)
