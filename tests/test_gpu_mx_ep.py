"""MX4 experts over the collective transport on a GPU: MoELayer.forward_block and the block's
stages with more than one rank, rows moving as bytes through all_to_all_single.

On one GPU the ranks are threads whose communicator hands tensors over on the host: a rank's
kernels wait for events of copies that were launched before, never for another rank's kernel.
With two GPUs the same runs as processes over NCCL.  Every output has the bits of the same
layer on one rank."""
from __future__ import annotations

import datetime
import os
import threading
import traceback
from types import SimpleNamespace as NS

import pytest
import torch
import torch.multiprocessing as mp

from easyinfra_b200 import configs as C
from easyinfra_b200 import ops
from easyinfra_b200.block import B200MoeAll2AllBlock
from easyinfra_b200.communicator import WorkHandler
from easyinfra_b200.layer import LayerParams, MoELayer
from easyinfra_b200.placement import Placement
from tests.chunk_protocol import load_trace, run_layers

pytestmark = pytest.mark.gpu
bf = torch.bfloat16
QWEN3 = C.small(C.CONFIGS["qwen3"], hidden=256, intermediate=128, num_experts=16, top_k=4, num_layers=1, placement=None)
QWEN15 = C.small(C.CONFIGS["qwen15"], hidden=256, intermediate=128, shared_intermediate=512, num_layers=1)


class ThreadGroup:
    """What ranks in threads of one process share."""

    def __init__(self, size):
        self.size, self.slots = size, [None] * size
        self.barrier = threading.Barrier(size, timeout=60)

    def swap(self, rank, mine, take):
        """Every rank's `mine`, given to take(rank, of all); inputs stay until all have taken."""
        stream, ready, done = torch.cuda.current_stream(), torch.cuda.Event(), torch.cuda.Event()
        ready.record(stream)
        self.slots[rank] = (mine, ready, done)
        self.barrier.wait()
        everyone = list(self.slots)
        for _, ev, _ in everyone:
            stream.wait_event(ev)
        take([m for m, _, _ in everyone])
        done.record(stream)
        self.barrier.wait()
        for _, _, ev in everyone:
            stream.wait_event(ev)


class ThreadComm:
    """GroupCommunicator's calls for one rank of a ThreadGroup."""

    def __init__(self, shared, rank):
        self.shared, self.local_rank, self.group_size = shared, rank, shared.size

    def all_gather_into_tensor(self, out, t, dim=0, async_op=False):
        self.shared.swap(self.local_rank, t, lambda all_: out.copy_(torch.cat(all_)))
        return WorkHandler(out)

    def all_to_all_single(self, out, t, out_splits=None, in_splits=None, async_op=False):
        def take(all_):
            at = 0
            for (src, splits), n in zip(all_, out_splits):
                a = sum(splits[:self.local_rank])
                assert splits[self.local_rank] == n
                out[at:at + n] = src[a:a + n]
                at += n
            assert at == out.shape[0]
        assert sum(in_splits) == t.shape[0] and t.dtype == out.dtype and t.shape[1:] == out.shape[1:]
        self.shared.swap(self.local_rank, (t, in_splits), take)
        return WorkHandler(out)


def on_ranks(size, fn):
    """[fn(rank, communicator) of every rank], each in a thread of its own."""
    shared, res, errs = ThreadGroup(size), [None] * size, []

    def go(r):
        try:
            res[r] = fn(r, ThreadComm(shared, r))
        except Exception:
            errs.append((r, traceback.format_exc()))
            shared.barrier.abort()

    ts = [threading.Thread(target=go, args=(r,)) for r in range(size)]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    assert not errs, "\n".join(f"rank {r}:\n{e}" for r, e in errs)
    torch.cuda.synchronize()
    return res


def mx4(w, swiglu):
    return ops.pack_mx4_weights(*ops.quantize_mx4(w), swiglu=swiglu)


def make_layer(shape, placement, rank, device, comm=None, shared="bf16", first_half=False):
    gb = C.gate_bias(shape, 0)
    gb = None if gb is None else gb.to(bf).float().to(device)
    if first_half:  # no token goes to an expert of the second half
        gb = torch.zeros(shape.num_experts, device=device)
        gb[shape.num_experts // 2:] = -1e4
    sgu, sd = C.shared_weights(shape, 0, device)
    if shared == "mx4" and sgu is not None:
        sgu, sd = mx4(sgu[None], True), mx4(sd[None], False)
    wgu, wd = C.expert_weights(shape, 0, placement.phy2log[rank].tolist(), device)
    p = LayerParams(C.router_weight(shape, 0, device), mx4(wgu, True), mx4(wd, False), gb, sgu, sd)
    return MoELayer(p, placement, shape.top_k, shape.norm_topk_prob, rank=rank, comm=comm, shared_gate=shape.shared_gate)


def inputs(shape, T, rank, device):
    return (2 * C.hidden_states(shape, T, rank=rank, device=device),
            C.hidden_states(shape, T, rank=rank, device=device, seed_offset=1))


def run_rank(shape, phy2log, rank, comm, device, Ts, shared, first_half):
    """forward_block, twice, and forward of one rank's tokens."""
    lay = make_layer(shape, Placement(phy2log, shape.num_experts), rank, device, comm, shared, first_half)
    res, hid = inputs(shape, Ts[rank], rank, device)
    a = lay.forward_block(res, hid)
    b = lay.forward_block(res, hid)
    assert all(torch.equal(u, v) for u, v in zip(a, b))
    x = C.hidden_states(shape, Ts[rank], rank=rank, device=device, seed_offset=2)
    return *a, lay.forward(x)


def on_one_rank(shape, phy2log, device, Ts, shared, first_half):
    one = make_layer(shape, Placement(phy2log.reshape(1, -1), shape.num_experts), 0, device, None, shared, first_half)
    return [(*one.forward_block(*inputs(shape, T, r, device)),
             one.forward(C.hidden_states(shape, T, rank=r, device=device, seed_offset=2))) for r, T in enumerate(Ts)]


SLOTS = torch.cat([torch.arange(16), torch.tensor([3, 3, 7, 0])])  # replicas among the slots
LAYERS = [  # shape, slots, tokens of every rank, shared expert, all tokens to the first half of the experts
    (QWEN3, SLOTS.view(2, -1), (40, 40), "bf16", False),
    (QWEN3, SLOTS.view(2, -1), (1, 1), "bf16", False),
    (QWEN3, SLOTS.view(4, -1), (700, 0, 9, 64), "bf16", False),
    (QWEN3, torch.arange(16).view(2, -1), (33, 5), "bf16", True),      # rank 1 receives nothing
    (QWEN3, torch.arange(16).view(2, -1), (0, 17), "bf16", True),      # and rank 0 sends nothing
    (QWEN15, torch.arange(60).view(2, -1), (12, 130), "bf16", False),
    (QWEN15, torch.arange(60).view(4, -1), (6, 0, 50, 3), "mx4", False),
]


@pytest.mark.parametrize("case", LAYERS)
def test_layer_over_a_communicator(cuda_device, case):
    shape, phy2log, Ts, shared, first_half = case
    got = on_ranks(len(Ts), lambda r, comm: run_rank(shape, phy2log, r, comm, cuda_device, Ts, shared, first_half))
    for g, w in zip(got, on_one_rank(shape, phy2log, cuda_device, Ts, shared, first_half)):
        assert all(torch.equal(a, b) for a, b in zip(g, w))


def make_blocks(device, ep_group, rank, n_layers=2):
    E, H, I = QWEN3.num_experts, QWEN3.hidden, QWEN3.intermediate
    blocks = []
    for layer in range(n_layers):
        blk = B200MoeAll2AllBlock(layer, H, I, "silu", False, False, E, QWEN3.top_k, True, False, None, ep_group,
                                  NS(group_size=1, local_rank=0), False, dtype=bf, device=device)
        P = blk.num_physical_experts
        wgu, wd = C.expert_weights(QWEN3, layer, list(range(rank * P, (rank + 1) * P)), device)
        with torch.no_grad():
            blk.gate.weight.copy_(C.router_weight(QWEN3, layer, device))
            blk.experts.experts_gate_up_weight.copy_(wgu)
            blk.experts.experts_down_weight.copy_(wd)
        blk.experts.quantize_mx4()
        blocks.append(blk)
    return blocks


def run_block(blk, res, hid):
    chunk = NS(active_variables=(res, hid))
    for _, compute, communicate in blk.get_stages():
        compute(chunk)
        communicate(chunk)
    torch.cuda.synchronize()
    return chunk.active_variables


def block_rank(rank, comm, device, scenario):
    """Two chunks over two layers, in the recorded order of stages, waits and records."""
    blocks = make_blocks(device, comm, rank)
    ins = [(C.hidden_states(QWEN3, T, rank=rank, seed_offset=10 + c),
            C.hidden_states(QWEN3, T, rank=rank, seed_offset=20 + c)) for c, T in enumerate((48, 5))]
    return run_layers(load_trace(scenario), blocks, ins, device)


def check_blocks(device, seen_of_ranks):
    alone = make_blocks(device, NS(group_size=1, local_rank=0), 0)
    for seen in seen_of_ranks:
        for layers in seen:
            for blk, (res_in, hid_in, res_out, hid_out) in zip(alone, layers):
                ro, out = run_block(blk, res_in.to(device), hid_in.to(device))
                assert torch.equal(ro.cpu(), res_out) and torch.equal(out.cpu(), hid_out)


@pytest.mark.parametrize("scenario", ["direct_ep2", "pools_ep2"])
def test_block_over_a_communicator(cuda_device, scenario):
    check_blocks(cuda_device, on_ranks(2, lambda r, comm: block_rank(r, comm, cuda_device, scenario)))


# ------------------------------------------------------------------ two GPUs
def _nccl_rank(rank, world, port, q):
    import torch.distributed as dist
    try:
        os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port), NCCL_NVLS_ENABLE="0")
        torch.cuda.set_device(rank)
        dev = torch.device("cuda", rank)
        dist.init_process_group("nccl", rank=rank, world_size=world, timeout=datetime.timedelta(seconds=120),
                                device_id=dev)
        from easyinfra_b200.communicator import GroupCommunicator
        comm = GroupCommunicator(group=dist.group.WORLD)
        for shape, phy2log, Ts, shared, first_half in LAYERS:
            if len(Ts) != world:
                continue
            got = run_rank(shape, phy2log, rank, comm, dev, Ts, shared, first_half)
            want = on_one_rank(shape, phy2log, dev, Ts, shared, first_half)[rank]
            assert all(torch.equal(a, b) for a, b in zip(got, want))
        for scenario in ("direct_ep2", "pools_ep2"):
            check_blocks(dev, [block_rank(rank, comm, dev, scenario)])
        dist.barrier(device_ids=[rank])
        dist.destroy_process_group()
        q.put((rank, None))
    except Exception:
        q.put((rank, traceback.format_exc()))


def test_two_gpus_over_nccl():
    if not torch.cuda.is_available() or torch.cuda.device_count() < 2:
        pytest.skip("needs 2 GPUs")
    from tests.test_gloo_ep import _free_port

    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    port = _free_port()
    procs = [ctx.Process(target=_nccl_rank, args=(r, 2, port, q)) for r in range(2)]
    for p in procs:
        p.start()
    res = [q.get(timeout=600) for _ in procs]
    for p in procs:
        p.join(timeout=120)
    for rank, err in res:
        assert err is None, f"rank {rank}: {err}"
