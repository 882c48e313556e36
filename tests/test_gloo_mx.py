"""MX8 rows over the collective transport, across real processes on CPU (gloo, world size 2 and
4): MoELayer's own count exchange, plan, dispatch and return, on rows whose bytes are known.
Among them a rank that sends nothing and one that receives nothing."""
from __future__ import annotations

import datetime
import os
import traceback

import numpy as np
import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

from easyinfra_b200 import ops
from easyinfra_b200.communicator import GroupCommunicator
from easyinfra_b200.layer import DispatchState, MoELayer
from tests.test_gloo_ep import _free_port

P, H = 3, 96


def rows_per_slot(world, how):
    """[source, slot] row counts."""
    c = torch.randint(0, 6, (world, world * P), generator=torch.Generator().manual_seed(world))
    if how == "one sends nothing":
        c[world - 1] = 0
    if how == "one receives nothing":
        c[:, :P] = 0
    return c


def sent_by(rank, rows):
    """A rank's send buffer: every byte says whose row it is."""
    g = torch.Generator().manual_seed(100 + rank)
    return torch.randint(0, 256, (rows, ops.mx8_row_bytes(H)), generator=g, dtype=torch.uint8)


def _exchange(rank, world, comm, how):
    counts = rows_per_slot(world, how)
    lay = MoELayer.__new__(MoELayer)
    lay.G, lay.P, lay.H, lay.rank, lay.device, lay.comm = world, P, H, rank, torch.device("cpu"), comm
    mine = sent_by(rank, int(counts[rank].sum()))
    route = ops.RouterOutput(None, None, None, counts[rank].to(torch.int32), None, None, None, None)
    st = DispatchState(T=0, route=route, perm=ops.PermuteOutput(ops.MX8Rows(mine, H), None, None, None))
    got = lay.exchange_counts(st)
    assert np.array_equal(got.reshape(world, world * P), counts.numpy())
    lay.plan_exchange(st, got)
    lay.dispatch(st)
    # rows of every source for this rank's slots, in source order
    parts = []
    for s in range(world):
        a = int(counts[s, :rank * P].sum())
        parts.append(sent_by(s, int(counts[s].sum()))[a:a + int(counts[s, rank * P:(rank + 1) * P].sum())])
    assert st.recv.dtype == torch.uint8 and torch.equal(st.recv, torch.cat(parts))
    assert st.expert_offsets.tolist() == [0] + counts[:, rank * P:(rank + 1) * P].sum(0).cumsum(0).tolist()
    # what returns is bf16 rows, each to its sender and place
    back = lay.combine_exchange(st, st.recv[:, :H].to(torch.bfloat16) + rank)
    owner = torch.repeat_interleave(torch.arange(world * P) // P, counts[rank])
    assert torch.equal(back, mine[:, :H].to(torch.bfloat16) + owner[:, None].to(torch.bfloat16))


def _worker(rank, world, port, q):
    try:
        os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
        dist.init_process_group("gloo", rank=rank, world_size=world, timeout=datetime.timedelta(seconds=60))
        import easyinfra_b200.layer as L
        L.upload_tables = lambda dev, *a: tuple(torch.from_numpy(np.asarray(t).astype(np.int32)) for t in a)
        comm = GroupCommunicator(group=dist.group.WORLD)
        for how in ("all", "one sends nothing", "one receives nothing"):
            _exchange(rank, world, comm, how)
        dist.barrier()
        dist.destroy_process_group()
        q.put((rank, None))
    except Exception:
        q.put((rank, traceback.format_exc()))


@pytest.mark.parametrize("world", [2, 4])
def test_mx8_rows_over_gloo(world):
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    port = _free_port()
    procs = [ctx.Process(target=_worker, args=(r, world, port, q)) for r in range(world)]
    for p in procs:
        p.start()
    res = [q.get(timeout=240) for _ in procs]
    for p in procs:
        p.join(timeout=60)
    for rank, err in res:
        assert err is None, f"rank {rank}: {err}"
