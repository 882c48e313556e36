"""What a captured stack and a workspace have to keep: a graph replays on the addresses that
it recorded, so the memory behind them must outlive it.  Without a GPU: the recording is
replaced, and weak references tell what is still held."""
from __future__ import annotations

import contextlib
import gc
import weakref
from types import SimpleNamespace as NS

import torch

from easyinfra_b200 import ops
from easyinfra_b200.stack import MoEStack


class _Layer:
    """A layer that writes into the buffers it is given, as MoELayer.forward_block does."""
    G, exchange, H, device = 1, None, 8, torch.device("cpu")

    def __init__(self, seen):
        self.seen = seen
        self.p = NS(gate_w=torch.zeros(2, 8))

    def forward_block(self, residual, hidden, out=None, residual_out=None):
        self.seen += [weakref.ref(out), weakref.ref(residual_out)]
        return residual_out.copy_(residual), out.copy_(residual)


def _without_gpu(monkeypatch):
    stream = NS(wait_stream=lambda other: None)
    monkeypatch.setattr(torch.cuda, "Stream", lambda device=None: stream)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: stream)
    monkeypatch.setattr(torch.cuda, "stream", lambda s: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "synchronize", lambda device=None: None)
    monkeypatch.setattr(torch.cuda, "CUDAGraph", lambda: NS(replay=lambda: None))
    monkeypatch.setattr(torch.cuda, "graph", lambda g, **kw: contextlib.nullcontext())
    monkeypatch.setattr(ops, "add_rmsnorm", lambda r, h, w, residual_out=None, norm=True: residual_out.copy_(r + h))


def test_captured_stack_keeps_what_it_recorded(monkeypatch):
    """The stack may go out of scope after capture(): its buffers and layers are the graph's."""
    _without_gpu(monkeypatch)
    seen = []
    layer = _Layer(seen)
    held = weakref.ref(layer)
    cap = MoEStack([layer]).capture(3)
    del layer
    gc.collect()
    assert seen and all(r() is not None for r in seen) and held() is not None
    out = weakref.ref(cap.output)
    del cap
    gc.collect()
    assert held() is None and out() is None and all(r() is None for r in seen)


def test_workspace_keeps_what_it_outgrew():
    """A graph that was captured with a small batch's workspace replays on it after a larger
    batch has made the workspace grow."""
    ws = ops.Workspace(torch.device("cpu"))
    first = ws.get(100)
    ref, at = weakref.ref(first), first.data_ptr()
    del first
    again = ws.get(64)
    assert again.data_ptr() == at                                      # large enough: the same one
    del again
    for n in (101, 1000, 100000):
        assert ws.get(n).numel() >= n
    gc.collect()
    assert ref() is not None and ref().data_ptr() == at
    held = sum(b.numel() for b in ws.outgrown)
    assert held <= ws.buf.numel()
