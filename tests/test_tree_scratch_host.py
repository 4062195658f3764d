"""A tree operator's scratch, without a device: a caller's is left alone until the first run, which clears it."""
import contextlib
import ctypes
from types import SimpleNamespace

import torch

from npu_sparse_attn_sharedkv_int8 import PreparedTreeAttention
from tests.test_tree_pages_host import good_tree


def test_a_callers_scratch_is_cleared_by_the_first_run(monkeypatch):
    capturing, seen = [False], []
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing[0])
    monkeypatch.setattr(torch.cuda, "device", lambda index: contextlib.nullcontext())
    buffers = {}

    def allocate(name, shape, dtype, device):
        buffers[name] = torch.full(shape, 7, dtype=dtype)
        return buffers[name]

    op = object.__new__(PreparedTreeAttention)
    op.args, op.out, op.device_index = good_tree(), None, 0
    op.argument_address = ctypes.addressof(op.args)
    op.native = SimpleNamespace(launch=lambda *a: seen.append(op.workspace.count_nonzero().item()))
    op._take_scratch(allocate, torch.device("cpu"))            # a wait for a stream would need a device
    assert op.args.workspace == buffers["tree_workspace"].data_ptr() and (op.workspace == 7).all()
    capturing[0] = True
    op.run()                                                   # a graph that clears each time it is replayed
    op.workspace.fill_(7)
    capturing[0] = False
    op.run()
    op.workspace.fill_(7)
    op.run()                                                   # cleared once; launches leave it zero
    assert seen == [0, 0, op.workspace.numel()]
