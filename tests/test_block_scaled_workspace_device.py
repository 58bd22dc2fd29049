"""The workspace of the block-scaled attention is sized on the query's device,
whichever is current (a stand-in for the device's switch: no GPU needed)."""

import contextlib

import torch


class _Query:
    shape, dtype = (4, 8, 128), torch.bfloat16

    def __init__(self, device):
        self.device_index = device

    def get_device(self):
        return self.device_index


def test_sized_on_the_querys_device(cflib, monkeypatch):
    from cacheflow_b200 import ops

    entered, current = [], [0]

    @contextlib.contextmanager
    def switch(d):
        entered.append(d)
        current[0], old = d, current[0]
        yield
        current[0] = old

    class Lib:
        seen = []

        @staticmethod
        def cf_paged_attention_fp8_block_workspace_size(_):
            Lib.seen.append(current[0])
            return 4096 * (1 + current[0])

    monkeypatch.setattr(torch.cuda, "device", switch)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: current[0])
    monkeypatch.setattr(ops._lib, "load", lambda: Lib)
    cache, tables = torch.zeros(8, 2, 16, 128, dtype=torch.uint8), torch.zeros(4, 64, dtype=torch.int32)
    size = ops.paged_attention_fp8_block_workspace_size
    assert size(_Query(1), cache, tables, 1000) == 8192 and entered == [1]
    assert size(_Query(0), cache, tables, 1000) == 4096 and entered == [1]
    assert size(_Query(-1), cache, tables, 1000) == 4096 and entered == [1]  # not on a GPU: as the current one
    assert Lib.seen == [1, 0, 0] and current == [0]
