"""The operators' workspace and launch are planned for the operands' device, not for the current one."""

import torch

from kernel_library import _operands


def test_both_calls_see_the_operands_device(monkeypatch):
    current, seen = [0], []

    class Device:
        def __init__(self, device):
            self.index = device.index

        def __enter__(self):
            self.before, current[0] = current[0], self.index

        def __exit__(self, *exc):
            current[0] = self.before

    class Stream:
        cuda_stream = 77

    monkeypatch.setattr(torch.cuda, "current_device", lambda: current[0])
    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device: Stream)
    monkeypatch.setattr(_operands._torch_call, "knows_operators", lambda: True)
    monkeypatch.setattr(torch, "empty", lambda n, dtype, device: (n, device.index))

    def query(arg, need):
        seen.append(("query", arg, current[0]))
        need._obj.value = 64
        return 0

    def run(*args):
        seen.append(("run", args, current[0]))
        return 0

    for index in (0, 1):
        device = torch.device("cuda", index)
        assert _operands.workspace(device, "operator", query, 5) == ((64, index), 64)
        _operands.launch(device, "operator", run, 5, 6)
        assert seen == [("query", 5, index), ("run", (5, 6, 77), index)] and current == [0]
        seen.clear()
