"""The named buffers of an engine: which replacements end a recorded step's life, and how buffers grow."""
import torch

from allpaca_b200.parts import Workspace


def test_only_buffers_that_a_recorded_step_holds_count():
    ws = Workspace(torch.device("cpu"))
    ws.get("a", (4,), torch.float32)
    ws.get("b", (4,), torch.float32)
    ws.get("a", (4,), torch.bfloat16)
    ws.recording = True
    ws.get("a", (2, 2), torch.float32)
    ws.get("a", (4,), torch.float32)                       # (the view that was handed out before)
    ws.recording = False
    before = ws.generation
    ws.get("b", (400,), torch.float32)                     # held by no graph
    ws.get("a", (400,), torch.bfloat16)                    # a buffer of its own
    ws.get("c", (7,), torch.float32)
    ws.get("a", (3,), torch.float32)                       # fits
    assert ws.generation == before
    ws.get("a", (5,), torch.float32)
    assert ws.generation > before
    # one that comes to be while a step is recorded
    ws.recording = True
    ws.get("d", (5,), torch.float32)
    ws.recording = False
    before = ws.generation
    ws.get("d", (6,), torch.float32)
    assert ws.generation > before
