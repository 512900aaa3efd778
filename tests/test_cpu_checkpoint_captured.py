"""The backward pass of a checkpoint in 8 bits is refused while a graph is captured, before it launches anything."""

from __future__ import annotations

import pytest
import torch

from moss_offload import kept8


def test_a_backward_pass_that_a_graph_captures_is_refused(monkeypatch) -> None:
    class Gradient:
        is_cuda = True

    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with torch.no_grad(), pytest.raises(RuntimeError, match="captured"):
        kept8._CheckpointFunction.backward(None, Gradient())
