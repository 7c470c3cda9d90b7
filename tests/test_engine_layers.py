"""What PagedLlama refuses, and takes, of layers that are no Llama's, when it is built."""

from __future__ import annotations

from dataclasses import replace

import pytest
import torch

from kvserve_amd.attention import HipAttention
from kvserve_amd.engine.model import build_model
from tests.engine_backends import TorchRefAttention
from tests.test_engine_operators import ALL, WindowedTorch


def test_backends_without_windows():
    class Any(WindowedTorch):
        @staticmethod
        def forward(*args, **kw):
            return WindowedTorch.forward(*args, **kw)

    with pytest.raises(ValueError, match="windows"):
        build_model(ALL, "cpu", torch.float32, 64, backend=TorchRefAttention)
    for backend in (WindowedTorch, HipAttention, Any):
        build_model(ALL, "cpu", torch.float32, 64, backend=backend)
    full = replace(ALL, full_layers=tuple(range(ALL.num_layers)))  # no layer has the window
    build_model(full, "cpu", torch.float32, 64, backend=TorchRefAttention)
