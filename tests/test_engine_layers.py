"""What PagedLlama refuses, and takes, of layers that are no Llama's, when it is built."""

from __future__ import annotations

from dataclasses import replace

import pytest
import torch

from kvserve_amd.attention import HipAttention
from kvserve_amd.engine.model import PagedLlama, build_model, random_weights
from kvserve_amd.engine.runner import ModelRunner
from kvserve_amd.linear4 import quantize_weight4
from tests.engine_backends import TorchRefAttention
from tests.test_engine_operators import ALL, POOLS, STEPS, WindowedTorch, _error, _model, _run


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


@pytest.mark.parametrize("rotary", [-2, 31, 66])
def test_rotated_elements(rotary):
    with pytest.raises(ValueError, match="rotary_dim"):
        build_model(replace(ALL, rotary_dim=rotary), "cpu", torch.float32, 64, backend=WindowedTorch)


def test_norms_of_config_and_weights():
    """Norms that one of the two lacks would be left out, or taken, without a word."""
    plain = replace(ALL, qk_norm=False)
    for cfg, of in ((ALL, plain), (plain, ALL)):
        with pytest.raises(ValueError, match="norms"):
            PagedLlama(cfg, random_weights(of, "cpu", torch.float32), WindowedTorch)
    w = random_weights(ALL, "cpu", torch.float32)
    w.layers[-1].k_norm = None
    with pytest.raises(ValueError, match="norms"):
        PagedLlama(ALL, w, WindowedTorch)


def test_rotations_that_the_kernel_does_not_take():
    """Pairs that are no multiple of 8 go step by step, unless the fused kernel is asked for."""
    cfg = replace(ALL, rotary_dim=24)
    assert not build_model(cfg, "cpu", torch.float32, 64).fused_rope and build_model(ALL, "cpu", torch.float32, 64).fused_rope
    with pytest.raises(ValueError, match="fused"):
        build_model(cfg, "cpu", torch.float32, 64, fused_rope=True)


@pytest.mark.gpu
def test_rotations_step_by_step(hip_device):
    cfg = replace(ALL, rotary_dim=24)
    model = _model(cfg, hip_device, torch.bfloat16, HipAttention)
    assert _error(model, _run(ModelRunner(model, num_blocks=96, max_model_len=256), cfg)) < POOLS["bf16"][1]


@pytest.mark.gpu
def test_gate_rows_that_fill_no_tile(hip_device):
    """An MLP of 648: 40.5 tiles of gate rows, which linear4_silu_mul does not take."""
    cfg = replace(ALL, intermediate_size=648)
    model = _model(cfg, hip_device, torch.bfloat16, HipAttention)
    for lw in model.w.layers:
        lw.w_gate_up = quantize_weight4(lw.w_gate_up, 128)
    errs = [_error(model, _run(ModelRunner(model, num_blocks=96, max_model_len=256, decode_graphs=g), cfg)) for g in (False, True)]
    assert max(errs) < POOLS["bf16"][1], errs


NEAR = [
    {"sliding_window": 23}, {"sliding_window": 25}, {"attention_sinks": 2}, {"attention_sinks": 4}, {"full_layers": ()},
    {"full_layers": (1, 2)}, {"full_layers": (0,)}, {"rotary_dim": 48}, {"rope_interleaved": False},
]  # fmt: skip


@pytest.mark.gpu
@pytest.mark.parametrize("pool", POOLS)
def test_no_other_layers_are_nearer(hip_device, pool):
    """The logits are nearer to the 64-bit model of their own config than to any that differs by one key of a window, one
    sink, one layer or the rotation, over prompts that a window leaves keys out of: whatever the errors, a model that
    computed one of the others would be nearer to that."""
    dtype, _ = POOLS[pool]
    model = _model(ALL, hip_device, torch.bfloat16, HipAttention, 128)
    got = [g for g in _run(ModelRunner(model, num_blocks=96, max_model_len=256, kv_cache_dtype=dtype), ALL)
           if len(g[0]) > ALL.sliding_window + ALL.attention_sinks + STEPS]  # fmt: skip
    assert len(got) == 2
    own = _error(model, got, dtype)
    for over in NEAR:
        model.cfg = replace(ALL, **over)
        assert own < _error(model, got, dtype), over
