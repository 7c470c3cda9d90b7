"""Mixed batches over E4M3 caches with GQA groups above 16: a decode row then takes two to four 16-row tiles, whose split
pieces are written in tile blocks, and the merge of a mixed batch has to read them so."""

import pytest
import torch

from kvserve_amd import HipAttention, last_launch_kernels, workloads
from oracle import fp8, torch_reference
from tests import paged_check as pc

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads", [(64, 1), (40, 2), (64, 2)], ids=str)
@pytest.mark.parametrize("head_dim", [64, 128])
def test_split_decodes_beside_chunks(hip_device, heads, head_dim):
    w = workloads.custom("wide", [1, 3, 1, 20], [5000, 1200, 64, 300], *heads, head_dim, 16, seed=1)
    b = workloads.materialize(w, torch.bfloat16, hip_device, seed=1)
    kc, vc = (fp8.quantize(x, 0.5).to(hip_device) for x in (b.k_cache, b.v_cache))
    HipAttention.write_kv(kc, vc, b.k_new, b.v_new, b.meta.slot_mapping, 0.5, 0.5)
    out = HipAttention.forward(b.q, kc, vc, b.meta, w.scale, None, 0.5, 0.5)
    assert last_launch_kernels() == ["decode", "prefill", "reduce"]
    m = b.meta
    ref = torch_reference.forward(b.q.float().cpu(), fp8.dequantize(kc.cpu(), 0.5), fp8.dequantize(vc.cpu(), 0.5),
                                  m.block_tables.cpu(), m.seq_lens.cpu(), m.query_lens.cpu(), w.scale)  # fmt: skip
    assert (out.float().cpu() - ref).abs().max().item() <= pc.TOL_16BIT
