"""attend of the connector's caches with one workspace for a decoding loop whose batch shrinks."""
import pytest
import torch

from tests.test_gpu_attention_ranges import check_rows
from tests.test_gpu_cache_ops import BF16, FMT, attention_case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", ["raw", "e4m3"])
def test_one_workspace_for_a_batch_that_shrinks(cuda_device, fmt):
    from heterofusedkernels_b200.connector import PagedKVCache, QuantizedPagedKVCache

    c = attention_case(fmt, BF16, 1, 8, 128, 16, 1200, [7, 0, 30, 1, 16] * 14, seed=1)
    blocks = len(c["k"])
    cache = PagedKVCache(1, blocks, 16, 1, 128, BF16, cuda_device) if fmt == "raw" else QuantizedPagedKVCache(1, blocks, 16, 1, 128, fmt, cuda_device)
    assert cache.kv_format == FMT[fmt]
    cache.k_caches[0].copy_(c["k"])
    cache.v_caches[0].copy_(c["v"])
    d = {n: c[n].to(cuda_device) for n in ("q", "prefix_table", "tables", "lens")}
    workspace = cache.attend_workspace(d["q"], c["prefix"], d["tables"])
    for n, prefix in ((70, 1200), (65, 1200), (64, 1200), (33, 900), (32, 1200), (5, 1200), (4, 1200), (1, 16)):
        workspace.fill_(0xFF)
        lse = torch.empty(n, 8, device=cuda_device)
        out = cache.attend(0, d["q"][:n], d["prefix_table"], prefix, d["tables"][:n], d["lens"][:n], lse=lse, workspace=workspace)
        part = dict(c, q=c["q"][:n], prefix=prefix, tables=c["tables"][:n], lens=c["lens"][:n])
        check_rows(part, out, lse, torch.ones(n, 8, dtype=torch.bool))
    with pytest.raises(RuntimeError, match="needed"):
        cache.attend(0, d["q"], d["prefix_table"], 1200, d["tables"], d["lens"], workspace=workspace[:workspace.numel() // 64])
    assert cache.status() == 0
