"""A step that the paged cache refuses leaves its pages as they were."""

from types import SimpleNamespace

import pytest
import torch

from tests.paged_reference import KINDS


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_rotate_and_attend_refuses_before_it_stores(kind, dtype):
    """Several tokens take 16-bit queries, over 16-bit pages of their own dtype; a single token any of the three."""
    from bpt_b200.integration import PagedQuantizedKVCache
    from bpt_b200.kernels.kv_write import rope_table

    cache = PagedQuantizedKVCache(SimpleNamespace(num_layers=1, num_kv_heads=2, head_dim=64), num_blocks=4, kind=kind)
    cache.reserve("a", 20)
    cos, sin = rope_table(32, 64, 1e4)
    g = torch.Generator().manual_seed(1)
    taken = {"bf16": (torch.bfloat16,), "f16": (torch.float16,)}.get(kind, (torch.float16, torch.bfloat16))
    for n in (5, 1):
        q, k, v = (torch.randn(1, h, n, 64, generator=g).to(dtype).cuda() for h in (4, 2, 2))
        meta = cache.prepare(["a"], torch.arange(n)[None].cuda())
        before = [p.clone() for p in (cache.layers[0].k_pool, cache.layers[0].v_pool)]
        if n == 1 or dtype in taken:
            assert cache.rotate_and_attend(0, q, k, v, meta, 0.125, cos, sin).dtype == dtype
            continue
        with pytest.raises(ValueError, match="queries of"):
            cache.rotate_and_attend(0, q, k, v, meta, 0.125, cos, sin)
        for pool, old in zip((cache.layers[0].k_pool, cache.layers[0].v_pool), before, strict=True):
            assert torch.equal(pool, old)
