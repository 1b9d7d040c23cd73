"""The launch arguments of `attend`: those that it has, and names that it has not."""

import pytest
import torch

from tests.paged_reference import make_cache, page_table


@pytest.mark.parametrize("kind", ["fp8", "bf16"])
@pytest.mark.parametrize("name", ["windows", "soft_cap", "alibi", "pld"])
def test_a_name_that_attend_does_not_have_is_refused(kind, name):
    """(no kernel runs: the call is refused before its tensors are looked at)"""
    from bpt_b200.kernels.kv_attention import PagedQuantKV, attend

    pool = torch.zeros(2, 16, 2, 64, dtype=torch.uint8 if kind == "fp8" else torch.bfloat16)
    kv = PagedQuantKV(kind, pool, pool, torch.zeros(1, 2, dtype=torch.int32), 16)
    with pytest.raises(TypeError, match=name):
        attend(torch.zeros(1, 4, 64), kv, torch.ones(1, dtype=torch.int32), 1.0, **{name: 3})


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["fp8", "bf16"])
def test_the_launch_arguments_that_attend_has(kind):
    """`kv_ready`, a promise, and `num_warps`, which only the reference's kernels read, change nothing."""
    from bpt_b200.kernels.kv_attention import attend

    g = torch.Generator().manual_seed(1)
    table, blocks = page_table([300, 20], 16, g)
    kv, _, _ = make_cache(kind, blocks, 16, 2, 128, table, g)
    q, n = torch.randn(2, 8, 128, generator=g).to(torch.bfloat16).cuda(), torch.tensor([300, 20], dtype=torch.int32).cuda()
    want = attend(q, kv, n, 0.1)
    assert torch.equal(want, attend(q, kv, n, 0.1, tokens=304, split=None, num_warps=4, pdl=True, kv_ready=True))
