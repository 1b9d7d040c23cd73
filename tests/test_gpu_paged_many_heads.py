"""Numbers of heads that the kernels for 8-bit codes cannot hold at a head size of 256."""

import pytest
import torch

from tests.paged_reference import assert_within, attention_row, make_cache, page_table


@pytest.mark.parametrize("heads,any_format", [(8, False), (12, False), (13, True), (16, True), (17, True)])
@pytest.mark.parametrize("kind", ["fp8", "int8"])
def test_heads_of_256_that_the_8_bit_kernels_cannot_hold_are_routed(kind, heads, any_format):
    """Two stages of 16 keys and values of 13 heads of 256 pass the 200 KB of shared memory that those kernels take."""
    from bpt_b200.kernels.kv_attention import PagedQuantKV, _any_format

    pool = torch.zeros(1, 16, heads, 256, dtype=torch.uint8)
    kv = PagedQuantKV(kind, pool, pool, torch.zeros(1, 1, dtype=torch.int32), 16)
    assert _any_format(torch.zeros(1, heads, 256), kv, 0.0, 0, None, None) is any_format


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["fp8", "int8"])
@pytest.mark.parametrize("hq,hkv", [(12, 12), (13, 13), (32, 16)])
def test_many_heads_of_256(kind, hq, hkv):
    from bpt_b200.kernels.kv_attention import attend, decode_attention, merge_partials

    g = torch.Generator().manual_seed(hq)
    lengths = [70, 0, 33]
    table, blocks = page_table(lengths, 16, g)
    kv, keys, values = make_cache(kind, blocks, 16, hkv, 256, table, g)
    q, n = torch.randn(3, hq, 256, generator=g), torch.tensor(lengths, dtype=torch.int32).cuda()
    k, v = ([x[table[b, : max(1, -(-m // 16))].long()].flatten(0, 1) for b, m in enumerate(lengths)] for x in (keys, values))
    want = torch.stack([attention_row(q[b].double(), k[b], v[b], m - 1, 0, m, 1 / 16) for b, m in enumerate(lengths)])
    for got in (attend(q.cuda(), kv, n, 1 / 16), merge_partials(*decode_attention(q.cuda(), kv, n, 1 / 16))):
        assert_within(got, want, torch.float32, values.abs().max().item(), 11)
