"""Windows and documents over a table whose pages before the first visible key were given back (their entries are -1)."""

import pytest
import torch

from tests.paged_reference import KINDS, assert_within, make_cache, page_table, sm_scale, visible
from tests.test_gpu_paged_prefill import product_bits, q_type
from tests.test_gpu_paged_prefill import reference as prefill_reference
from tests.test_gpu_paged_read import bits, reference


def evict(table, firsts, bs):
    """The table with -1 for each sequence's pages that end before its first visible key."""
    kept = table.clone()
    for b, first in enumerate(firsts):
        kept[b, : first // bs] = -1
    return kept.cuda()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("bs", [8, 16, 32, 64])
def test_decode(kind, bs):
    from bpt_b200 import _lib
    from bpt_b200.kernels.kv_attention import attend, decode_attention, merge_partials

    lengths, starts = [500, 77, 1031], [0, 60, 1000]
    g = torch.Generator().manual_seed(bs)
    table, blocks = page_table(lengths, bs, g)
    kv, keys, values = make_cache(kind, blocks, bs, 2, 128, table, g)
    q = torch.randn(3, 6, 128, generator=g)
    n, vmax = torch.tensor(lengths, dtype=torch.int32).cuda(), values.abs().max().item()
    assert _lib.device_error() == 0
    for window, first in ((50, None), (59, starts), (0, starts)):
        kv.block_table = evict(table, [visible(m - 1, m, first[b] if first else 0, window)[0] for b, m in enumerate(lengths)], bs)
        more = {"window": window, "key_starts": None if first is None else torch.tensor(first, dtype=torch.int32).cuda()}
        want = reference(q, keys, values, table, lengths, bs, window, starts=first)
        got = attend(q.cuda(), kv, n, sm_scale(128), **more)
        assert_within(got, want, torch.float32, vmax, bits(kind))
        got = merge_partials(*decode_attention(q.cuda(), kv, n, sm_scale(128), split=128, **more))
        assert_within(got, want, torch.float32, vmax, bits(kind))
        assert _lib.device_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("bs", [8, 16, 32, 64])
@pytest.mark.parametrize("seqs", [[(470, 60), (91, 30)], [(2500, 3)]], ids=["tiles", "parts"])
def test_prefill(kind, bs, seqs):
    from bpt_b200 import _lib
    from bpt_b200.kernels.prefill_attention import prefill_attend

    lengths = [c + n for c, n in seqs]
    g = torch.Generator().manual_seed(bs + 1)
    table, blocks = page_table(lengths, bs, g)
    kv, keys, values = make_cache(kind, blocks, bs, 2, 128, table, g)
    q = torch.randn(sum(n for _, n in seqs), 14, 128, generator=g).to(q_type(kind))
    cu = torch.tensor([0] + [n for _, n in seqs]).cumsum(0).to(torch.int32).cuda()
    n, vmax = torch.tensor(lengths, dtype=torch.int32).cuda(), values.abs().max().item()
    starts = torch.cat([torch.full((new,), ctx - 29, dtype=torch.int32) for ctx, new in seqs])
    assert _lib.device_error() == 0
    for window, first in ((40, None), (1000, None), (0, starts)):
        kv.block_table = evict(table, [visible(c, c + 1, c - 29 if first is not None else 0, window)[0] for c, _ in seqs], bs)
        got = prefill_attend(q.cuda(), kv, cu, n, sm_scale(128), window=window, key_starts=None if first is None else first.cuda())
        want = prefill_reference(q, keys, values, table, seqs, bs, window=window, starts=first)
        assert_within(got, want, q.dtype, vmax, product_bits(kind, q.dtype))
        assert _lib.device_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
def test_a_visible_page_that_is_not_there_is_still_recorded(kind):
    from bpt_b200 import _lib
    from bpt_b200.kernels.kv_attention import attend
    from bpt_b200.kernels.prefill_attention import prefill_attend

    g = torch.Generator().manual_seed(9)
    table, blocks = page_table([200], 8, g)
    kv, _, _ = make_cache(kind, blocks, 8, 2, 128, table, g)
    n, cu = torch.tensor([200], dtype=torch.int32).cuda(), torch.tensor([0, 1], dtype=torch.int32).cuda()
    q = torch.randn(1, 4, 128, generator=g).to(q_type(kind)).cuda()
    kv.block_table = evict(table, [200 - 50 + 8], 8)  # the page of the first visible key too
    assert _lib.device_error() == 0
    attend(q, kv, n, sm_scale(128), window=50)
    assert _lib.device_error() == 2
    prefill_attend(q, kv, cu, n, sm_scale(128), window=50)
    assert _lib.device_error() == 2
