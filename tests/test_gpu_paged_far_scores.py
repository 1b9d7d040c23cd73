"""Scores so large that fp32 holds only every second or fourth whole number: the largest one's key is the output."""

import pytest
import torch

from tests.paged_reference import DTYPES, KINDS, make_cache, page_table


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("factor", [2.0**10, 2.0**20, 2.0**24, -(2.0**20)])
@pytest.mark.parametrize("lengths", [[900], [33, 700, 5]], ids=["one", "three"])
def test_scores_beyond_24_bits(kind, factor, lengths):
    """The scores differ by far more than their rounding (N(0, D) times the factor), so all of the probability is on one key;
    what comes out is its value.

    Tolerance: half a step of the output's type, and the rounding of that one probability in the product, 8 (bf16 prefill) or
    11 bits: in the prefill it is 2^(rounding of the largest score), not 1. The prefill takes scores below 2^27 (at 2^24 times
    N(0, D) they pass 2^30)."""
    from bpt_b200.kernels.kv_attention import attend, decode_attention, merge_partials
    from bpt_b200.kernels.prefill_attention import prefill_attend

    g = torch.Generator().manual_seed(len(lengths))
    table, blocks = page_table(lengths, 16, g)
    kv, keys, values = make_cache(kind, blocks, 16, 2, 128, table, g)
    q = torch.randn(len(lengths), 4, 128, generator=g).to(DTYPES.get(kind, torch.bfloat16))
    want = torch.zeros(len(lengths), 4, 128, dtype=torch.float64)
    for b, n in enumerate(lengths):
        k, v = (x[table[b, : -(-n // 16)].long()].flatten(0, 1)[:n].repeat_interleave(2, dim=1) for x in (keys, values))
        s = torch.einsum("hd,nhd->hn", q[b].double(), k) * factor
        first, second = s.topk(2, dim=-1).values.unbind(-1)
        assert ((first - second) > 40 + 2.0**-20 * s.abs().amax(-1)).all()
        want[b] = v[s.argmax(-1), torch.arange(4)]
    n, cu = torch.tensor(lengths, dtype=torch.int32).cuda(), torch.arange(len(lengths) + 1, dtype=torch.int32).cuda()
    outs = [(attend(q.cuda(), kv, n, factor, window=1 << 20), 11),
            (merge_partials(*decode_attention(q.cuda(), kv, n, factor, window=1 << 20, split=128)), 11)]
    if abs(factor) < 2.0**24:
        outs.append((prefill_attend(q.cuda(), kv, cu, n, factor), 8 if kind == "bf16" else 11))
    for got, bits in outs:
        half = torch.finfo(got.dtype).eps / 2
        assert ((got.double().cpu() - want).abs() <= (half + 2.0**-bits) * want.abs()).all()
