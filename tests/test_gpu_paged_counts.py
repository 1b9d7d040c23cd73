"""Every visible key counts once: keys of zeros give every score the same value, and values with a single one at dim
(j + h) mod D make the output the number of keys of each residue over their count, so one key lost or taken twice at the edge
of a page, step, part or window moves an output by its whole share.

Tolerance: the powers (1), their products with the values and the sums of both are whole numbers times one power of two (INT8:
times one f16 scale) that fp32 holds exactly. What is left are the division, the factors that join parts, 2^x of differences of
base-2 logarithms below 16 (their rounding 2^-20 at most, 2^x itself 2^-22), and half a step of the output's type: 2^-18
relative beside that half step."""

import pytest
import torch

from tests.paged_reference import DTYPES, KINDS, page_table, sm_scale, tolerance, visible
from tests.test_gpu_paged_prefill import case, product_bits, reference


def counting_cache(kind, lengths, bs, hkv, d, g):
    """A cache of the sequences above, anything else in the pool far off; and the value of a one."""
    from bpt_b200.kernels.kv_attention import PagedQuantKV

    table, blocks = page_table(lengths, bs, g)
    values = torch.full((blocks, bs, hkv, d), 100.0)
    for b, n in enumerate(lengths):
        j = torch.arange(n)
        for h in range(hkv):
            values[table[b, j // bs].long(), j % bs, h] = torch.nn.functional.one_hot((j + h) % d, d).float()
    keys, scales, one = torch.zeros_like(values), (1.0, 1.0), 1.0
    if kind in DTYPES:
        pools = [x.to(DTYPES[kind]) for x in (keys, values)]
    elif kind == "fp8":
        pools, scales = [(x * 64).clamp(max=448).to(torch.float8_e4m3fn).view(torch.uint8) for x in (keys, values)], (1 / 64, 1 / 64)
    else:
        s = torch.full((blocks, bs, hkv), 1 / 127, dtype=torch.float16)
        pools, scales, one = [(x * 127).clamp(max=127).to(torch.int8) for x in (keys, values)], (s.cuda(), s.cuda()), 127 * float(s[0, 0, 0])
    return PagedQuantKV(kind, pools[0].cuda(), pools[1].cuda(), table.cuda(), bs, *scales), one


def counts(lo, hi, hq, hkv, d, one):
    if hi <= lo:
        return torch.zeros(hq, d, dtype=torch.float64)
    heads = [torch.bincount((torch.arange(lo, hi) + h) % d, minlength=d).double() * (one / (hi - lo)) for h in range(hkv)]
    return torch.stack(heads).repeat_interleave(hq // hkv, dim=0)


def check(got, want):
    half = 0.0 if got.dtype == torch.float32 else torch.finfo(got.dtype).eps / 2
    off = (got.double().cpu() - want).abs() - want * (half + 2.0**-18)
    assert not torch.isnan(off).any() and (off <= 0).all(), f"{off.max().item():.3g} over at {off.flatten().argmax().item()}"


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("d,bs", [(64, 16), (128, 8), (128, 64), (256, 16)])
@pytest.mark.parametrize("lengths", [[4099], [1, 15, 16, 17, 127, 128, 129, 1000, 2311], list(range(1, 2000, 31))],
                         ids=["one", "nine", "many"])
def test_decode(kind, d, bs, lengths):
    from bpt_b200.kernels.kv_attention import attend, decode_attention, merge_partials

    g = torch.Generator().manual_seed(d)
    kv, one = counting_cache(kind, lengths, bs, 2, d, g)
    q, n = torch.randn(len(lengths), 6, d, generator=g).cuda(), torch.tensor(lengths, dtype=torch.int32).cuda()
    for window in (1 << 20, 777, 1):
        want = torch.stack([counts(*visible(m - 1, m, window=window), 6, 2, d, one) for m in lengths])
        check(attend(q, kv, n, sm_scale(d), window=window), want)
        check(attend(q, kv, n, sm_scale(d), window=window, softcap=20.0), want)
        check(merge_partials(*decode_attention(q, kv, n, sm_scale(d), window=window, split=208)), want)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("d,bs", [(64, 16), (128, 8), (128, 64), (256, 16)])
@pytest.mark.parametrize("seqs", [[(4000, 5)], [(2000, 33), (0, 300), (63, 1)], [(i * 97 % 700, 1 + i * 41 % 120) for i in range(20)]],
                         ids=["parts", "three", "many"])
def test_prefill(kind, d, bs, seqs):
    from bpt_b200.kernels.prefill_attention import prefill_attend

    g = torch.Generator().manual_seed(d)
    lengths = [c + n for c, n in seqs]
    kv, one = counting_cache(kind, lengths, bs, 2, d, g)
    q = torch.randn(sum(n for _, n in seqs), 6, d, generator=g).to(DTYPES.get(kind, torch.float16)).cuda()
    cu = torch.tensor([0] + [n for _, n in seqs]).cumsum(0).to(torch.int32).cuda()
    n = torch.tensor(lengths, dtype=torch.int32).cuda()
    for window, cap in ((0, 0.0), (777, 20.0), (1, 0.0)):
        want = torch.stack([counts(*visible(c + i, c + new, window=window), 6, 2, d, one) for c, new in seqs for i in range(new)])
        check(prefill_attend(q, kv, cu, n, sm_scale(d), window=window, softcap=cap), want)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("cap", [0.0, 25.0])
@pytest.mark.parametrize("alibi", [False, True])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_every_instance_of_the_prefill(kind, d, cap, alibi, sign):
    """Each page type, head size, cap, bias and sign of the factor has a kernel of its own."""
    from bpt_b200.kernels.prefill_attention import prefill_attend

    seqs = [(70, 40), (0, 33), (700, 2)]
    kv, keys, values, q, table, cu, lengths = case(kind, seqs, 8, 2, d, 16, seed=d, q_spread=2.0)
    slopes = 2.0 ** -torch.arange(1, 9).float() if alibi else None
    want = reference(q * sign, keys, values, table, seqs, 16, softcap=cap, slopes=slopes)
    got = prefill_attend(q.cuda(), kv, cu.cuda(), lengths.cuda(), sign * sm_scale(d), softcap=cap,
                         alibi_slopes=None if slopes is None else slopes.cuda())
    off = (got.double().cpu() - want).abs() - tolerance(want, q.dtype, values.abs().max().item(), product_bits(kind, q.dtype))
    assert not torch.isnan(off).any() and (off <= 0).all()
