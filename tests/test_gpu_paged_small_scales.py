"""INT8 pages whose values are small or differ much in size from key to key: the scales (fp16, max|v| / 127) and their
products with the probabilities then lie in f16's subnormal range or below it.

Tolerance, beside half a step of the output's type: an output is sum_j p_j v_j, and what each probability may be off by shows
in proportion to that key's own values, so the measure is the sum of p_j max_d |v_jd|. A probability is off by the rounding of
fp32 scores (2^-11, as in `paged_reference.tolerance`) in the sum and in what divides it: 2^-10; by its rounding to a matrix
operand of 11 bits, 2^-11; and, for keys far below the largest product of a probability and a scale, by half a step of the
smallest f16, 2^-25, in units of at most twice that product: N 2^-24 of it for N keys, times the largest code, 127. That last
part knows of a key only its scale: a key of nothing but zeros has, by the format, scale 1.0 and code 0, so its product can be
the largest while the sum of p_j max_d |v_jd| holds nothing of it (the case "one", whose first key often rounds to zeros); it
is taken from sum_j p_j 127 s_j, which is at least the largest product times 127."""

import pytest
import torch

from tests.paged_reference import page_table, sm_scale

HQ, HKV, D = 6, 2, 128


def int8_cache(keys, values, table, bs):
    """Pools of keys and values [num_blocks, bs, Hkv, D], what they stand for in 64 bits, and 127 value scales."""
    from bpt_b200.kernels.kv_attention import PagedQuantKV

    pools, scales, stored, sizes = [], [], [], None
    for x in (keys, values):
        s = (x.abs().amax(-1) / 127).to(torch.float16)
        s[s == 0] = 1.0
        code = (x / s.float()[..., None]).round().clamp(-128, 127).to(torch.int8)
        pools.append(code.cuda())
        scales.append(s.cuda())
        stored.append(code.double() * s.double()[..., None])
        sizes = 127 * s.double()
    return PagedQuantKV("int8", pools[0], pools[1], table.cuda(), bs, scales[0], scales[1]), stored[0], stored[1], sizes


def row(q, k, v, sizes, lo, hi):
    """Attention of q [Hq, D] over the keys lo .. hi - 1, and what it may be off by but for the output's rounding (above)."""
    rep = q.shape[0] // k.shape[1]
    k, v, sizes = (x[lo:hi].repeat_interleave(rep, dim=1) for x in (k, v, sizes))
    p = torch.softmax(torch.einsum("hd,nhd->hn", q.double(), k) * sm_scale(D), dim=-1)
    off = torch.einsum("hn,nh->h", p, (2.0**-10 + 2.0**-11) * v.abs().amax(-1) + (hi - lo) * 2.0**-24 * sizes)
    return torch.einsum("hn,nhd->hd", p, v), off[:, None]


def check(got, want, allowed):
    half = 0.0 if got.dtype == torch.float32 else torch.finfo(got.dtype).eps / 2
    off = (got.double().cpu() - want).abs() / (half * want.abs() + allowed)
    worst = off.max().item()  # (NaN if any is)
    assert worst <= 1, f"{worst:.3g} of what is allowed"


def inputs(sizes, lengths, bs, seed):
    g = torch.Generator().manual_seed(seed)
    table, blocks = page_table(lengths, bs, g)
    keys, values = (torch.randn(blocks, bs, HKV, D, generator=g) for _ in range(2))
    if sizes == "mixed":  # from key to key, over six powers of ten
        values = values * 10.0 ** (-6 * torch.rand(blocks, bs, HKV, 1, generator=g))
    elif sizes == "one":  # a key that takes nearly all the probability and has almost no value, among large ones
        keys = keys * 0.1
        keys[table[:, 0].long(), 0] = 3.0
        values[table[:, 0].long(), 0] *= 1e-6
    elif sizes == "sink":  # a key that takes most of it, its value's share about that of each other key
        keys = keys * 0.1
        keys[table[:, 0].long(), 0] = 1.0
        values[table[:, 0].long(), 0] *= 1e-4
    else:
        values = values * sizes
    return table, *int8_cache(keys, values, table, bs), g


SIZES = [1.0, 1e-2, 1e-3, 1e-4, 1e-5, "mixed", "one", "sink"]


@pytest.mark.gpu
@pytest.mark.parametrize("sizes", SIZES)
def test_decode(sizes):
    from bpt_b200.kernels.kv_attention import attend, decode_attention, merge_partials

    lengths = [2000, 17, 600]
    table, kv, keys, values, scales, g = inputs(sizes, lengths, 16, 1)
    q = torch.randn(3, HQ, D, generator=g) * (1.0 if sizes in ("one", "sink") else 2.0)
    if sizes in ("one", "sink"):
        q = q.abs()
    rows = [row(q[b], *(x[table[b, : -(-n // 16)].long()].flatten(0, 1) for x in (keys, values, scales)), 0, n) for b, n in enumerate(lengths)]
    want, allowed = (torch.stack(x) for x in zip(*rows, strict=True))
    n = torch.tensor(lengths, dtype=torch.int32).cuda()
    check(attend(q.cuda(), kv, n, sm_scale(D), window=5000), want, allowed)
    check(merge_partials(*decode_attention(q.cuda(), kv, n, sm_scale(D), window=5000, split=256)), want, allowed)


@pytest.mark.gpu
@pytest.mark.parametrize("sizes", SIZES)
@pytest.mark.parametrize("seqs", [[(300, 40), (0, 70)], [(1500, 3)]], ids=["tiles", "parts"])
def test_prefill(sizes, seqs):
    from bpt_b200.kernels.prefill_attention import prefill_attend

    lengths = [c + n for c, n in seqs]
    table, kv, keys, values, scales, g = inputs(sizes, lengths, 16, 2)
    q = torch.randn(sum(n for _, n in seqs), HQ, D, generator=g) * (1.0 if sizes in ("one", "sink") else 2.0)
    q = (q.abs() if sizes in ("one", "sink") else q).to(torch.bfloat16)
    rows, at = [], 0
    for b, (ctx, new) in enumerate(seqs):
        cached = [x[table[b, : -(-lengths[b] // 16)].long()].flatten(0, 1) for x in (keys, values, scales)]
        for i in range(new):
            rows.append(row(q[at], *cached, 0, ctx + i + 1))
            at += 1
    want, allowed = (torch.stack(x) for x in zip(*rows, strict=True))
    cu = torch.tensor([0] + [n for _, n in seqs]).cumsum(0).to(torch.int32).cuda()
    got = prefill_attend(q.cuda(), kv, cu, torch.tensor(lengths, dtype=torch.int32).cuda(), sm_scale(D))
    check(got, want, allowed)
