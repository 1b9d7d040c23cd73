"""A key that takes nearly all of the probability beside a long tail of keys that take 2^-25.2 of its share each, and all of the
output: its own value is zero. A probability is a matrix operand of 16 bits, so a tail at f16's smallest values must not be
rounded away.

Tolerance, beside half a step of the output's type: the output is sum_j p_j v_j over the tail, so the measure is the sum of
p_j max_d |v_jd|; a probability is off by the rounding of the fp32 scores (2^-11, as in `paged_reference.tolerance`) in the sum
and in what divides it, 2^-10, and by its own rounding to 8 bits (bf16 prefill) or at least 11.

The prefill over f16 and E4M3 pages is not held to this: its probabilities are f16 of at most 1 where a row's largest is met,
and it states that it loses those below 2^-25."""

import math

import pytest
import torch

from tests.paged_reference import DTYPES, KINDS, page_table

D, HKV, REP = 128, 2, 3


def tail_cache(kind, lengths, bs, g):
    """Keys of zeros but for the first of each sequence, all ones; values between 0.5 and 1.5, the first key's zero
    (INT8: its scale as small as it goes). The values as they are stored, in 64 bits."""
    from bpt_b200.kernels.kv_attention import PagedQuantKV

    table, blocks = page_table(lengths, bs, g)
    keys, values = torch.zeros(blocks, bs, HKV, D), 0.5 + torch.rand(blocks, bs, HKV, D, generator=g)
    first = table[:, 0].long()
    keys[first, 0], values[first, 0] = 1.0, 0.0
    if kind in DTYPES:
        pools, scales = [x.to(DTYPES[kind]) for x in (keys, values)], (1.0, 1.0)
        stored = pools[1].double()
    elif kind == "fp8":
        pools, scales = [x.mul(64).to(torch.float8_e4m3fn) for x in (keys, values)], (1 / 64, 1 / 64)
        stored = pools[1].double() / 64
        pools = [p.view(torch.uint8) for p in pools]
    else:
        s = [(x.abs().amax(-1) / 127).to(torch.float16).clamp(min=2.0**-24) for x in (keys, values)]
        s[0][:] = 2.0**-6  # (1 is 64 of them)
        pools = [(x / t.float()[..., None]).round().clamp(-128, 127).to(torch.int8) for x, t in zip((keys, values), s, strict=True)]
        stored, scales = pools[1].double() * s[1].double()[..., None], [t.cuda() for t in s]
    return PagedQuantKV(kind, pools[0].cuda(), pools[1].cuda(), table.cuda(), bs, *scales), stored, table


def expected(stored, table, n, bs):
    """The output over the first n keys of a sequence, and its measure."""
    v = stored[table[: -(-n // bs)].long()].flatten(0, 1)[1:n]
    share = 2.0**-25.2 / (1 + (n - 1) * 2.0**-25.2)
    out, most = v.sum(0) * share, v.abs().amax(-1).sum(0) * share
    return out.repeat_interleave(REP, dim=0), most.repeat_interleave(REP, dim=0)[:, None]


def check(got, want, most, bits):
    half = 0.0 if got.dtype == torch.float32 else torch.finfo(got.dtype).eps / 2
    off = (got.double().cpu() - want).abs() / (half * want.abs() + most * (2.0**-10 + 2.0**-bits))
    worst = off.max().item()  # (NaN if any is)
    assert worst <= 1, f"{worst:.3g} of what is allowed"


def query(rows):
    """Queries whose score with a key of ones is 25.2 ln 2 under `factor`, exactly so in every type: all elements 1."""
    return torch.ones(rows, HKV * REP, D), 25.2 * math.log(2) / D


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("lengths", [[20000], [3000] * 70], ids=["parts", "many"])
def test_decode(kind, lengths):
    from bpt_b200.kernels.kv_attention import attend, decode_attention, merge_partials

    g = torch.Generator().manual_seed(1)
    kv, stored, table = tail_cache(kind, lengths, 16, g)
    q, factor = query(len(lengths))
    n = torch.tensor(lengths, dtype=torch.int32).cuda()
    want, most = (torch.stack(x) for x in zip(*(expected(stored, table[b], m, 16) for b, m in enumerate(lengths)), strict=True))
    check(attend(q.cuda(), kv, n, factor, window=1 << 20), want, most, 11)
    check(merge_partials(*decode_attention(q.cuda(), kv, n, factor, window=1 << 20, split=65536)), want, most, 11)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("seqs", [[(20000, 3)], [(2000, 1000), (2900, 60)]], ids=["parts", "tiles"])
def test_prefill(kind, seqs):
    from bpt_b200.kernels.prefill_attention import prefill_attend

    g = torch.Generator().manual_seed(2)
    lengths = [c + n for c, n in seqs]
    kv, stored, table = tail_cache(kind, lengths, 16, g)
    q, factor = query(sum(n for _, n in seqs))
    q = q.to(DTYPES.get(kind, torch.bfloat16))
    cu = torch.tensor([0] + [n for _, n in seqs]).cumsum(0).to(torch.int32).cuda()
    got = prefill_attend(q.cuda(), kv, cu, torch.tensor(lengths, dtype=torch.int32).cuda(), factor)
    at = 0
    for b, (ctx, new) in enumerate(seqs):
        for i in range(0, new, 1 if new < 100 else 37):
            check(got[at + i], *expected(stored, table[b], ctx + i + 1, 16), 8 if kind == "bf16" else 11)
        at += new
