"""The paged operators in 64 bits on the CPU: what tests/test_gpu_paged_append.py, test_gpu_paged_read.py and
test_gpu_paged_prefill.py compare with."""

from __future__ import annotations

import math

import torch

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
KINDS = ("bf16", "f16", "fp8", "int8")


def make_cache(kind, num_blocks, block_size, kv_heads, head_dim, table, generator, spread=1.0):
    """A filled pool on the GPU and its keys and values in float64 [num_blocks, block_size, Hkv, D] on the CPU."""
    from bpt_b200.kernels.kv_attention import PagedQuantKV

    shape = (num_blocks, block_size, kv_heads, head_dim)
    pools, values, scales = [], [], []
    for _ in range(2):
        x = torch.randn(shape, generator=generator) * spread
        if kind in DTYPES:
            pool, scale = x.to(DTYPES[kind]), 1.0
            val = pool.double()
        elif kind == "fp8":
            scale = 1.0 / 64
            pool = (x / scale).clamp(-448, 448).to(torch.float8_e4m3fn)
            val, pool = pool.double() * scale, pool.view(torch.uint8)
        else:
            scale = (x.abs().amax(-1) / 127).to(torch.float16)
            pool = (x / scale.float()[..., None]).round().clamp(-128, 127).to(torch.int8)
            val, scale = pool.double() * scale.double()[..., None], scale.cuda()
        pools.append(pool.cuda())
        values.append(val)
        scales.append(scale)
    kv = PagedQuantKV(kind, pools[0], pools[1], table.cuda(), block_size, scales[0], scales[1])
    return kv, values[0], values[1]


def page_table(lengths, block_size, generator, spare=2):
    """(table [B, width], blocks in the pool): every sequence's pages at random places."""
    need = [max(1, -(-n // block_size)) for n in lengths]
    total = sum(need) + spare
    perm = torch.randperm(total, generator=generator).to(torch.int32)
    table, at = torch.zeros(len(need), max(need), dtype=torch.int32), 0
    for i, n in enumerate(need):
        table[i, :n] = perm[at : at + n]
        at += n
    return table, total


def visible(pos, length, start=0, window=0, prefix=0):
    """(lo, hi): the keys lo <= j < hi that a query at `pos` of a sequence of `length` tokens sees."""
    return max(0, start, pos - window + 1 if window else 0), min(length, max(pos + 1, prefix))


def attention_row(q, keys, values, pos, lo, hi, scale, softcap=0.0, slopes=None):
    """q [Hq, D] double, keys / values [N, Hkv, D] double -> [Hq, D]; zeros where nothing is visible."""
    hq, d = q.shape
    rep = hq // keys.shape[1]
    if hi <= lo:
        return torch.zeros(hq, d, dtype=torch.float64)
    k = keys[lo:hi].repeat_interleave(rep, dim=1)
    v = values[lo:hi].repeat_interleave(rep, dim=1)
    s = torch.einsum("hd,nhd->hn", q, k) * scale
    if softcap:
        s = softcap * torch.tanh(s / softcap)
    if slopes is not None:
        s = s - slopes.double()[:, None] * (pos - torch.arange(lo, hi)).abs().double()
    return torch.einsum("hn,nhd->hd", torch.softmax(s, dim=-1), v)


def tolerance(want, out_dtype, vmax, product_bits):
    """What a kernel that sums in fp32 may be off by: the output's own rounding (half a step of its type), the rounding of
    the probabilities to `product_bits` significant bits (half a step each, so at most that part of the largest value), and
    the scores' fp32 sums: D <= 256 terms of 2^-24 each on sums of at most 16, twice (scores and their exponentials),
    2 * 256 * 2^-24 * 16 = 2^-11 of the largest value."""
    half = 0.0 if out_dtype == torch.float32 else torch.finfo(out_dtype).eps / 2
    return half * want.abs() + vmax * (2.0 ** -product_bits + 2.0**-11)


def assert_within(got, want, out_dtype, vmax, product_bits):
    off = (got.double().cpu() - want).abs() - tolerance(want, out_dtype, vmax, product_bits)
    assert not torch.isnan(off).any(), "NaN"
    assert (off <= 0).all(), f"{off.max().item():.3g} over the tolerance at {off.flatten().argmax().item()}"


def sm_scale(d):
    return 1.0 / math.sqrt(d)
