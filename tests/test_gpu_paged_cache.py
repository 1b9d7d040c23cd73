"""The paged operators as they are used together: through `PagedQuantizedKVCache` and through the decode step, against 64 bits.

What each of them stores and returns on its own is in test_gpu_paged_append.py, test_gpu_paged_read.py and
test_gpu_paged_prefill.py.
"""

import math
from types import SimpleNamespace

import pytest
import torch

from tests.paged_reference import DTYPES, KINDS, assert_within, attention_row, page_table, visible
from tests.paged_reference import make_cache as filled_cache

HQ, HKV, D = 4, 2, 128


def make_cache(kind):
    from bpt_b200.integration import PagedQuantizedKVCache

    cfg = SimpleNamespace(num_layers=1, num_kv_heads=HKV, head_dim=D)
    return PagedQuantizedKVCache(cfg, num_blocks=64, block_size=16, kind=kind, k_scale=1 / 64, v_scale=1 / 64)


def steps(cache):
    """(rows, positions) of a run: a prompt per row, a second chunk of one of them, two decode steps of all rows."""
    lens = {"a": 37, "b": 16, "c": 70}
    for row, n in lens.items():
        cache.reserve(row, n + 24)
        yield [row], torch.arange(n)[None]
    yield ["b"], torch.arange(16, 25)[None]
    lens["b"] = 25
    for i in range(2):
        yield list(lens), torch.tensor([[n + i] for n in lens.values()])


def expected(q, cache, meta, scale, **scores):
    """q [B, Hq, Q, D] in double over what the cache holds, in double."""
    window = scores.pop("window", 0)
    keys, values = (x.double().cpu() for x in cache.dequantized(0, meta))  # [B, Hkv, kv_len, D]
    want = torch.zeros(q.shape, dtype=torch.float64)
    for i in range(q.shape[0]):
        for t in range(q.shape[2]):
            pos = int(meta.positions[i, t])
            lo, hi = visible(pos, int(meta.lengths[i]), window=window)
            want[i, :, t] = attention_row(q[i, :, t], keys[i].transpose(0, 1), values[i].transpose(0, 1), pos, lo, hi, scale,
                                          **scores)
    return want, values.abs().max()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("q_dtype", ["pages", torch.float32])
def test_attend_over_16_bit_pages(kind, q_dtype):
    """`attend`: k and v are stored as they are (rounded once), prompts and chunks by `prefill_attend` where q has the
    pages' dtype and by the unfused path where it has not, single tokens by the decode read."""
    cache, g = make_cache(kind), torch.Generator().manual_seed(5)
    dtype = DTYPES[kind] if q_dtype == "pages" else q_dtype
    for rows, positions in steps(cache):
        b, n = positions.shape
        q, k, v = (torch.randn(b, h, n, D, generator=g).to(dtype) for h in (HQ, HKV, HKV))
        meta = cache.prepare(rows, positions.cuda())
        got = cache.attend(0, q.cuda(), k.cuda(), v.cuda(), meta, scale=1 / math.sqrt(D))
        assert got.dtype == dtype and got.shape == q.shape
        keys, values = cache.dequantized(0, meta)
        for i in range(b):
            at = positions[i].cuda()
            assert torch.equal(keys[i][:, at].cpu(), k[i].to(DTYPES[kind]).float())
            assert torch.equal(values[i][:, at].cpu(), v[i].to(DTYPES[kind]).float())
        want, vmax = expected(q.double(), cache, meta, 1 / math.sqrt(D))
        assert_within(got, want, dtype, vmax, 8 if kind == "bf16" else 11)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("scores", [{}, {"softcap": 15.0, "window": 20}], ids=["plain", "capped_window"])
def test_rotate_and_attend(kind, scores):
    """The projections' views, not rotated: the tokens' rows rotate and are stored by `rope_kv_append` (compared bit for bit
    with a call of its own on a second cache), and the attention is that of the stored pages in 64 bits."""
    from bpt_b200.kernels.kv_write import rope_kv_append, rope_table

    cache, twin, g = make_cache(kind), make_cache(kind), torch.Generator().manual_seed(6)
    dtype = DTYPES.get(kind, torch.bfloat16)
    cos, sin = rope_table(128, 64, 1e4)  # the first half of each head rotates
    norms = [(1 + 0.1 * torch.randn(D, generator=g)).to(dtype).cuda() for _ in range(2)]
    for rows, positions in steps(cache):
        b, n = positions.shape
        twin.tables = cache.tables
        qkv = torch.randn(b, n, HQ + 2 * HKV, D, generator=g).to(dtype).cuda()
        q, k, v = (x.transpose(1, 2) for x in qkv.split([HQ, HKV, HKV], dim=2))
        meta = cache.prepare(rows, positions.cuda())
        got = cache.rotate_and_attend(0, q, k, v, meta, 1 / math.sqrt(D), cos, sin, q_norm=norms[0], k_norm=norms[1], **scores)
        turned = rope_kv_append(*(x.flatten(0, 1) for x in qkv.split([HQ, HKV, HKV], dim=2)), twin.layer_view(0, meta),
                                meta.positions, cos, sin, meta.write_blocks, meta.write_offsets, q_norm=norms[0],
                                k_norm=norms[1])
        assert torch.equal(cache.layers[0].k_pool, twin.layers[0].k_pool)
        assert torch.equal(cache.layers[0].v_pool, twin.layers[0].v_pool)
        turned = turned.view(b, n, HQ, D).transpose(1, 2).double().cpu()
        want, vmax = expected(turned, cache, meta, 1 / math.sqrt(D), **scores)
        assert got.dtype == dtype and got.shape == q.shape
        assert_within(got, want, dtype, vmax, 8 if kind == "bf16" else 11)


def decoder(seed, layers=1):
    from bpt_b200.decode import Qwen3Decoder, Qwen3Dims

    dims = Qwen3Dims(layers=layers, intermediate=1024, vocab=512)
    return Qwen3Decoder(dims, torch.tensor([40, 17, 100, 0]), seed=seed, capacity=8, kv_kind="bf16")


@pytest.mark.gpu
def test_decode_step_over_bf16_pages():
    """One layer's step from its own projection: the new token's pages hold the normalised, rotated key rounded once, no
    other slot changes, and the attention is that of the pages in 64 bits."""
    dec = decoder(3)
    dec.tokens.copy_(torch.tensor([1, 7, 300, 42]))
    d, layer = dec.dims, dec.layers[0]
    before = [layer.kv.k_pool.clone(), layer.kv.v_pool.clone()]
    at = dec.lengths.cpu().long()
    dec.step()
    torch.cuda.synchronize()
    assert torch.equal(dec.lengths.cpu().long(), at + 1)
    qkv = dec.qkv.double().cpu().view(dec.batch, -1, d.head_dim)
    q, k, v = qkv.split([d.q_heads, d.kv_heads, d.kv_heads], dim=1)

    def turned(x, w):  # in 64 bits
        x = x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + d.eps) * w.double().cpu()
        half = d.head_dim // 2
        inv = d.rope_theta ** (-torch.arange(half, dtype=torch.float64) * 2 / d.head_dim)
        a = (at[:, None] * inv)[:, None]
        lo, hi = x[..., :half], x[..., half:]
        return torch.cat([lo * a.cos() - hi * a.sin(), hi * a.cos() + lo * a.sin()], dim=-1)

    table = dec.block_table.cpu().long()
    blocks, offsets = table.gather(1, (at // 16)[:, None])[:, 0], at % 16
    want_k, want_q = turned(k, layer.k_norm), turned(q, layer.q_norm)
    k_pool, v_pool = layer.kv.k_pool.cpu(), layer.kv.v_pool.cpu()
    # one rounding to bf16, of fp32 sums of 128 squares and two products (below 2^-16 of the row's largest)
    for got, want in ((k_pool[blocks, offsets], want_k), (dec.q.cpu(), want_q)):
        off = (got.double() - want).abs()
        assert (off <= 2.0**-8 * want.abs() + 2.0**-16 * want.abs().amax(-1, keepdim=True)).all()
    assert torch.equal(v_pool[blocks, offsets].double(), v)
    for pool, old in ((k_pool, before[0].cpu()), (v_pool, before[1].cpu())):
        old[blocks, offsets] = pool[blocks, offsets]
        assert torch.equal(pool, old)
    want = torch.zeros(dec.batch, d.q_heads, d.head_dim, dtype=torch.float64)
    for i in range(dec.batch):
        pages = table[i, : int(at[i]) // 16 + 1]
        keys, values = (p[pages].flatten(0, 1).double() for p in (k_pool, v_pool))
        want[i] = attention_row(dec.q[i].double().cpu(), keys, values, int(at[i]), 0, int(at[i]) + 1, dec.scale)
    assert_within(dec.attn, want, torch.bfloat16, v_pool.double().abs().max(), 8)


@pytest.mark.gpu
def test_decode_step_over_bf16_pages_replays():
    eager, graphed = decoder(5, layers=2), decoder(5, layers=2)
    graphed.capture()  # one eager step inside, then the capture
    eager.step()
    for _ in range(3):
        eager.step()
        graphed.step()
    torch.cuda.synchronize()
    assert torch.equal(eager.lengths, graphed.lengths) and torch.equal(eager.tokens, graphed.tokens)
    assert torch.equal(eager.hidden, graphed.hidden)
    for a, b in zip(eager.layers, graphed.layers, strict=True):
        assert torch.equal(a.kv.k_pool, b.kv.k_pool) and torch.equal(a.kv.v_pool, b.kv.v_pool)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("bs,d", [(128, 128), (1024, 64), (256, 256)])
def test_pages_longer_than_a_step(kind, bs, d):
    """Pages that a kernel reads in several steps, the last one of each sequence filled in part."""
    from bpt_b200.kernels.kv_attention import attend
    from bpt_b200.kernels.prefill_attention import prefill_attend

    g = torch.Generator().manual_seed(bs)
    seqs = [(300, 40), (0, 130), (1100, 3)]  # cached, new
    lengths = [c + n for c, n in seqs]
    table, blocks = page_table(lengths, bs, g)
    kv, keys, values = filled_cache(kind, blocks, bs, HKV, d, table, g)
    dtype, scale, vmax = DTYPES.get(kind, torch.bfloat16), 1 / math.sqrt(d), values.abs().max()
    q = torch.randn(sum(n for _, n in seqs), HQ, d, generator=g).to(dtype)
    cu = torch.tensor([0] + [n for _, n in seqs]).cumsum(0).to(torch.int32)
    n = torch.tensor(lengths, dtype=torch.int32).cuda()

    def row(b, x, pos, window):
        pages = table[b, : -(-lengths[b] // bs)].long()
        k, v = (y[pages].flatten(0, 1) for y in (keys, values))
        lo, hi = visible(pos, lengths[b], window=window)
        return attention_row(x.double(), k, v, pos, lo, hi, scale)

    for window in (0, 90):
        got = prefill_attend(q.cuda(), kv, cu.cuda(), n, scale, window=window)
        want = torch.stack([row(b, q[int(cu[b]) + i], c + i, window) for b, (c, new) in enumerate(seqs) for i in range(new)])
        assert_within(got, want, dtype, vmax, 8 if kind == "bf16" else 11)
        last = q[cu[1:].long() - 1]
        got = attend(last.cuda(), kv, n, scale, window=window)
        want = torch.stack([row(b, last[b], lengths[b] - 1, window) for b in range(len(seqs))])
        assert_within(got, want, torch.float32, vmax, 8 if kind == "bf16" else 11)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["fp8", "int8"])
@pytest.mark.parametrize("hq,hkv", [(7, 1), (6, 2), (20, 20)])
def test_numbers_of_heads_that_the_8_bit_kernels_leave(kind, hq, hkv):
    from bpt_b200.kernels.kv_attention import attend, decode_attention, merge_partials

    g = torch.Generator().manual_seed(hq)
    lengths = [70, 0, 33]
    table, blocks = page_table(lengths, 16, g)
    kv, keys, values = filled_cache(kind, blocks, 16, hkv, D, table, g)
    q, n = torch.randn(3, hq, D, generator=g), torch.tensor(lengths, dtype=torch.int32).cuda()
    k, v = ([x[table[b, : max(1, -(-m // 16))].long()].flatten(0, 1) for b, m in enumerate(lengths)] for x in (keys, values))
    want = torch.stack([attention_row(q[b].double(), k[b], v[b], m - 1, 0, m, 1 / math.sqrt(D)) for b, m in enumerate(lengths)])
    for got in (attend(q.cuda(), kv, n, 1 / math.sqrt(D)), merge_partials(*decode_attention(q.cuda(), kv, n, 1 / math.sqrt(D)))):
        assert_within(got, want, torch.float32, values.abs().max(), 11)


def test_refusals_need_no_gpu():
    from bpt_b200.decode import Qwen3Decoder, Qwen3Dims
    from bpt_b200.integration import PagedQuantizedKVCache

    cfg = SimpleNamespace(num_layers=1, num_kv_heads=HKV, head_dim=D)
    with pytest.raises(ValueError, match="kind"):
        PagedQuantizedKVCache(cfg, num_blocks=4, kind="int4")
    with pytest.raises(ValueError, match="CUDA device"):
        PagedQuantizedKVCache(cfg, num_blocks=4, kind="bf16", device="cpu")
    for bad in ({"kv_kind": "int8"}, {"kv_kind": "bf16", "fused": False}):
        with pytest.raises(ValueError, match="kv_kind"):
            Qwen3Decoder(Qwen3Dims(layers=1), torch.tensor([4]), device="cpu", **bad)
