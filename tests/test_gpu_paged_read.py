"""attend / decode_attention over paged caches of every format with caps, windows, distance bias and first visible keys,
against attention in 64 bits; the refusals run on the CPU."""

import pytest
import torch

from tests.paged_reference import KINDS, assert_within, attention_row, make_cache, page_table, sm_scale, visible


def case(kind, lengths, hq, hkv, d, bs, seed=0, q_dtype=torch.float32, q_spread=1.0, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    table, blocks = page_table(lengths, bs, g)
    kv, keys, values = make_cache(kind, blocks, bs, hkv, d, table, g, spread)
    q = (torch.randn(len(lengths), hq, d, generator=g) * q_spread).to(q_dtype)
    return kv, keys, values, q, table


def reference(q, keys, values, table, lengths, bs, window=0, softcap=0.0, slopes=None, starts=None):
    rows = []
    for b, n in enumerate(lengths):
        pages = table[b, : max(1, -(-n // bs))].long()
        k, v = (x[pages].flatten(0, 1) for x in (keys, values))
        lo, hi = visible(n - 1, n, starts[b] if starts is not None else 0, window)
        rows.append(attention_row(q[b].double(), k, v, n - 1, lo, hi, sm_scale(q.shape[2]), softcap, slopes))
    return torch.stack(rows)


def bits(kind):
    return 16 if kind == "bf16" else 20


CASES = [
    # lengths, Hq, Hkv, D, block size, window, softcap, alibi, starts
    ([1], 1, 1, 64, 16, 0, 0.0, False, None),
    ([0, 1, 15, 16, 17, 129], 16, 8, 128, 16, 0, 0.0, False, None),
    ([700, 0, 33], 7, 1, 128, 8, 0, 30.0, False, None),
    ([513, 2049], 14, 2, 64, 64, 0, 0.0, True, None),
    ([300, 5, 1000, 64], 5, 5, 256, 32, 0, 0.0, False, [0, 5, 999, 100]),
    ([1000, 31, 400], 16, 1, 128, 16, 100, 20.0, True, [0, 0, 399]),
    ([4000], 32, 4, 128, 16, 1, 0.0, False, None),
    ([257, 255], 12, 4, 256, 8, 77, 50.0, False, [250, 200]),
    ([90, 91], 9, 3, 64, 1024, 0, 0.0, True, [-5, 3]),
]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("case_", CASES, ids=range(len(CASES)))
@pytest.mark.parametrize("split", [None, 64])
def test_attend_matches_64_bits(kind, case_, split):
    from bpt_b200 import _lib
    from bpt_b200.kernels.kv_attention import attend

    lengths, hq, hkv, d, bs, window, cap, alibi, starts = case_
    if kind in ("fp8", "int8") and not (window or cap or alibi or starts):
        cap = 40.0  # without an option these caches read by their own kernel
    kv, keys, values, q, table = case(kind, lengths, hq, hkv, d, bs, seed=hq + d, q_spread=3.0 if cap else 1.0)
    slopes = 2.0 ** -torch.arange(1, hq + 1).float() if alibi else None
    want = reference(q, keys, values, table, lengths, bs, window, cap, slopes, starts)
    for out_dtype in (torch.float32, torch.bfloat16):
        out = torch.full((len(lengths), hq, d), float("nan"), dtype=out_dtype, device="cuda")
        got = attend(q.cuda(), kv, torch.tensor(lengths, dtype=torch.int32).cuda(), sm_scale(d), softcap=cap, window=window,
                     alibi_slopes=None if slopes is None else slopes.cuda(), split=split, out=out,
                     key_starts=None if starts is None else torch.tensor(starts, dtype=torch.int32).cuda())
        assert got is out
        assert_within(got, want, out_dtype, values.abs().max().item(), bits(kind))
        for b, n in enumerate(lengths):  # nothing visible: zeros
            if n == 0 or (starts and starts[b] >= n):
                assert (got[b] == 0).all()
    assert _lib.device_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
def test_partials_join_to_the_same(kind):
    from bpt_b200.kernels.kv_attention import decode_attention, merge_partials

    lengths = [530, 0, 64, 129]
    kv, keys, values, q, table = case(kind, lengths, 6, 2, 128, 16, seed=4)
    out, lse = decode_attention(q.cuda(), kv, torch.tensor(lengths, dtype=torch.int32).cuda(), sm_scale(128), split=128,
                                window=400, softcap=25.0)
    assert out.shape == (4, 6, 5, 128) and lse.shape == (4, 6, 5)
    assert torch.isneginf(lse[1]).all() and (out[1] == 0).all()
    assert torch.isneginf(lse[0, :, 0]).all()  # keys 0-127 are behind the window
    want = reference(q, keys, values, table, lengths, 16, 400, 25.0)
    assert_within(merge_partials(out, lse), want, torch.float32, values.abs().max().item(), bits(kind))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("q_dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_q_types_strides_and_range(kind, q_dtype):
    """q of any dtype and stride, also far outside f16's range; scores stay small by the scale."""
    from bpt_b200.kernels.kv_attention import attend

    lengths = [200, 37]
    kv, keys, values, q, table = case(kind, lengths, 4, 2, 128, 16, seed=5, q_dtype=q_dtype)
    big = 1.0 if q_dtype == torch.float16 else 2.0**20
    wide = torch.zeros(2, 8, 128, dtype=q_dtype)
    wide[:, ::2] = q * big
    want = reference(q, keys, values, table, lengths, 16)
    got = attend(wide.cuda()[:, ::2], kv, torch.tensor(lengths).cuda(), sm_scale(128) / big)
    assert_within(got, want, torch.float32, values.abs().max().item(), bits(kind))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
def test_what_is_not_visible_is_not_read(kind):
    """NaN in every slot that no query sees (stale pages, the rest of the last page, keys before the window): no trace."""
    from bpt_b200.kernels.kv_attention import attend

    lengths = [203, 16, 77]
    kv, keys, values, q, table = case(kind, lengths, 8, 2, 128, 16, seed=6)
    seen = torch.zeros(kv.num_blocks, 16, dtype=torch.bool)
    for b, n in enumerate(lengths):
        for j in range(max(0, n - 50), n):
            seen[table[b, j // 16], j % 16] = True
    for pool in (kv.k_pool, kv.v_pool):
        if kind in ("bf16", "f16"):
            pool[~seen.cuda()] = float("nan")
        elif kind == "fp8":
            pool[~seen.cuda()] = 0x7F
    if kind == "int8":
        kv.k_scale[~seen.cuda()] = float("nan")
        kv.v_scale[~seen.cuda()] = float("inf")
    want = reference(q, keys, values, table, lengths, 16, window=50, softcap=30.0)
    got = attend(q.cuda(), kv, torch.tensor(lengths, dtype=torch.int32).cuda(), sm_scale(128), window=50, softcap=30.0)
    assert_within(got, want, torch.float32, values.abs().max().item(), bits(kind))


@pytest.mark.gpu
def test_bad_blocks_and_lengths_are_left_out_and_recorded():
    from bpt_b200 import _lib
    from bpt_b200.kernels.kv_attention import attend

    lengths = [64, 64]
    for bs in (8, 16):
        kv, keys, values, q, table = case("bf16", lengths, 4, 2, 128, bs, seed=7)
        bad = table.clone()
        bad[0, 1], bad[1, 2] = kv.num_blocks, -1
        kv.block_table = bad.cuda()
        assert _lib.device_error() == 0
        got = attend(q.cuda(), kv, torch.tensor([64, 100], dtype=torch.int32).cuda(), sm_scale(128))  # 100: more than 64 slots
        assert _lib.device_error() == 2
        for b, hole in ((0, 1), (1, 2)):
            keep = [j for j in range(64) if j // bs != hole]
            k, v = (x[table[b].long()].flatten(0, 1)[keep] for x in (keys, values))
            want = attention_row(q[b].double(), k, v, 63, 0, len(keep), sm_scale(128))
            assert_within(got[b], want, torch.float32, values.abs().max().item(), 16)


@pytest.mark.gpu
def test_a_wrong_tokens_hint_and_repeated_calls_give_the_same():
    """`tokens` bounds the launch, not the result; nothing of one call's workspace shows in the next."""
    from bpt_b200.kernels.kv_attention import attend

    lengths = [3000, 10, 1500]
    kv, keys, values, q, table = case("bf16", lengths, 8, 4, 64, 16, seed=8)
    want = reference(q, keys, values, table, lengths, 16)
    n = torch.tensor(lengths, dtype=torch.int32).cuda()
    vmax = values.abs().max().item()
    first = attend(q.cuda(), kv, n, sm_scale(64))
    for tokens, split in ((100, None), (3000, 16), (3000, 1024), (1, 16), (None, None)):
        assert_within(attend(q.cuda(), kv, n, sm_scale(64), tokens=tokens, split=split), want, torch.float32, vmax, 16)
    assert torch.equal(first, attend(q.cuda(), kv, n, sm_scale(64)))  # no order of arrival shows in the result


@pytest.mark.gpu
def test_two_graphs_and_two_streams_do_not_share_a_workspace():
    from bpt_b200.kernels.kv_attention import attend

    calls = []
    for seed in (9, 10):
        kv, keys, values, q, table = case("bf16", [2000, 900], 8, 4, 128, 16, seed=seed)
        n = torch.tensor([2000, 900], dtype=torch.int32).cuda()
        calls.append((q.cuda(), kv, n, attend(q.cuda(), kv, n, sm_scale(128), split=64)))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    graphs, outs = [], []
    for q, kv, n, _ in calls:  # both captured on one stream, replayed on two
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs.append(attend(q, kv, n, sm_scale(128), split=64))
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):
        for graph, stream in zip(graphs, streams, strict=True):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for (_, _, _, want), out in zip(calls, outs, strict=True):
        assert torch.equal(out, want)
    eager = []
    for (q, kv, n, _), stream in zip(calls, streams, strict=True):
        with torch.cuda.stream(stream):
            eager.append(attend(q, kv, n, sm_scale(128), split=64))
    torch.cuda.synchronize()
    for (_, _, _, want), out in zip(calls, eager, strict=True):
        assert torch.equal(out, want)


@pytest.mark.gpu
def test_a_long_cache_passes_32_bits():
    """Byte offsets above 2^32 into the pools: the last pages of a pool of 4.6 GB."""
    from bpt_b200.kernels.kv_attention import PagedQuantKV, attend

    hkv, d, bs = 8, 256, 16
    nb = (1 << 32) // (bs * hkv * d * 2) + 4096
    pools = [torch.empty(nb, bs, hkv, d, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    g = torch.Generator().manual_seed(11)
    keys, values = (torch.randn(4, bs, hkv, d, generator=g).to(torch.bfloat16) for _ in range(2))
    for pool, x in zip(pools, (keys, values), strict=True):
        pool[-4:] = x.cuda()
    table = torch.arange(nb - 4, nb, dtype=torch.int32)[None]
    q = torch.randn(1, 8, d, generator=g)
    kv = PagedQuantKV("bf16", pools[0], pools[1], table.cuda(), bs)
    got = attend(q.cuda(), kv, torch.tensor([61], dtype=torch.int32).cuda(), sm_scale(d))
    want = attention_row(q[0].double(), keys.double().flatten(0, 1), values.double().flatten(0, 1), 60, 0, 61, sm_scale(d))
    assert_within(got[0], want, torch.float32, values.abs().max().item(), 16)


def test_refusals_need_no_gpu():
    from bpt_b200 import _lib

    L = _lib.lib()

    def call(**kw):
        a = {"q": 64, "qd": 2, "qb": 512, "qh": 128, "kp": 64, "vp": 64, "kind": 4, "ks": 1.0, "vs": 1.0, "kss": None, "vss": None,
             "bt": 64, "bts": 4, "btw": 4, "len": 64, "starts": None, "slopes": None, "cap": 0.0, "window": 0, "B": 2, "Hq": 4,
             "Hkv": 2, "D": 128, "bs": 16, "nb": 8, "split": 64, "n": 1, "tokens": 8, "scale": 1.0, "out": 64, "od": 2, "po": None,
             "pl": None, "ws": None, "wsb": 0, "flags": 0, "stream": None} | kw
        return _lib.paged_read(*(0 if x is None else x for x in a.values()))

    assert call(B=0) == _lib.OK
    for name in ("q", "kp", "vp", "bt", "len", "out"):
        assert call(**{name: None}) == _lib.ERR_INVALID and b"null" in L.bpt_last_error()
    assert call(D=96) == _lib.ERR_UNSUPPORTED and call(bs=24) == _lib.ERR_UNSUPPORTED and call(bs=4) == _lib.ERR_UNSUPPORTED
    assert call(kind=0) == _lib.ERR_INVALID and call(qd=7) == _lib.ERR_INVALID and call(od=7) == _lib.ERR_INVALID
    assert call(Hq=3) == _lib.ERR_INVALID and call(tokens=0) == _lib.ERR_INVALID
    for bad in ({"split": 24}, {"split": 0}, {"n": 0}):
        assert call(po=64, pl=64, **bad) == _lib.ERR_INVALID and b"split" in L.bpt_last_error()
    assert call(window=-1) == _lib.ERR_INVALID and call(cap=-1.0) == _lib.ERR_INVALID and call(cap=float("nan")) == _lib.ERR_INVALID
    assert call(bts=3) == _lib.ERR_INVALID and call(btw=0) == _lib.ERR_INVALID
    assert call(tokens=4000) == _lib.ERR_WORKSPACE
    assert call(tokens=4000, ws=64, wsb=100) == _lib.ERR_WORKSPACE and call(tokens=4000, ws=72, wsb=1 << 30) == _lib.ERR_ALIGNMENT
    assert call(po=64) == _lib.ERR_INVALID  # partials without their log-sum-exps
    assert call(kind=1, ks=0.0) == _lib.ERR_INVALID and call(kind=2) == _lib.ERR_INVALID
    assert call(kp=72) == _lib.ERR_ALIGNMENT
    assert L.bpt_paged_read_workspace_bytes(16, 8, 128, 4) >= 2 * 8 * 8 * 129 * 4


@pytest.mark.gpu
def test_python_refusals():
    from bpt_b200.kernels.kv_attention import QuantKV, attend, decode_attention

    kv, _, _, q, _ = case("bf16", [20], 4, 2, 64, 16, q_dtype=torch.bfloat16)
    n, q = torch.tensor([20], dtype=torch.int32).cuda(), q.cuda()

    def refused(q=q, kv=kv, n=n, **kw):
        with pytest.raises(ValueError):
            attend(q, kv, n, 1.0, **kw)

    with pytest.raises(ValueError):
        decode_attention(q, kv, n, 1.0, split=24)
    refused(q=q.cpu())
    refused(q=q[:, :3])
    refused(q=q.double())
    refused(n=n.float())
    refused(n=n.repeat(2))
    refused(window=-1)
    refused(softcap=-2.0)
    refused(alibi_slopes=torch.ones(3, device="cuda"))
    refused(key_starts=torch.zeros(2, dtype=torch.int32, device="cuda"))
    refused(out=torch.empty(1, 4, 32, device="cuda"))
    codes = torch.zeros(1, 2, 32, 64, dtype=torch.uint8, device="cuda")
    grid, per = torch.zeros(1, 2, 1, 64, dtype=torch.float16, device="cuda"), torch.zeros(1, 2, 32, dtype=torch.float16, device="cuda")
    refused(kv=QuantKV(8, 32, codes, codes, grid, grid, per, per), softcap=3.0)
