"""prefill_attend over paged caches of every format, ragged batches, caps, windows, documents, prefixes and distance bias,
against attention in 64 bits; the refusals run on the CPU."""

import pytest
import torch

from tests.paged_reference import DTYPES, KINDS, assert_within, attention_row, make_cache, page_table, sm_scale, visible


def q_type(kind, i=0):
    return DTYPES.get(kind, (torch.bfloat16, torch.float16)[i % 2])


def case(kind, seqs, hq, hkv, d, bs, seed=0, q_dtype=None, q_spread=1.0):
    """seqs: (cached, new) per sequence."""
    g = torch.Generator().manual_seed(seed)
    lengths = [c + n for c, n in seqs]
    table, blocks = page_table(lengths, bs, g)
    kv, keys, values = make_cache(kind, blocks, bs, hkv, d, table, g)
    t = sum(n for _, n in seqs)
    q = (torch.randn(t, hq, d, generator=g) * q_spread).to(q_dtype or q_type(kind))
    cu = torch.tensor([0] + [n for _, n in seqs]).cumsum(0).to(torch.int32)
    return kv, keys, values, q, table, cu, torch.tensor(lengths, dtype=torch.int32)


def reference(q, keys, values, table, seqs, bs, window=0, softcap=0.0, slopes=None, starts=None, prefix=None, positions=None):
    rows, at = [], 0
    for b, (ctx, new) in enumerate(seqs):
        n = ctx + new
        pages = table[b, : max(1, -(-n // bs))].long()
        k, v = (x[pages].flatten(0, 1) for x in (keys, values))
        for i in range(new):
            p = ctx + i if positions is None else int(positions[at])
            lo, hi = visible(p, n, int(starts[at]) if starts is not None else 0, window, prefix[b] if prefix else 0)
            rows.append(attention_row(q[at].double(), k, v, p, lo, hi, sm_scale(q.shape[2]), softcap, slopes))
            at += 1
    return torch.stack(rows)


def product_bits(kind, q_dtype):
    # what the probabilities keep in the product: bf16 8 bits, f16 11, half a step lost
    return 8 if kind == "bf16" else 11


CASES = [
    # sequences (cached, new), Hq, Hkv, D, block size, window, softcap, alibi, prefix, documents
    ([(0, 1)], 1, 1, 64, 16, 0, 0.0, False, None, False),
    ([(0, 65)], 4, 4, 128, 16, 0, 0.0, False, None, False),
    ([(0, 3), (5, 0), (130, 40), (16, 17)], 14, 2, 128, 8, 0, 0.0, False, None, False),
    ([(300, 20), (0, 100)], 6, 2, 64, 64, 50, 0.0, True, None, False),
    ([(0, 129), (63, 2)], 5, 1, 256, 32, 0, 30.0, False, None, False),
    ([(10, 70), (0, 5)], 16, 2, 128, 16, 0, 0.0, False, [40, 3], False),
    ([(0, 200)], 3, 3, 64, 16, 0, 0.0, False, None, True),
    ([(100, 90), (7, 33)], 8, 1, 128, 16, 31, 20.0, True, [60, 500], True),
    ([(2000, 2), (1500, 9)], 4, 2, 128, 16, 0, 0.0, False, None, False),  # few rows, many keys: several parts
    ([(1999, 4)], 16, 8, 256, 16, 700, 50.0, False, [1800], False),
]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("case_", CASES, ids=range(len(CASES)))
def test_prefill_matches_64_bits(kind, case_):
    from bpt_b200 import _lib
    from bpt_b200.kernels.prefill_attention import prefill_attend

    seqs, hq, hkv, d, bs, window, cap, alibi, prefix, documents = case_
    kv, keys, values, q, table, cu, lengths = case(kind, seqs, hq, hkv, d, bs, seed=hq * d, q_dtype=q_type(kind, hq),
                                                   q_spread=3.0 if cap else 1.0)
    t = q.shape[0]
    slopes = 2.0 ** -torch.arange(1, hq + 1).float() if alibi else None
    starts = None
    if documents:  # documents of 37 keys; one token's document starts behind it: it sees nothing (or its prefix's rest)
        pos = torch.cat([torch.arange(c, c + n) for c, n in seqs])
        starts = (pos // 37 * 37).to(torch.int32)
        starts[t // 2] = 1 << 20
    want = reference(q, keys, values, table, seqs, bs, window, cap, slopes, starts, prefix)
    out = torch.full((t + 3, hq, d), float("nan"), dtype=q.dtype, device="cuda")
    out[t:] = 5.0
    wide = torch.cat([q, torch.zeros(3, hq, d, dtype=q.dtype)]).cuda()  # three rows behind the last sequence
    more = {"softcap": cap, "window": window, "alibi_slopes": None if slopes is None else slopes.cuda(), "out": out,
            "key_starts": None if starts is None else torch.cat([starts, starts[:3].new_zeros(3)]).cuda(),
            "prefix_lens": None if prefix is None else torch.tensor(prefix).cuda()}
    got = prefill_attend(wide, kv, cu.cuda(), lengths.cuda(), sm_scale(d), **more)
    assert got is out and (out[t:] == 5.0).all()
    assert_within(out[:t], want, q.dtype, values.abs().max().item(), product_bits(kind, q.dtype))
    if documents:
        assert (out[t // 2] == 0).all()
    assert _lib.device_error() == 0
    again = prefill_attend(wide, kv, cu.cuda(), lengths.cuda(), sm_scale(d), **{**more, "out": None}, tokens=int(lengths.max()))
    assert_within(again[:t], want, q.dtype, values.abs().max().item(), product_bits(kind, q.dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
def test_positions_strides_and_a_padded_batch(kind):
    """Positions that are not the sequence's last (padding tokens sit at -1 and get zeros), q as a strided view."""
    from bpt_b200.kernels.prefill_attention import prefill_attend

    seqs = [(20, 12), (0, 12)]
    kv, keys, values, q, table, cu, lengths = case(kind, seqs, 8, 2, 64, 16, seed=1)
    positions = torch.tensor([3, 31, 7, 7, 0, 25, -1, 30, 12, 100, 1, 2, 0, 1, 2, 3, 4, -1, -1, -1, -5, 11, 9, 8])
    want = reference(q, keys, values, table, seqs, 16, positions=positions, window=9)
    fused = torch.zeros(24, 12, 80, dtype=q.dtype)
    fused[:, 2:10, 8:72] = q
    view = fused.cuda()[:, 2:10, 8:72]
    assert view.stride() == (960, 80, 1)
    got = prefill_attend(view, kv, cu.cuda(), lengths.cuda(), sm_scale(64), positions=positions.cuda(), window=9)
    assert_within(got, want, q.dtype, values.abs().max().item(), product_bits(kind, q.dtype))
    assert (got[6] == 0).all() and (got[20] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
def test_what_no_query_sees_is_not_read(kind):
    from bpt_b200.kernels.prefill_attention import prefill_attend

    seqs = [(100, 30), (0, 75)]
    kv, keys, values, q, table, cu, lengths = case(kind, seqs, 4, 2, 128, 16, seed=2)
    seen = torch.zeros(kv.num_blocks, 16, dtype=torch.bool)
    for b, (ctx, new) in enumerate(seqs):
        for j in range(max(0, ctx - 39), ctx + new):
            seen[table[b, j // 16], j % 16] = True
    for pool in (kv.k_pool, kv.v_pool):
        if kind in DTYPES:
            pool[~seen.cuda()] = float("nan")
        elif kind == "fp8":
            pool[~seen.cuda()] = 0x7F
    if kind == "int8":
        kv.k_scale[~seen.cuda()] = float("nan")
        kv.v_scale[~seen.cuda()] = float("inf")
    want = reference(q, keys, values, table, seqs, 16, window=40)
    got = prefill_attend(q.cuda(), kv, cu.cuda(), lengths.cuda(), sm_scale(128), window=40)
    assert_within(got, want, q.dtype, values.abs().max().item(), product_bits(kind, q.dtype))


@pytest.mark.gpu
def test_bad_blocks_are_left_out_and_recorded():
    from bpt_b200 import _lib
    from bpt_b200.kernels.prefill_attention import prefill_attend

    for bs in (8, 16):
        seqs = [(40, 24)]
        kv, keys, values, q, table, cu, lengths = case("bf16", seqs, 4, 2, 128, bs, seed=3)
        bad = table.clone()
        bad[0, 1] = kv.num_blocks + 5
        kv.block_table = bad.cuda()
        assert _lib.device_error() == 0
        got = prefill_attend(q.cuda(), kv, cu.cuda(), lengths.cuda(), sm_scale(128))
        assert _lib.device_error() == 2
        k, v = (x[table[0].long()].flatten(0, 1) for x in (keys, values))
        for i in range(24):
            keep = [j for j in range(41 + i) if j // bs != 1]
            want = attention_row(q[i].double(), k[keep], v[keep], 0, 0, len(keep), sm_scale(128))
            assert_within(got[i], want, q.dtype, values.abs().max().item(), 8)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["bf16", "fp8"])
def test_long_ragged_batch_equals_the_decode_read(kind):
    """Every last token of a ragged batch, read by decode too; and a large batch of many short sequences."""
    from bpt_b200.kernels.kv_attention import attend
    from bpt_b200.kernels.prefill_attention import prefill_attend

    seqs = [(i * 37 % 200, 1 + i * 13 % 90) for i in range(70)]
    kv, keys, values, q, table, cu, lengths = case(kind, seqs, 8, 2, 128, 16, seed=4, q_dtype=torch.bfloat16)
    got = prefill_attend(q.cuda(), kv, cu.cuda(), lengths.cuda(), sm_scale(128), softcap=30.0)
    last = (cu[1:] - 1).long()
    want = attend(q[last].cuda(), kv, lengths.cuda(), sm_scale(128), softcap=30.0)
    vmax = values.abs().max().item()
    assert_within(got[last.cuda()], want.double().cpu(), q.dtype, vmax, product_bits(kind, q.dtype))
    rows = torch.cat([torch.arange(cu[b], cu[b + 1]) for b in (0, 31, 32, 69)])
    full = reference(q, keys, values, table, seqs, 16, softcap=30.0)
    assert_within(got[rows.cuda()], full[rows], q.dtype, vmax, product_bits(kind, q.dtype))


@pytest.mark.gpu
def test_graphs_do_not_share_a_workspace():
    from bpt_b200.kernels.prefill_attention import prefill_attend

    side, calls = torch.cuda.Stream(), []
    for seed in (5, 6):
        seqs = [(3000, 5)]
        kv, _, _, q, _, cu, lengths = case("bf16", seqs, 4, 2, 128, 16, seed=seed)
        args = (q.cuda(), kv, cu.cuda(), lengths.cuda(), sm_scale(128))
        want = prefill_attend(*args)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = prefill_attend(*args)
        calls.append((graph, out, want, torch.cuda.Stream(), args))
    for _ in range(20):
        for graph, _, _, stream, _ in calls:
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for _, out, want, _, _ in calls:
        assert torch.equal(out, want)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
def test_append_then_prefill_then_decode(kind):
    """The operators as they are used: a prompt in two chunks, then a decode step, each appended with its rotation and read
    back, against the same sequence in 64 bits over what the cache holds."""
    from bpt_b200.kernels.kv_attention import PagedQuantKV, attend
    from bpt_b200.kernels.kv_write import rope_kv_append, rope_table
    from bpt_b200.kernels.prefill_attention import prefill_attend

    hq, hkv, d, bs, dt = 8, 2, 128, 16, torch.bfloat16 if kind != "f16" else torch.float16
    g = torch.Generator().manual_seed(7)
    table, blocks = page_table([90], bs, g)
    kv, _, _ = make_cache(kind, blocks, bs, hkv, d, table, g)
    cos, sin = rope_table(128, d, 1e4)
    done = 0
    for n in (50, 30, 1):
        qkv = torch.randn(n, hq + 2 * hkv, d, generator=g).to(dt).cuda()
        pos = torch.arange(done, done + n, dtype=torch.int32, device="cuda")
        q = rope_kv_append(qkv[:, :hq], qkv[:, hq : hq + hkv], qkv[:, hq + hkv :], kv, pos, cos, sin,
                           kv.block_table[0, (pos // bs).long()], pos % bs)
        done += n
        length = torch.tensor([done], dtype=torch.int32, device="cuda")
        if n > 1:
            got = prefill_attend(q, kv, torch.tensor([0, n], dtype=torch.int32, device="cuda"), length, sm_scale(d))
        else:
            got = attend(q, kv, length, sm_scale(d), out=torch.empty_like(q), softcap=1e4)
        read = []
        for pool, scale in ((kv.k_pool, kv.k_scale), (kv.v_pool, kv.v_scale)):
            x = pool.cpu()
            x = (x.view(torch.float8_e4m3fn) if kind == "fp8" else x).double()
            x = x * (scale.cpu().double()[..., None] if kind == "int8" else scale)
            read.append(x[table[0].long()].flatten(0, 1))
        # softcap 1e4 leaves scores of a few units as they are to one part in 1e7
        want = torch.stack([attention_row(q[i].double().cpu(), read[0], read[1], done - n + i, 0, done - n + i + 1, sm_scale(d))
                            for i in range(n)])
        assert_within(got, want, dt, read[1].abs().max().item(), 8)
    assert isinstance(kv, PagedQuantKV)


def test_refusals_need_no_gpu():
    from bpt_b200 import _lib

    L = _lib.lib()

    def call(**kw):
        a = {"q": 64, "qd": 2, "qt": 512, "qh": 128, "kp": 64, "vp": 64, "kind": 4, "ks": 1.0, "vs": 1.0, "kss": None, "vss": None,
             "bt": 64, "bts": 4, "btw": 4, "cu": 64, "len": 64, "pos": None, "starts": None, "prefix": None, "slopes": None,
             "cap": 0.0, "window": 0, "T": 20000, "B": 2, "Hq": 4, "Hkv": 2, "D": 128, "bs": 16, "nb": 8, "tokens": 64,
             "scale": 1.0, "out": 64, "ws": None, "wsb": 0, "flags": 0, "stream": None} | kw
        return _lib.paged_prefill(*(0 if x is None else x for x in a.values()))

    assert call(T=0) == _lib.OK and call(B=0) == _lib.OK
    for name in ("q", "kp", "vp", "bt", "cu", "len", "out"):
        assert call(**{name: None}) == _lib.ERR_INVALID and b"null" in L.bpt_last_error()
    assert call(qd=0) == _lib.ERR_INVALID and call(qd=1) == _lib.ERR_UNSUPPORTED  # f16 queries over bf16 pages
    assert call(D=80) == _lib.ERR_UNSUPPORTED and call(bs=48) == _lib.ERR_UNSUPPORTED
    assert call(Hq=5) == _lib.ERR_INVALID and call(window=-1) == _lib.ERR_INVALID and call(cap=-1.0) == _lib.ERR_INVALID
    assert call(tokens=0) == _lib.ERR_INVALID and call(qt=516) == _lib.ERR_ALIGNMENT and call(out=72) == _lib.ERR_ALIGNMENT
    assert call(kind=2) == _lib.ERR_INVALID and call(T=-1) == _lib.ERR_INVALID and call(B=1 << 20) == _lib.ERR_INVALID
    few = {"T": 4, "tokens": 4000, "btw": 4000, "bts": 4000}
    assert L.bpt_paged_prefill_workspace_bytes(4, 2, 4, 2, 128, 4, 4000) > 0
    assert call(**few) == _lib.ERR_WORKSPACE and call(**few, ws=64, wsb=64) == _lib.ERR_WORKSPACE
    assert call(**few, ws=72, wsb=1 << 40) == _lib.ERR_ALIGNMENT


@pytest.mark.gpu
def test_python_refusals():
    from bpt_b200.kernels.prefill_attention import prefill_attend

    kv, _, _, q, _, cu, lengths = case("bf16", [(0, 4)], 4, 2, 64, 16)
    q, cu, lengths = q.cuda(), cu.cuda(), lengths.cuda()

    def refused(q=q, cu=cu, lengths=lengths, **kw):
        with pytest.raises(ValueError):
            prefill_attend(q, kv, cu, lengths, 0.1, **kw)

    refused(q=q.cpu())
    refused(q=q.float())
    refused(q=q.half())
    refused(q=q[:, :3])
    refused(q=q[0])
    refused(cu=cu[:1])
    refused(cu=cu.float())
    refused(lengths=lengths.repeat(2))
    refused(positions=torch.zeros(3, dtype=torch.int32, device="cuda"))
    refused(key_starts=torch.zeros(3, dtype=torch.int32, device="cuda"))
    refused(prefix_lens=torch.zeros(2, dtype=torch.int32, device="cuda"))
    refused(alibi_slopes=torch.zeros(2, device="cuda"))
    refused(out=torch.empty(4, 4, 64, device="cuda"))
    refused(window=-2)
