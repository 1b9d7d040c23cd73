"""rope_kv_append against the rotation and the stores in 64 bits: every cache format, dtype and head dim, partial and
interleaved rotation, strided inputs, padding tokens, far positions; the refusals run on the CPU."""

import pytest
import torch

from tests.paged_reference import DTYPES, KINDS


def rotate(x, cos, sin, interleaved):
    """x [T, H, R] double, cos / sin [T, R / 2] double."""
    r = x.shape[-1]
    i = torch.arange(r // 2)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + r // 2)
    y = torch.empty_like(x)
    c, s = cos[:, None], sin[:, None]
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., b] * c + x[..., a] * s
    return y


def reference(x, w, eps, cos, sin, interleaved):
    x = x.double()
    if w is not None:
        x = x * (x.square().mean(-1, keepdim=True) + eps).rsqrt() * w.double()
    r = 2 * cos.shape[1]
    return torch.cat([rotate(x[..., :r], cos, sin, interleaved), x[..., r:]], -1)


def inputs(t, hq, hkv, d, dtype, g, strided):
    if strided:  # the fused projection's output with slack after each row
        big = torch.randn(t, (hq + 2 * hkv) * d + 16, generator=g).to(dtype).cuda()
        return [big[:, a * d : b * d].view(t, -1, d) for a, b in ((0, hq), (hq, hq + hkv), (hq + hkv, hq + 2 * hkv))]
    return [torch.randn(t, n, d, generator=g).to(dtype).cuda() for n in (hq, hkv, hkv)]


def pool(kind, nb, bs, hkv, d, device="cuda"):
    from bpt_b200.kernels.kv_attention import PagedQuantKV

    table = torch.zeros(1, 1, dtype=torch.int32, device=device)
    shape = (nb, bs, hkv, d)
    if kind in DTYPES:
        return PagedQuantKV(kind, *(torch.full(shape, 7.0, dtype=DTYPES[kind], device=device) for _ in range(2)), table, bs)
    if kind == "fp8":
        return PagedQuantKV(kind, *(torch.full(shape, 9, dtype=torch.uint8, device=device) for _ in range(2)), table, bs, 1 / 64,
                            1 / 32)
    return PagedQuantKV(kind, *(torch.full(shape, 9, dtype=torch.int8, device=device) for _ in range(2)), table, bs,
                        *(torch.full(shape[:3], 0.5, dtype=torch.float16, device=device) for _ in range(2)))


def check_rows(got, want, dtype):
    """One rounding to dtype of a value that fp32 gives to within 2^-20 of the row's largest."""
    half = torch.finfo(dtype).eps / 2
    off = (got.double().cpu() - want).abs() - half * want.abs() - 2.0**-20 * want.abs().amax(-1, keepdim=True)
    assert (off <= 0).all(), off.max()


def check_store(kv, name, slots, want, untouched):
    p, s = getattr(kv, f"{name}_pool").cpu(), getattr(kv, f"{name}_scale")
    flat = p.view(-1, *p.shape[2:])
    if kv.kind in DTYPES:
        check_rows(flat[slots], want, DTYPES[kv.kind])
    elif kv.kind == "fp8":
        got = flat[slots].view(torch.float8_e4m3fn).double() * s
        y = want.clamp(-448 * s, 448 * s)
        # half a step of E4M3 (2^-4 of the value; 2^-10 of the scale among its subnormals), and fp32's own 2^-20
        off = (got - y).abs() - torch.maximum(y.abs() * 2**-4, torch.tensor(s * 2.0**-10).double()) - 2.0**-20 * want.abs().amax(-1, keepdim=True)
        assert (off <= 0).all(), off.max()
    else:
        scale = s.cpu().view(-1, s.shape[2])[slots].double()
        amax = want.abs().amax(-1)
        # the scale is one rounding to f16 of max / 127; a code is half a step off, and what the scale's rounding takes off
        # the largest code: it saturates at 127, 2^-11 * 127 = 0.06 of a step short
        assert ((scale - amax / 127).abs() <= 2.0**-11 * amax / 127 + 2.0**-25 + 2.0**-19 * amax / 127).all()
        off = (flat[slots].double() * scale[..., None] - want).abs() - (0.5 + 0.07) * scale[..., None]
        assert (off <= 0).all(), off.max()
        rest = s.cpu().view(-1, s.shape[2])[untouched]
        assert (rest == 0.5).all()
    assert (flat[untouched].float() == (7.0 if kv.kind in DTYPES else 9)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("t,hq,hkv,d,rotary,interleaved,norm,dtype,bs", [
    (1, 16, 8, 128, 128, False, True, torch.bfloat16, 16),
    (5, 3, 1, 64, 32, True, False, torch.float16, 8),
    (33, 14, 2, 64, 64, False, True, torch.bfloat16, 64),
    (7, 5, 5, 256, 64, False, True, torch.float16, 16),
    (3, 2, 1, 256, 256, True, False, torch.float32, 32),
    (2100, 7, 1, 128, 112, False, False, torch.bfloat16, 16),  # a warp takes several groups of heads
    (300, 40, 8, 128, 16, True, True, torch.float32, 16),
])
def test_append_matches_the_formula(kind, t, hq, hkv, d, rotary, interleaved, norm, dtype, bs):
    from bpt_b200 import _lib
    from bpt_b200.kernels.kv_write import rope_kv_append, rope_table

    g = torch.Generator().manual_seed(t + d)
    q, k, v = inputs(t, hq, hkv, d, dtype, g, strided=t % 2 == 1)
    nb = -(-t // bs) + 3
    kv = pool(kind, nb, bs, hkv, d)
    slots = torch.randperm(nb * bs, generator=g)
    slots, untouched = slots[:t], slots[t:]
    reach = 100_003
    positions = torch.randint(0, reach, (t,), generator=g)
    positions[0] = reach - 1
    cos, sin = rope_table(reach, rotary, 1e4)
    weights = [(1 + 0.2 * torch.randn(d, generator=g)).to(dtype) if norm else None for _ in range(2)]
    got = rope_kv_append(q, k, v, kv, positions.cuda(), cos, sin, (slots // bs).int().cuda(), (slots % bs).cuda(),
                         q_norm=weights[0].cuda() if norm else None, k_norm=weights[1].cuda() if norm else None, eps=1e-5,
                         interleaved=interleaved)
    c, s = cos.cpu()[positions].double(), sin.cpu()[positions].double()
    check_rows(got, reference(q.cpu(), weights[0], 1e-5, c, s, interleaved), dtype)
    check_store(kv, "k", slots, reference(k.cpu(), weights[1], 1e-5, c, s, interleaved), untouched)
    check_store(kv, "v", slots, v.cpu().double(), untouched)
    assert _lib.device_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
def test_padding_and_bad_tokens(kind):
    """Block -1: nothing of the token is touched. A bad slot stores nothing and rotates q; a position outside the table
    skips the token. Both are recorded."""
    from bpt_b200 import _lib
    from bpt_b200.kernels.kv_write import rope_kv_append, rope_table

    g = torch.Generator().manual_seed(1)
    q, k, v = inputs(6, 4, 2, 128, torch.bfloat16, g, strided=False)
    kv = pool(kind, 2, 16, 2, 128)
    cos, sin = rope_table(32, 128)
    out = torch.full_like(q, 3.0)
    blocks = torch.tensor([0, -1, 1, 2, 0, -7], dtype=torch.int32).cuda()
    offsets = torch.tensor([3, 0, 4, 0, 16, 0], dtype=torch.int32).cuda()
    positions = torch.tensor([1, 2**31 - 1, 32, 5, 6, 7], dtype=torch.int32).cuda()
    assert _lib.device_error() == 0
    rope_kv_append(q, k, v, kv, positions, cos, sin, blocks, offsets, q_out=out)
    assert _lib.device_error() in (2, 3, 4)
    assert (out[1] == 3).all() and (out[2] == 3).all()
    want = reference(q.cpu(), None, 0, cos.cpu()[positions.cpu().clamp(0, 31).long()].double(),
                     sin.cpu()[positions.cpu().clamp(0, 31).long()].double(), False)
    for i in (0, 3, 4, 5):
        check_rows(out[i : i + 1], want[i : i + 1], torch.bfloat16)
    rest = torch.tensor([i for i in range(32) if i != 3])
    check_store(kv, "v", torch.tensor([3]), v[:1].cpu().double(), rest)


@pytest.mark.gpu
def test_special_values_reach_the_cache():
    """Infinities and NaN stay what they are in 16-bit caches and saturate or stay NaN in E4M3; a negative zero keeps its sign."""
    from bpt_b200.kernels.kv_write import rope_kv_append, rope_table

    cos, sin = rope_table(4, 64)
    x = torch.zeros(1, 1, 128, dtype=torch.bfloat16)
    x[0, 0, 100], x[0, 0, 101], x[0, 0, 102], x[0, 0, 103], x[0, 0, 104] = float("inf"), float("-inf"), float("nan"), -0.0, 1e30
    x = x.cuda()
    at = torch.zeros(1, dtype=torch.int32, device="cuda")
    for kind in ("bf16", "fp8"):
        kv = pool(kind, 1, 16, 1, 128)
        rope_kv_append(x, x, x, kv, at, cos, sin, at, at)
        got = kv.k_pool[0, 0, 0].cpu()
        if kind == "bf16":
            put = [100, 101, 103, 104]  # bit for bit; a NaN keeps no payload
            assert torch.equal(got[put].view(torch.int16), x[0, 0, put].cpu().view(torch.int16)) and got[102].isnan()
        else:
            assert got[100:105].tolist()[:2] == [0x7E, 0xFE] and got[102].item() & 0x7F == 0x7F
            assert got[103].item() == 0x80 and got[104].item() == 0x7E


@pytest.mark.gpu
def test_append_in_a_graph_and_on_another_stream():
    from bpt_b200.kernels.kv_write import rope_kv_append, rope_table

    g = torch.Generator().manual_seed(2)
    q, k, v = inputs(8, 4, 2, 128, torch.bfloat16, g, strided=False)
    cos, sin = rope_table(64, 128)
    pos = torch.arange(8, dtype=torch.int32, device="cuda")
    blocks, offsets = torch.zeros_like(pos), pos.clone()
    want_kv = pool("bf16", 1, 16, 2, 128)
    want = rope_kv_append(q, k, v, want_kv, pos, cos, sin, blocks, offsets)
    kv, out = pool("bf16", 1, 16, 2, 128), torch.empty_like(q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        rope_kv_append(q, k, v, kv, pos, cos, sin, blocks, offsets, q_out=out, pdl=True)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want) and torch.equal(kv.k_pool, want_kv.k_pool) and torch.equal(kv.v_pool, want_kv.v_pool)


def test_refusals_need_no_gpu():
    """The C entry refuses before any launch, with a status and a message."""
    from bpt_b200 import _lib

    L = _lib.lib()

    def call(**kw):
        a = {"q": 64, "k": 64, "v": 64, "dtype": 2, "qs": 512, "qh": 128, "ks": 256, "kh": 128, "vs": 256, "vh": 128, "T": 4,
             "Hq": 4, "Hkv": 2, "D": 128, "rotary": 128, "pos": 64, "cos": 64, "sin": 64, "rows": 8, "il": 0, "qn": None,
             "kn": None, "eps": 1e-6, "out": 64, "wb": 64, "wo": 64, "kp": 64, "vp": 64, "kind": 4, "ksc": 1.0, "vsc": 1.0,
             "kss": None, "vss": None, "bs": 16, "nb": 4, "flags": 0, "stream": None} | kw
        return _lib.rope_kv_append(*(0 if x is None else x for x in a.values()))

    assert call(T=0) == _lib.OK
    assert call(T=-1) == _lib.ERR_INVALID
    for name in ("q", "k", "v", "pos", "cos", "sin", "out", "wb", "wo", "kp", "vp"):
        assert call(**{name: None}) == _lib.ERR_INVALID and b"null" in L.bpt_last_error()
    assert call(D=96) == _lib.ERR_UNSUPPORTED and b"D=96" in L.bpt_last_error()
    assert call(rotary=24) == _lib.ERR_UNSUPPORTED and call(rotary=144) == _lib.ERR_UNSUPPORTED
    assert call(rotary=0) == _lib.ERR_UNSUPPORTED
    assert call(dtype=3) == _lib.ERR_INVALID and call(kind=5) == _lib.ERR_INVALID
    assert call(kind=1, ksc=0.0) == _lib.ERR_INVALID and b"positive" in L.bpt_last_error()
    assert call(kind=2) == _lib.ERR_INVALID and b"scale pools" in L.bpt_last_error()
    assert call(q=72) == _lib.ERR_ALIGNMENT and call(ks=260) == _lib.ERR_ALIGNMENT
    assert call(rows=0) == _lib.ERR_INVALID and call(nb=0) == _lib.ERR_INVALID


@pytest.mark.gpu
def test_python_refusals():
    from bpt_b200.kernels.kv_write import rope_kv_append, rope_table

    g = torch.Generator().manual_seed(3)
    q, k, v = inputs(4, 4, 2, 128, torch.bfloat16, g, strided=False)
    kv = pool("bf16", 1, 16, 2, 128)
    cos, sin = rope_table(8, 128)
    at = torch.arange(4, dtype=torch.int32, device="cuda")
    zero = torch.zeros_like(at)
    good = [q, k, v, kv, at, cos, sin, zero, at]

    def refused(**changes):
        args = [changes.get(str(i), a) for i, a in enumerate(good)]
        with pytest.raises(ValueError):
            rope_kv_append(*args, **{n: c for n, c in changes.items() if not n.isdigit()})

    refused(**{"0": q.cpu()})
    refused(**{"0": q.half()})
    refused(**{"0": q[:3]})
    refused(**{"1": k[:, :1], "2": v[:, :1]})
    refused(**{"3": pool("bf16", 1, 16, 2, 64)})
    refused(**{"5": cos.bfloat16()})
    refused(**{"4": at[:3]})
    refused(**{"4": at.float()})
    refused(q_norm=torch.ones(64, dtype=torch.bfloat16, device="cuda"))
    refused(q_out=torch.empty(4, 4, 128, device="cuda"))
