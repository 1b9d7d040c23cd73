"""Stores of new tokens into 16-bit pages without rotation, at slots inside and outside the pool."""

import math
from types import SimpleNamespace

import pytest
import torch


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("q_len", [1, 5])
def test_a_slot_outside_a_16_bit_pool_is_not_written(kind, dtype, q_len):
    """Write slots outside the pool (a caller's own metadata) leave the pool as it is and are recorded, as over 8-bit pages;
    -1 is padding. The other tokens are stored, rounded once."""
    from bpt_b200 import _lib
    from bpt_b200.integration import PagedQuantizedKVCache

    cache = PagedQuantizedKVCache(SimpleNamespace(num_layers=1, num_kv_heads=2, head_dim=64), num_blocks=8, block_size=16, kind=kind)
    for name in ("a", "b", "c"):
        cache.reserve(name, 20)
    positions = torch.arange(3, 3 + q_len).repeat(3, 1)
    meta = cache.prepare(["a", "b", "c"], positions.cuda())
    g = torch.Generator().manual_seed(q_len)
    q, k, v = (torch.randn(3, h, q_len, 64, generator=g).to(dtype).cuda() for h in (4, 2, 2))
    assert _lib.device_error() == 0
    kv = cache.layers[0]
    for block, offset, code in ((-1, 0, 0), (8, 0, 2), (0, 16, 3)):
        for pool in (kv.k_pool, kv.v_pool):
            pool.fill_(7.0)
        blocks, offsets = meta.write_blocks.clone(), meta.write_offsets.clone()
        blocks[1], offsets[1] = block, offset
        bad = SimpleNamespace(**{**meta.__dict__, "write_blocks": blocks, "write_offsets": offsets})
        cache._append(0, k, v, bad)
        assert _lib.device_error() == code
        for pool, x in ((kv.k_pool, k), (kv.v_pool, v)):
            want = torch.full(pool.shape, 7.0, dtype=pool.dtype, device="cuda")
            for b in (0, 2):
                for i in range(q_len):
                    want[meta.write_blocks[b, i], meta.write_offsets[b, i]] = x[b, :, i].to(pool.dtype)
            assert torch.equal(pool, want)
    assert not math.isnan(float(cache.attend(0, q, k, v, meta, 0.125).float().sum()))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["bf16", "f16", "fp8", "int8"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("b,q_len,hkv,d", [(1, 1, 1, 64), (3, 7, 5, 128), (2, 300, 8, 256)])
def test_store_equals_the_append_at_angle_zero(kind, dtype, b, q_len, hkv, d):
    """Cos 1 and sin 0 leave keys as they are: the rotating store is the same kernel's other half."""
    from bpt_b200.kernels.kv_write import rope_kv_append, store_kv_paged
    from tests.test_gpu_paged_append import pool

    g = torch.Generator().manual_seed(d + q_len)
    k, v = (torch.randn(b, q_len, hkv, d, generator=g).to(dtype).cuda().transpose(1, 2) for _ in range(2))
    blocks = -(-b * q_len // 16) + 2
    slots = torch.randperm(blocks * 16, generator=g)[: b * q_len].view(b, q_len).cuda()
    kv, twin = pool(kind, blocks, 16, hkv, d), pool(kind, blocks, 16, hkv, d)
    store_kv_paged(k, v, kv, slots // 16, slots % 16)
    one, zero = torch.ones(1, d // 2, device="cuda"), torch.zeros(1, d // 2, device="cuda")
    tokens = [x.transpose(1, 2).reshape(-1, hkv, d) for x in (k, v)]
    rope_kv_append(tokens[0], *tokens, twin, torch.zeros(b * q_len, dtype=torch.int32, device="cuda"), one, zero, slots // 16, slots % 16)
    for name in ("k_pool", "v_pool") + (("k_scale", "v_scale") if kind == "int8" else ()):
        assert torch.equal(getattr(kv, name), getattr(twin, name))


def test_store_refusals_need_no_gpu():
    from bpt_b200 import _lib

    L = _lib.lib()

    def call(**kw):
        a = {"q": 0, "k": 64, "v": 64, "dtype": 2, "qs": 0, "qh": 0, "ks": 256, "kh": 128, "vs": 256, "vh": 128, "T": 4, "Hq": 0,
             "Hkv": 2, "D": 128, "rotary": 0, "pos": 0, "cos": 0, "sin": 0, "rows": 0, "il": 0, "qn": 0, "kn": 0, "eps": 0.0,
             "out": 0, "wb": 64, "wo": 64, "kp": 64, "vp": 64, "kind": 4, "ksc": 1.0, "vsc": 1.0, "kss": 0, "vss": 0, "bs": 16,
             "nb": 4, "flags": 0, "stream": 0} | kw
        return _lib.rope_kv_append(*a.values())

    assert call(T=0) == _lib.OK
    for name in ("k", "v", "wb", "wo", "kp", "vp"):
        assert call(**{name: 0}) == _lib.ERR_INVALID and b"null" in L.bpt_last_error()
    for bad in ({"rotary": 128}, {"pos": 64}, {"qn": 64}, {"kn": 64}):
        assert call(**bad) == _lib.ERR_INVALID and b"without queries" in L.bpt_last_error()
    assert call(Hq=-1, q=64, pos=64, cos=64, sin=64, out=64, rotary=128, rows=8) == _lib.ERR_INVALID
    assert call(Hkv=0) == _lib.ERR_INVALID and call(D=80) == _lib.ERR_UNSUPPORTED and call(ks=260) == _lib.ERR_ALIGNMENT


@pytest.mark.gpu
def test_store_python_refusals():
    from bpt_b200.kernels.kv_write import store_kv_paged
    from tests.test_gpu_paged_append import pool

    kv = pool("bf16", 2, 16, 2, 64)
    k, at = torch.zeros(1, 2, 3, 64, device="cuda"), torch.zeros(1, 3, dtype=torch.int32, device="cuda")
    for args in ((k[0], k[0], kv, at, at), (k, k.half(), kv, at, at), (k[..., :32], k[..., :32], kv, at, at), (k, k, kv, at[:, :2], at),
                 (k, k, kv, at, at.float()), (k.double(), k.double(), kv, at, at), (k.cpu(), k.cpu(), kv, at, at)):
        with pytest.raises(ValueError):
            store_kv_paged(*args)
