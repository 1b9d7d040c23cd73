"""The quantized KV-cache write path on sm_100a.

- `quantize_kv_paged(k, v, kv, write_blocks, write_offsets)`: quantize this step's keys and values
  [B, Hkv, Q, D] to FP8 or INT8 and scatter them into a `PagedQuantKV` pool. The write of
  `PagedKVCache.update` (`src/fastserve/engine/kv_cache.py:150-161`) with the store of `kv/quant.py:40-48`
  in front of it.
- `rope_kv_append` and `store_kv_paged`: the same slots of a paged cache of any kind, with rotation (and QK-norm) on the way
  or as the keys and values come.
- `quantize_kv(k, v, bits, group)`: the reference's `kernels/reference.py:132-160` (KIVI codes and grids) on
  the GPU, returning a `QuantKV`; `quantize_kv_into` writes whole groups into an existing cache, as
  `QuantizedKVCache._append` does (`integration/kv_cache.py:139-158`).
"""

from __future__ import annotations

import torch

from bpt_b200 import _lib
from bpt_b200._lib import FLAG_PDL, addr, as_int32, check, dtype_code, lib, on_device, ptr, require_cuda, stream_of
from bpt_b200.kernels.kv_attention import PagedQuantKV, QuantKV, pool_format


def quantize_kv_paged(k: torch.Tensor, v: torch.Tensor, kv: PagedQuantKV, write_blocks: torch.Tensor,
                      write_offsets: torch.Tensor) -> None:
    """Store k, v [B, Hkv, Q, D] at slot write_offsets[b, i] of block write_blocks[b, i] (int32 [B, Q])."""
    device = require_cuda(k, v, kv.k_pool, write_blocks, write_offsets)
    if k.shape != v.shape or k.dim() != 4:
        raise ValueError(f"k and v must both be [B, Hkv, Q, D], got {tuple(k.shape)} and {tuple(v.shape)}")
    if k.stride() != v.stride() or k.stride(-1) != 1:
        k, v = k.contiguous(), v.contiguous()
    b, hkv, q, d = k.shape
    nb, bs, hkv_pool, d_pool = kv.k_pool.shape
    if (hkv, d) != (hkv_pool, d_pool):
        raise ValueError(f"k has {hkv} heads of {d}, the pool {hkv_pool} of {d_pool}")
    wb = write_blocks.to(torch.int32).contiguous()
    wo = write_offsets.to(torch.int32).contiguous()
    if tuple(wb.shape) != (b, q) or tuple(wo.shape) != (b, q):
        raise ValueError(f"write_blocks / write_offsets must be [{b}, {q}]")
    if kv.kind == "fp8":
        code, ks, vs, kss, vss = _lib.KV_FP8, float(kv.k_scale), float(kv.v_scale), None, None
    elif kv.kind == "int8":
        code, ks, vs, kss, vss = _lib.KV_INT8, 1.0, 1.0, kv.k_scale, kv.v_scale
    else:
        raise ValueError(f"kind must be 'fp8' or 'int8', got {kv.kind!r}")
    st = lib().bpt_paged_kv_write(
        ptr(k), ptr(v), dtype_code(k.dtype), k.stride(0), k.stride(1), k.stride(2), b, hkv, q, d, ptr(wb), ptr(wo),
        ptr(kv.k_pool), ptr(kv.v_pool), code, ks, vs, ptr(kss), ptr(vss), bs, nb, stream_of(device))
    check(st, "quantize_kv_paged")


def rope_table(positions: int, rotary_dim: int, theta: float = 1e6, device="cuda") -> tuple[torch.Tensor, torch.Tensor]:
    """cos, sin [positions, rotary_dim / 2] in fp32 for angles p * theta^(-2i / rotary_dim) (engine/rope.py:12-28), from
    angles in 64 bits: in 32, position 100,000 is off by up to 0.004 radians."""
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be even, got {rotary_dim}")
    inv = float(theta) ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64, device=device) / rotary_dim)
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * inv
    return angle.cos().float(), angle.sin().float()


def _aligned_rows(x: torch.Tensor) -> tuple[torch.Tensor, tuple]:
    """x [T, H, D] and its strides, or a copy's whose rows start on 16 bytes."""
    unit, stride = 16 // x.element_size(), x.stride()
    if stride[2] != 1 or stride[0] % unit or stride[1] % unit or x.data_ptr() % 16:
        x = x.clone(memory_format=torch.contiguous_format)
        stride = x.stride()
    return x, stride


def rope_kv_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, kv: PagedQuantKV, positions: torch.Tensor,
                   cos: torch.Tensor, sin: torch.Tensor, write_blocks: torch.Tensor, write_offsets: torch.Tensor, *,
                   q_norm: torch.Tensor | None = None, k_norm: torch.Tensor | None = None, eps: float = 1e-6,
                   interleaved: bool = False, q_out: torch.Tensor | None = None, pdl: bool = False) -> torch.Tensor:
    """Rotate T new tokens' q [T, Hq, D] and k [T, Hkv, D] and store k, v [T, Hkv, D] in the pools; returns the rotated q.

    positions, write_blocks, write_offsets: [T] whole numbers: each token's row of cos / sin (fp32 [positions, R / 2]; the
    first R dims rotate, the rest pass) and the slot that receives its key and value; slots of one call must be distinct. A
    token with write_blocks -1 is padding: nothing of it is read, stored or written to q_out. q, k and v may be views of one
    projection's output (any token and head strides). `q_norm` / `k_norm` [D]: RMSNorm weights applied per head before
    the rotation. `interleaved`: dims 2i and 2i + 1 rotate together instead of i and i + R / 2. Rows are rounded once, from
    fp32, to q_out's type (q's) and to the cache's format.
    """
    device = require_cuda(q, k, v, kv.k_pool, kv.v_pool, positions, cos, sin, write_blocks, write_offsets, q_norm, k_norm,
                          q_out)
    q_shape, k_shape, dtype = q.shape, k.shape, q.dtype
    if len(q_shape) != 3 or len(k_shape) != 3 or k_shape != v.shape or q_shape[::2] != k_shape[::2]:
        raise ValueError(f"q must be [T, Hq, D], k and v [T, Hkv, D], got {tuple(q_shape)}, {tuple(k_shape)} and "
                         f"{tuple(v.shape)}")
    if dtype != k.dtype or dtype != v.dtype:
        raise ValueError(f"q, k and v must share a dtype, got {dtype}, {k.dtype} and {v.dtype}")
    t, hq, d = q_shape
    hkv = k_shape[1]
    code, ks, vs, kss, vss, nb, bs, pool_heads, pool_dim = pool_format(kv)
    if hkv != pool_heads or d != pool_dim:
        raise ValueError(f"k has {hkv} heads of {d}, the pool {pool_heads} of {pool_dim}")
    table = cos.shape
    if len(table) != 2 or table != sin.shape or cos.dtype != torch.float32 or sin.dtype != torch.float32:
        raise ValueError("cos and sin must be float32 [positions, rotary / 2]")
    for w in (q_norm, k_norm):
        if w is not None and (w.shape != (d,) or w.dtype != dtype):
            raise ValueError(f"norm weights must be [{d}] in {dtype}")
    if positions.numel() != t or write_blocks.numel() != t or write_offsets.numel() != t:
        raise ValueError(f"positions, write_blocks and write_offsets must hold {t} entries")
    if q_out is not None and (q_out.shape != q_shape or q_out.dtype != dtype or not q_out.is_contiguous()):
        raise ValueError(f"q_out must be a contiguous [{t}, {hq}, {d}] tensor of {dtype}")
    with on_device(device):
        if q_out is None:
            q_out = torch.empty(q_shape, dtype=dtype, device=device)
        q, q_stride = _aligned_rows(q)
        k, k_stride = _aligned_rows(k)
        v, v_stride = _aligned_rows(v)
        cos, sin = cos.contiguous(), sin.contiguous()
        q_norm = q_norm if q_norm is None else q_norm.contiguous()
        k_norm = k_norm if k_norm is None else k_norm.contiguous()
        pos, wb, wo = as_int32(positions), as_int32(write_blocks), as_int32(write_offsets)
        st = _lib.rope_kv_append(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), dtype_code(dtype), q_stride[0], q_stride[1], k_stride[0], k_stride[1],
            v_stride[0], v_stride[1], t, hq, hkv, d, 2 * table[1], pos.data_ptr(), cos.data_ptr(), sin.data_ptr(), table[0],
            bool(interleaved), addr(q_norm), addr(k_norm), float(eps), q_out.data_ptr(), wb.data_ptr(), wo.data_ptr(),
            kv.k_pool.data_ptr(), kv.v_pool.data_ptr(), code, ks, vs, addr(kss), addr(vss), bs, nb,
            FLAG_PDL if pdl else 0, stream_of(device))
    check(st, "rope_kv_append")
    return q_out


def store_kv_paged(k: torch.Tensor, v: torch.Tensor, kv: PagedQuantKV, write_blocks: torch.Tensor,
                   write_offsets: torch.Tensor) -> None:
    """Store k, v [B, Hkv, Q, D] (fp32, f16 or bf16) as they come at the slots write_blocks / write_offsets [B, Q] of a paged
    cache, rounded once: the store of `rope_kv_append` alone, for pages that `quantize_kv_paged` does not write (16-bit ones).

    A token with write_blocks -1 is padding and is not stored; a slot outside the pool is not written and is recorded.
    """
    device = require_cuda(k, v, kv.k_pool, kv.v_pool, write_blocks, write_offsets)
    if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype:
        raise ValueError(f"k and v must both be [B, Hkv, Q, D] of one dtype, got {tuple(k.shape)} in {k.dtype} and "
                         f"{tuple(v.shape)} in {v.dtype}")
    b, hkv, q, d = k.shape
    code, ks, vs, kss, vss, nb, bs, pool_heads, pool_dim = pool_format(kv)
    if hkv != pool_heads or d != pool_dim:
        raise ValueError(f"k has {hkv} heads of {d}, the pool {pool_heads} of {pool_dim}")
    if write_blocks.shape != (b, q) or write_offsets.shape != (b, q):
        raise ValueError(f"write_blocks / write_offsets must be [{b}, {q}]")
    with on_device(device):
        k, k_stride = _aligned_rows(k.transpose(1, 2).flatten(0, 1))  # [B * Q, Hkv, D]
        v, v_stride = _aligned_rows(v.transpose(1, 2).flatten(0, 1))
        wb, wo = as_int32(write_blocks), as_int32(write_offsets)
        st = _lib.rope_kv_append(
            0, k.data_ptr(), v.data_ptr(), dtype_code(k.dtype), 0, 0, k_stride[0], k_stride[1], v_stride[0], v_stride[1], b * q,
            0, hkv, d, 0, 0, 0, 0, 0, False, 0, 0, 0.0, 0, wb.data_ptr(), wo.data_ptr(), kv.k_pool.data_ptr(),
            kv.v_pool.data_ptr(), code, ks, vs, addr(kss), addr(vss), bs, nb, 0, stream_of(device))
    check(st, "store_kv_paged")


def empty_quant_kv(batch: int, kv_heads: int, tokens: int, head_dim: int, bits: int, group: int, device,
                   dtype=torch.bfloat16) -> QuantKV:
    """A zeroed KIVI cache laid out as QuantizedKVCache allocates one (integration/kv_cache.py:84-107)."""
    if bits == 16:
        shape = (batch, kv_heads, tokens, head_dim)
        return QuantKV(16, group, torch.zeros(shape, dtype=dtype, device=device), torch.zeros(shape, dtype=dtype, device=device))
    codes = (batch, kv_heads, tokens, head_dim // 2 if bits == 4 else head_dim)

    def grid(*shape):
        return torch.zeros(shape, dtype=torch.float16, device=device)

    return QuantKV(bits, group, torch.zeros(codes, dtype=torch.uint8, device=device),
                   torch.zeros(codes, dtype=torch.uint8, device=device), grid(batch, kv_heads, tokens // group, head_dim),
                   grid(batch, kv_heads, tokens // group, head_dim), grid(batch, kv_heads, tokens),
                   grid(batch, kv_heads, tokens))


def quantize_kv_into(k: torch.Tensor, v: torch.Tensor, kv: QuantKV, t0: int) -> None:
    """Quantize whole key groups k, v [B, Hkv, T, D] into `kv` at token offset t0 (a group boundary)."""
    device = require_cuda(k, v, kv.k_codes)
    if kv.bits == 16:
        kv.k_codes[:, :, t0 : t0 + k.shape[2]] = k
        kv.v_codes[:, :, t0 : t0 + v.shape[2]] = v
        return
    b, h, t, d = k.shape
    if t % kv.group:
        raise ValueError(f"{t} tokens are not a whole number of groups of {kv.group}")
    k, v = k.contiguous(), v.contiguous()
    st = lib().bpt_kivi_quantize(
        ptr(k), ptr(v), dtype_code(k.dtype), b, h, t, d, kv.bits, kv.group, ptr(kv.k_codes), ptr(kv.v_codes),
        ptr(kv.k_scale), ptr(kv.k_zero), ptr(kv.v_scale), ptr(kv.v_zero), kv.k_codes.shape[2], kv.k_scale.shape[2], t0,
        stream_of(device))
    check(st, "quantize_kv")


def quantize_kv(k: torch.Tensor, v: torch.Tensor, bits: int, group: int = 32) -> QuantKV:
    """reference.quantize_kv on the GPU: k, v [B, Hkv, T, D] -> a QuantKV holding exactly T tokens."""
    if bits == 16:
        return QuantKV(16, group, k.contiguous(), v.contiguous())
    if bits not in (4, 8):
        raise ValueError(f"bits must be 4, 8 or 16, got {bits}")
    b, h, t, d = k.shape
    if t % group:
        raise ValueError(f"{t} tokens are not a whole number of groups of {group}")
    kv = empty_quant_kv(b, h, t, d, bits, group, k.device)
    quantize_kv_into(k, v, kv, 0)
    return kv
