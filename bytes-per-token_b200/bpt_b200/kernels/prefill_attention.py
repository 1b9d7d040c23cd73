"""Prefill attention over a paged cache: the new tokens of a ragged batch over their sequences' pages (`csrc/paged_prefill.cu`).

`prefill_attend` is the read that follows `rope_kv_append` when sequences bring more than one new token: prompts, chunks of
long prompts, speculated tokens. The reference gathers every page into a contiguous tensor and runs a masked attention over it
(`engine/kv_cache.py:165-169`, `engine/attention.py:12-31`); here the pages are read in place, one pass with an online softmax.
"""

from __future__ import annotations

import torch

from bpt_b200 import _lib
from bpt_b200._lib import FLAG_PDL, addr, as_int32, check, dtype_code, lib, on_device, require_cuda, stream_of
from bpt_b200.kernels.kv_attention import PagedQuantKV, _row_tensor, _scratch, block_table_of, pool_format


def prefill_attend(q: torch.Tensor, kv: PagedQuantKV, cu_seqlens: torch.Tensor, lengths: torch.Tensor, scale: float, *,
                   positions: torch.Tensor | None = None, tokens: int | None = None, softcap: float = 0.0, window: int = 0,
                   alibi_slopes: torch.Tensor | None = None, key_starts: torch.Tensor | None = None,
                   prefix_lens: torch.Tensor | None = None, out: torch.Tensor | None = None,
                   workspace: torch.Tensor | None = None, pdl: bool = False) -> torch.Tensor:
    """Causal attention of new tokens q [T, Hq, D] over the pages of their B sequences: [T, Hq, D] in q's dtype.

    Sequence b's new tokens are rows cu_seqlens[b] .. cu_seqlens[b + 1] - 1 of q (int32 [B + 1]); their keys and values are in
    `kv` already, and lengths[b] counts them. They are the last ones of their sequence unless `positions` [T] says where each
    sits. A token at p sees the keys max(0, key_starts[row], p - window + 1) <= j < min(length, max(p + 1, prefix_lens[b])):

    - `window` w > 0: the last w keys only; `key_starts` [T]: the first key of the token's document, where several share a
      sequence; `prefix_lens` [B]: a prefix that every token sees whole;
    - `softcap` c > 0: scores become c * tanh(score / c); `alibi_slopes` [Hq]: they fall by slope * |p - j|.

    A token that sees no key gets zeros; rows of q that belong to no sequence leave `out` as it is. q is f16 or bf16, of the
    pages' own dtype where they are 16-bit. Tokens are taken in tiles of neighbours in their sequence (128 rows, 64 over INT8
    pages; a token has a row per query head of a KV head). A value that is NaN or infinite reaches every token of a tile if its
    key lies between the first and the last that the tile's tokens see, whether or not one of them sees it; before the first
    and behind the last it reaches none. Table entries between those two have to name blocks of the pool. `tokens` bounds the longest length (no host sync on lengths.max()).
    `workspace`: `bpt_paged_prefill_workspace_bytes` bytes of any content (a workspace of `attend`'s that is large enough serves
    too: its first 256 KiB, where `attend` keeps counters, are left alone).
    """
    device = require_cuda(q, kv.k_pool, kv.v_pool, kv.block_table, cu_seqlens, lengths, positions, alibi_slopes, key_starts,
                          prefix_lens, out, workspace)
    code, ks, vs, kss, vss, nb, bs, hkv, d = pool_format(kv)
    shape = q.shape
    if len(shape) != 3 or shape[2] != d or shape[1] % hkv:
        raise ValueError(f"pool shape {tuple(kv.k_pool.shape)} does not match q {tuple(shape)}")
    if q.dtype not in (torch.float16, torch.bfloat16):
        raise ValueError(f"q must be float16 or bfloat16, got {q.dtype}")
    t, hq, _ = shape
    table, b, table_stride, table_width = block_table_of(kv)
    if cu_seqlens.shape != (b + 1,) or lengths.shape != (b,):
        raise ValueError(f"cu_seqlens must be [{b + 1}] and lengths [{b}], got {tuple(cu_seqlens.shape)} and "
                         f"{tuple(lengths.shape)}")
    if window < 0 or softcap < 0:
        raise ValueError(f"window and softcap must not be negative, got {window} and {softcap}")
    if out is not None and (out.shape != shape or out.dtype != q.dtype or not out.is_contiguous()):
        raise ValueError(f"out must be a contiguous [{t}, {hq}, {d}] tensor of {q.dtype}")
    tokens = max(table_width * bs if tokens is None else int(tokens), 1)
    with on_device(device):
        stride = q.stride()
        if stride[2] != 1 or stride[0] % 8 or stride[1] % 8 or q.data_ptr() % 16:
            q = q.clone(memory_format=torch.contiguous_format)
            stride = q.stride()
        cu, lengths = as_int32(cu_seqlens), as_int32(lengths)
        positions = _row_tensor("positions", positions, (t,), torch.int32)
        starts = _row_tensor("key_starts", key_starts, (t,), torch.int32)
        prefix = _row_tensor("prefix_lens", prefix_lens, (b,), torch.int32)
        slopes = _row_tensor("alibi_slopes", alibi_slopes, (hq,), torch.float32)
        if out is None:
            out = torch.empty(shape, dtype=q.dtype, device=device)
        if workspace is None:
            need = int(lib().bpt_paged_prefill_workspace_bytes(t, b, hq, hkv, d, code, tokens))
            workspace = _scratch(need, device) if need else None
        st = _lib.paged_prefill(
            q.data_ptr(), dtype_code(q.dtype), stride[0], stride[1], kv.k_pool.data_ptr(), kv.v_pool.data_ptr(), code, ks, vs,
            addr(kss), addr(vss), table.data_ptr(), table_stride, table_width, cu.data_ptr(), lengths.data_ptr(),
            addr(positions), addr(starts), addr(prefix), addr(slopes), float(softcap), int(window), t, b, hq, hkv, d, bs, nb, tokens, float(scale),
            out.data_ptr(), addr(workspace), 0 if workspace is None else workspace.numel() * workspace.element_size(),
            FLAG_PDL if pdl else 0, stream_of(device))
    check(st, "prefill_attend")
    return out
