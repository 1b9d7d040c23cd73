"""The paged-cache operators as they are measured: the rotated append, the decode read and the prefill read.

Three operators share one paged key-value cache, pools [num_blocks, block_size, Hkv, D] of bf16, f16, E4M3 bytes (one
scale per tensor) or int8 codes (one f16 scale per token and KV head):

- "append": optional RMSNorm of q and k per head, rotation of q and k, keys and values stored at their slots;
- "decode": one query token per sequence over its pages;
- "prefill": the new tokens of a ragged batch over their sequences' pages.

A query at position p of a sequence of L tokens sees the keys j with lo <= j < hi,
    lo = max(0, key_start, p - window + 1 if window), hi = min(L, max(p + 1, prefix)),
under the scores cap * tanh(scale * q.k / cap) (cap 0: scale * q.k) - slope[head] * |p - j|; no visible key gives 0.

`run` computes them in plain torch where `own` is false, by the framework's calls where it is true.
"""

from __future__ import annotations

import functools
import math
import os
import random
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SCALE_E4M3 = 1.0 / 64.0  # per-tensor scale of the E4M3 pools: N(0, 1) data uses 7 of its 448 / 64 range


# ---- the cases -----------------------------------------------------------------------------------------------------


def _append(name, **kw):
    base = {"name": name, "op": "append", "kind": "bf16", "dtype": "bf16", "hq": 16, "hkv": 8, "d": 128, "rotary": 128,
            "interleaved": False, "norm": True, "tokens": 64, "bs": 16, "reach": 4096}
    return base | kw


def _attend(name, op, **kw):
    base = {"name": name, "op": op, "kind": "bf16", "dtype": "bf16", "hq": 16, "hkv": 8, "d": 128, "bs": 16, "seqs": 1,
            "ctx_lo": 0, "ctx_hi": 0, "new_lo": 1, "new_hi": 1, "spread": 1, "softcap": 0.0, "window": 0,
            "alibi": False, "prefix": 0, "documents": 0}
    return base | kw


def listed():
    return [
        # one decode step of 64 sequences of the Qwen3-1.7B layer (QK-norm, 16 / 8 heads): the latency of a call
        _append("append decode 64"),
        # the prompts of a prefill batch, packed: bandwidth
        _append("append prompt 8192", tokens=8192),
        # an E4M3 cache under a model that rotates half of each head, in pairs (2i, 2i + 1), without QK-norm
        _append("append fp8 2001", kind="fp8", dtype="f16", hq=24, hkv=4, d=64, rotary=32, interleaved=True, norm=False,
                tokens=2001, reach=32768),
        # one chat session: the latency of a decode read
        _attend("decode one 1000", "decode", ctx_lo=999, ctx_hi=999),
        # the batch of the framework's decode benchmark (32 sequences of 512 to 4,096 tokens), over a bf16 cache
        _attend("decode batch 32", "decode", seqs=32, ctx_lo=511, ctx_hi=4095),
        # long documents under a tanh cap, four query heads per KV head
        _attend("decode long 8x32768", "decode", kind="f16", dtype="f16", hq=32, seqs=8, ctx_lo=32767, ctx_hi=32767,
                softcap=30.0),
        # a sliding window and a distance bias over an E4M3 cache, seven query heads per KV head
        _attend("decode fp8 window 17", "decode", kind="fp8", hq=28, hkv=4, seqs=17, ctx_lo=100, ctx_hi=16000,
                window=4096, alibi=True),
        # a short turn on top of a long session: few rows, a long cache
        _attend("prefill chunk 33 over 8192", "prefill", ctx_lo=8192, ctx_hi=8192, new_lo=33, new_hi=33),
        # prompts of a serving batch, ragged
        _attend("prefill ragged 12", "prefill", seqs=12, new_lo=17, new_hi=2000),
        # one long prompt, four query heads per KV head
        _attend("prefill long 8192", "prefill", hq=32, new_lo=8192, new_hi=8192),
        # heads of 256 with a sliding window and a tanh cap, f16
        _attend("prefill d256 capped", "prefill", kind="f16", dtype="f16", d=256, hq=16, hkv=8, new_lo=4096,
                new_hi=4096, window=1024, softcap=50.0),
        # a chunk of a long prompt over an E4M3 cache: packed documents, a shared prefix, a distance bias
        _attend("prefill fp8 documents", "prefill", kind="fp8", d=64, hq=16, hkv=4, seqs=2, ctx_lo=3001, ctx_hi=6000,
                new_lo=1500, new_hi=2047, alibi=True, prefix=500, documents=3),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "decode", "prefill"])
    kind = rng.choice(["bf16", "bf16", "f16", "fp8"])
    dtype = kind if kind in ("bf16", "f16") else rng.choice(["bf16", "f16"])
    hkv = rng.choice([1, 2, 4, 8])
    rep = rng.choice([1, 2, 3, 4, 5, 7, 8])
    d = rng.choice([64, 128, 128, 256])
    bs = rng.choice([8, 16, 16, 32, 64])
    if op == "append":
        case = _append("", kind=kind, dtype=dtype, hkv=hkv, hq=hkv * rep, d=d, bs=bs, tokens=_log(rng, 1, 8192),
                       rotary=rng.choice([d, d, d // 2]), interleaved=rng.random() < 0.3, norm=rng.random() < 0.5,
                       reach=_log(rng, 512, 131072))
    else:
        if op == "decode":
            kind = rng.choice([kind, kind, "int8"])
            seqs, hi = _log(rng, 1, 64), _log(rng, 16, 32768)
            while seqs * hi > 262144:
                seqs, hi = max(1, seqs // 2), hi - hi // 3
            kw = {"ctx_lo": rng.choice([-1, 0, hi // 7, hi // 2]), "ctx_hi": hi - 1}
        else:
            seqs, new, ctx = _log(rng, 1, 16), _log(rng, 2, 4096), rng.choice([0, 0, _log(rng, 1, 16384)])
            while seqs * hkv * rep * new * (new + ctx) > 1 << 31 or seqs * (new + ctx) > 131072:
                seqs, new, ctx = max(1, seqs // 2), new - new // 3, ctx - ctx // 3
            kw = {"ctx_lo": ctx // 3, "ctx_hi": ctx, "new_lo": rng.choice([0, 1, new // 4, new]), "new_hi": new,
                  "prefix": rng.choice([0, 0, max(1, (new + ctx) // 5)])}
        case = _attend("", op, kind=kind, dtype=dtype, hkv=hkv, hq=hkv * rep, d=d, bs=bs, seqs=seqs,
                       spread=rng.randrange(1 << 20), softcap=rng.choice([0.0, 0.0, 20.0, 50.0]),
                       window=rng.choice([0, 0, _log(rng, 1, 4096)]), alibi=rng.random() < 0.3,
                       documents=rng.choice([0, 0, 2, 5]), **kw)
        if kind in ("fp8", "int8") and op == "decode" and not (case["softcap"] or case["window"] or case["alibi"]):
            case["softcap"] = 30.0  # without an option these read by the quantized decode kernel that is there
    del case["name"]
    return case


def _lengths(case):
    """(cached tokens before, new tokens) of every sequence."""
    rng = random.Random(case["spread"])
    got = [(rng.randint(case["ctx_lo"], case["ctx_hi"]), rng.randint(case["new_lo"], case["new_hi"]))
           for _ in range(case["seqs"])]
    if not any(n for _, n in got):
        got[0] = (got[0][0], max(1, case["new_hi"]))
    return got


def _starts(case):
    """The first key that each new token's document lets it see, or None."""
    if not case["documents"]:
        return None
    rng, starts = random.Random(case["spread"] + 7), []
    for ctx, new in _lengths(case):
        cuts = sorted([0] + [rng.randint(0, max(0, ctx + new - 1)) for _ in range(case["documents"] - 1)])
        k = 0
        for p in range(ctx, ctx + new):
            while k + 1 < len(cuts) and cuts[k + 1] <= p:
                k += 1
            starts.append(cuts[k])
    return starts


def _interval(case, ctx, t, new, start):
    """(lo, hi) of the keys that new token t of a sequence sees."""
    p, length = ctx + t, ctx + new
    lo = max(0, start, p - case["window"] + 1 if case["window"] else 0)
    return lo, min(length, max(p + 1, case["prefix"] if case["op"] == "prefill" else 0))


_SIZE = {"bf16": 2, "f16": 2, "f32": 4, "fp8": 1, "int8": 1}


@functools.lru_cache(maxsize=64)
def _work(items):
    case = dict(items)
    d, hq, hkv, el = case["d"], case["hq"], case["hkv"], _SIZE[case["dtype"]]
    if case["op"] == "append":
        t = case["tokens"]
        read = t * (hq + 2 * hkv) * d * el + t * case["rotary"] * 4 + 12 * t + (2 * d * el if case["norm"] else 0)
        wrote = t * hq * d * el + 2 * t * hkv * d * _SIZE[case["kind"]]
        return {"bytes": read + wrote, "flops": t * (hq + hkv) * (3 * case["rotary"] + (4 * d if case["norm"] else 0))}
    starts, at, pairs, keys, rows = _starts(case), 0, 0, 0, 0
    for ctx, new in _lengths(case):
        low, high = None, 0
        for t in range(new):
            lo, hi = _interval(case, ctx, t, new, starts[at] if starts else 0)
            at += 1
            if hi > lo:
                pairs += hi - lo
                low, high = lo if low is None else min(low, lo), max(high, hi)
        keys += high - low if low is not None else 0
        rows += new
    per_key = 2 * hkv * (d * _SIZE[case["kind"]] + (2 if case["kind"] == "int8" else 0))
    return {"bytes": keys * per_key + 4 * keys // case["bs"] + 2 * rows * hq * d * el, "flops": 4 * pairs * hq * d}


def work(case):
    return _work(tuple(sorted((k, v) for k, v in case.items() if k != "name")))


# ---- the inputs ----------------------------------------------------------------------------------------------------


def _store(x, kind):
    """x [..., Hkv, D] float32 as a pool of `kind` and its scales."""
    if kind in ("bf16", "f16"):
        return x.to(DTYPES[kind]), 1.0
    if kind == "fp8":
        return (x / SCALE_E4M3).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8), SCALE_E4M3
    scale = (x.abs().amax(-1) / 127).to(torch.float16)
    return (x / scale.float()[..., None]).round().clamp(-128, 127).to(torch.int8), scale


def prepare(case, seed):
    dev = "cuda"
    g = torch.Generator(device=dev).manual_seed(seed)
    d, hq, hkv, bs, dt = case["d"], case["hq"], case["hkv"], case["bs"], DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(shape, generator=g, device=dev)

    if case["op"] == "append":
        t, r = case["tokens"], case["rotary"]
        pages = 2 * (-(-t // bs)) + 1
        # the fused projection's output (an outlier channel per head, as keys have) and its three parts
        qkv = randn(t, hq + 2 * hkv, d)
        qkv[:, : hq + hkv, d // 3] *= 8
        qkv = qkv.to(dt).view(t, -1)
        q, k, v = (x.view(t, -1, d) for x in qkv.split([hq * d, hkv * d, hkv * d], dim=1))
        angle = torch.arange(case["reach"], dtype=torch.float64, device=dev)[:, None] * (
            1e6 ** (-torch.arange(0, r, 2, dtype=torch.float64, device=dev) / r))
        slots = torch.randperm(pages * bs, generator=g, device=dev)[:t]  # distinct slots anywhere in the pool
        pools = [_store(randn(pages, bs, hkv, d), case["kind"]) for _ in range(2)]
        norms = [(1 + 0.1 * randn(d)).to(dt) if case["norm"] else None for _ in range(2)]
        return {"op": "append", "kind": case["kind"], "bs": bs, "q": q, "k": k, "v": v, "q_norm": norms[0],
                "k_norm": norms[1], "eps": 1e-6, "interleaved": case["interleaved"],
                "positions": torch.randint(0, case["reach"], (t,), generator=g, device=dev, dtype=torch.int32),
                "cos": angle.cos().float(), "sin": angle.sin().float(), "q_out": torch.empty(t, hq, d, dtype=dt, device=dev),
                "blocks": (slots // bs).int(), "offsets": (slots % bs).int(), "k_pool": pools[0][0],
                "v_pool": pools[1][0], "k_scale": pools[0][1], "v_scale": pools[1][1],
                "table": torch.zeros(1, 1, dtype=torch.int32, device=dev)}

    seqs = _lengths(case)
    need = [max(1, -(-(ctx + new) // bs)) for ctx, new in seqs]
    pages, width, cpu = sum(need) + 3, max(need), torch.Generator().manual_seed(seed)
    perm = torch.randperm(pages, generator=cpu).int()
    table, at = torch.zeros(len(seqs), width, dtype=torch.int32), 0
    for i, n in enumerate(need):
        table[i, :n] = perm[at : at + n]
        at += n
    k_pool, k_scale = _store(randn(pages, bs, hkv, d), case["kind"])
    v_pool, v_scale = _store(randn(pages, bs, hkv, d), case["kind"])
    new = [n for _, n in seqs]
    starts = _starts(case)
    q = (randn(sum(new), hq, d) * (4.0 if case["softcap"] else 1.0)).to(dt)
    slopes = 2.0 ** (-8.0 * torch.arange(1, hq + 1, device=dev) / hq)
    cu = torch.tensor([0] + new).cumsum(0).int()
    return {"op": case["op"], "kind": case["kind"], "bs": bs, "q": q, "scale": d ** -0.5, "table": table.to(dev),
            "k_pool": k_pool, "v_pool": v_pool, "k_scale": k_scale, "v_scale": v_scale,
            "lengths": torch.tensor([c + n for c, n in seqs], dtype=torch.int32, device=dev), "cu": cu.to(dev),
            "max_new": max(new), "longest": max(1, max(c + n for c, n in seqs)), "softcap": case["softcap"],
            "window": case["window"], "slopes": slopes if case["alibi"] else None,
            "starts": None if starts is None else torch.tensor(starts, dtype=torch.int32, device=dev),
            "prefix": torch.full((len(seqs),), case["prefix"], dtype=torch.int32, device=dev) if case["prefix"] else None,
            "out": torch.empty_like(q)}


# ---- the plain forms -----------------------------------------------------------------------------------------------


def _rotate(x, cos, sin, interleaved):
    """x [T, H, R] rotated by the angles of cos, sin [T, 1, R / 2]."""
    if interleaved:
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    a, b = x.chunk(2, dim=-1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)


def _plain_append(s):
    at = s["positions"].long()
    cos, sin = s["cos"][at][:, None], s["sin"][at][:, None]
    r = 2 * cos.shape[-1]

    def turned(x, w):
        x = x.float()
        if w is not None:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + s["eps"]) * w.float()
        return torch.cat([_rotate(x[..., :r], cos, sin, s["interleaved"]), x[..., r:]], dim=-1)

    def stored(x, scale, pool):
        if s["kind"] == "fp8":
            return (x / scale).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
        return x.to(pool.dtype)

    q, k = turned(s["q"], s["q_norm"]).to(s["q"].dtype), turned(s["k"], s["k_norm"])
    where = (s["blocks"].long(), s["offsets"].long())
    s["k_pool"][where] = stored(k, s["k_scale"], s["k_pool"])
    s["v_pool"][where] = stored(s["v"].float(), s["v_scale"], s["v_pool"])
    return q, _values(s["k_pool"], s["kind"]), _values(s["v_pool"], s["kind"])


def _values(pool, kind):
    return pool.view(torch.float8_e4m3fn) if kind == "fp8" else pool


def _read(pool, scale, kind, table):
    """The pages of `table` as float32 [B, Hkv, N, D]."""
    x = _values(pool, kind)[table.long()] if kind != "fp8" else pool[table.long()].view(torch.float8_e4m3fn)
    x = x.float()
    if kind == "fp8":
        x = x * scale
    elif kind == "int8":
        x = x * scale[table.long()].float()[..., None]
    return x.flatten(1, 2).transpose(1, 2)


def _plain_attention(s):
    q, cu, lengths, most = s["q"], s["cu"].long(), s["lengths"].long(), s["max_new"]
    t, hq, d = q.shape
    k = _read(s["k_pool"], s["k_scale"], s["kind"], s["table"])
    v = _read(s["v_pool"], s["v_scale"], s["kind"], s["table"])
    b, hkv, n, _ = k.shape
    rep = hq // hkv
    new = cu[1:] - cu[:-1]
    slot = torch.arange(most, device=q.device)
    rows = (cu[:-1, None] + slot).clamp(max=t - 1)  # [B, most]: a sequence's rows, padded
    pos = (lengths - new)[:, None] + slot
    lo = torch.zeros_like(pos) if s["starts"] is None else s["starts"].long()[rows]
    if s["window"]:
        lo = torch.maximum(lo, pos - s["window"] + 1)
    hi = pos + 1
    if s["prefix"] is not None:
        hi = torch.maximum(hi, s["prefix"].long()[:, None])
    hi = torch.minimum(hi, lengths[:, None])
    j = torch.arange(n, device=q.device)
    seen = ((j >= lo[..., None]) & (j < hi[..., None]))[:, None, None]  # [B, 1, 1, most, N]
    x = q.float()[rows].view(b, most, hkv, rep, d).permute(0, 2, 3, 1, 4).reshape(b, hkv, rep * most, d)
    w = (x @ k.transpose(2, 3)).mul_(s["scale"]).view(b, hkv, rep, most, n)
    if s["softcap"]:
        w = w.div_(s["softcap"]).tanh_().mul_(s["softcap"])
    if s["slopes"] is not None:
        far = (pos[..., None] - j).abs().float()[:, None, None]
        w.sub_(s["slopes"].view(1, hkv, rep, 1, 1) * far)
    w.masked_fill_(~seen, -math.inf)
    top = w.amax(-1, keepdim=True)
    w.sub_(top.masked_fill_(top == -math.inf, 0.0)).exp_()
    total = w.sum(-1, keepdim=True)
    o = (w.view(b, hkv, rep * most, n) @ v).view(b, hkv, rep, most, d) / total.masked_fill_(total == 0, 1.0)
    o = o.permute(0, 3, 1, 2, 4).reshape(b, most, hq, d)
    token = torch.arange(t, device=q.device)
    seq = torch.bucketize(token, cu[1:], right=True)
    return o[seq, token - cu[seq]].to(q.dtype)


# ---- the framework's calls -----------------------------------------------------------------------------------------


@functools.lru_cache(maxsize=1)
def _framework():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "bytes-per-token_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    from bpt_b200.kernels.kv_attention import PagedQuantKV, attend
    from bpt_b200.kernels.kv_write import rope_kv_append
    from bpt_b200.kernels.prefill_attention import prefill_attend

    return PagedQuantKV, attend, rope_kv_append, prefill_attend


def run(state):
    s = state
    if not own:
        return _plain_append(s) if s["op"] == "append" else _plain_attention(s)
    cache, attend, rope_kv_append, prefill_attend = _framework()
    kv = cache(s["kind"], s["k_pool"], s["v_pool"], s["table"], s["bs"], s["k_scale"], s["v_scale"])
    if s["op"] == "append":
        q = rope_kv_append(s["q"], s["k"], s["v"], kv, s["positions"], s["cos"], s["sin"], s["blocks"], s["offsets"],
                           q_norm=s["q_norm"], k_norm=s["k_norm"], eps=s["eps"], interleaved=s["interleaved"],
                           q_out=s["q_out"])
        return q, _values(s["k_pool"], s["kind"]), _values(s["v_pool"], s["kind"])
    more = {"tokens": s["longest"], "softcap": s["softcap"], "window": s["window"], "alibi_slopes": s["slopes"],
            "key_starts": s["starts"], "out": s["out"]}
    if s["op"] == "decode":
        return attend(s["q"], kv, s["lengths"], s["scale"], **more)
    return prefill_attend(s["q"], kv, s["cu"], s["lengths"], s["scale"], prefix_lens=s["prefix"], **more)


# ---- the definition in 64 bits -------------------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_append(s) if case["op"] == "append" else _exact_attention(case, s)


def _exact_append(s):
    r = 2 * s["cos"].shape[1]
    angle = torch.complex(s["cos"][s["positions"].long()].double(), s["sin"][s["positions"].long()].double())[:, None]

    def turned(x, w):
        x = x.double()
        if w is not None:
            x = x / (x.square().mean(-1, keepdim=True) + s["eps"]).sqrt() * w.double()
        head = x[..., :r]
        pair = head.unflatten(-1, (r // 2, 2)) if s["interleaved"] else head.unflatten(-1, (2, r // 2)).transpose(-1, -2)
        z = torch.complex(pair[..., 0], pair[..., 1]) * angle
        pair = torch.stack([z.real, z.imag], dim=-1 if s["interleaved"] else -2)
        return torch.cat([pair.flatten(-2), x[..., r:]], dim=-1)

    def filled(pool, x, scale):
        y = _values(pool, s["kind"]).double()
        y[s["blocks"].long(), s["offsets"].long()] = (x / scale).clamp(-448, 448) if s["kind"] == "fp8" else x
        return y

    return (turned(s["q"], s["q_norm"]), filled(s["k_pool"], turned(s["k"], s["k_norm"]), s["k_scale"]),
            filled(s["v_pool"], s["v"].double(), s["v_scale"]))


def _exact_attention(case, s):
    t, hq, d = s["q"].shape
    hkv = case["hkv"]
    rep, dev, bs = hq // hkv, s["q"].device, case["bs"]
    out = torch.zeros(t, hq, d, dtype=torch.float64, device=dev)
    starts, at = _starts(case), 0
    for i, (ctx, new) in enumerate(_lengths(case)):
        length = ctx + new
        if length > 0 and new > 0:
            pages = s["table"][i, : -(-length // bs)].long()
            bounds = torch.tensor([_interval(case, ctx, u, new, starts[at + u] if starts else 0) for u in range(new)],
                                  device=dev)
            j, p = torch.arange(length, device=dev), torch.arange(ctx, length, device=dev)
            seen = (j >= bounds[:, :1]) & (j < bounds[:, 1:])
            gap = (p[:, None] - j).abs().double()
            for h in range(hkv):
                kv = []
                for pool, scale in ((s["k_pool"], s["k_scale"]), (s["v_pool"], s["v_scale"])):
                    x = pool[pages, :, h]
                    x = (x.view(torch.float8_e4m3fn) if case["kind"] == "fp8" else x).double()
                    if case["kind"] == "int8":
                        x = x * scale[pages, :, h].double()[..., None]
                    elif case["kind"] == "fp8":
                        x = x * scale
                    kv.append(x.reshape(-1, d)[:length])
                for g in range(h * rep, (h + 1) * rep):
                    a = s["q"][at : at + new, g].double() @ kv[0].T * s["scale"]
                    if case["softcap"]:
                        a = case["softcap"] * torch.tanh(a / case["softcap"])
                    if s["slopes"] is not None:
                        a = a - s["slopes"][g].double() * gap
                    a = torch.softmax(a.masked_fill(~seen, -math.inf), dim=-1).nan_to_num(0.0)
                    out[at : at + new, g] = a @ kv[1]
        at += new
    return out
