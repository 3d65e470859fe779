"""Cases for the operators that keep and read a long context in less memory: attention with score forms (tanh cap,
distance bias, per-row key intervals), the 8-bit cache with one scale per block of rows and head, and eviction from it
by accumulated attention weight.

`run` computes them in plain torch operations, or, where `own` is set, calls the framework."""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEV = "cuda"


# ---------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # a short prompt with an image or instruction prefix that every token sees, capped scores: the first request of a server
        dict(name="prefill_prefix_small", op="prefill", B=1, H=8, Hkv=8, S=130, d=64, io="float32", cache="float32", softcap=30.0, alibi=False, mask="prefix"),
        # documents packed into rows of a batch of prompts (the benchmark's prefill shape), capped scores
        dict(name="prefill_documents", op="prefill", B=8, H=32, Hkv=32, S=1024, d=128, io="float16", cache="float16", softcap=50.0, alibi=False, mask="documents"),
        # one long prompt with distance bias and shared K/V heads, ragged length
        dict(name="prefill_alibi_long", op="prefill", B=1, H=32, Hkv=8, S=4001, d=128, io="float16", cache="float16", softcap=0.0, alibi=True, mask="causal"),
        # one short sequence: latency of a decode step with capped scores
        dict(name="decode_capped_short", op="decode", B=1, H=8, Hkv=8, T=97, most=90, least=90, d=128, io="float32", cache="float32", softcap=30.0, alibi=False, window=0),
        # a serving batch at the benchmark's decode shape, distance bias
        dict(name="decode_alibi_batch", op="decode", B=16, H=32, Hkv=32, T=2048, most=2047, least=1024, d=128, io="float16", cache="float16", softcap=0.0, alibi=True, window=0),
        # the prompts of a batch into the 8-bit cache
        dict(name="append_prompt", op="append", B=8, Hkv=32, S=1024, T=1088, d=128, block=64, code="int8", io="float16", most=0, least=0, ragged=True),
        # a chunk of a few tokens (drafted, or a tool's answer) into partly filled blocks, straight from the int32 projections
        dict(name="append_chunk", op="append", B=5, Hkv=8, S=7, T=512, d=128, block=32, code="e4m3", io="int32", most=480, least=3, ragged=False),
        # one short sequence over the 8-bit cache: latency
        dict(name="cache8_decode_one", op="decode8", B=1, H=8, Hkv=8, T=128, most=99, least=99, d=64, block=16, code="e4m3", io="float16", out="float16", softcap=0.0, alibi=False, weights=False, window=0),
        # the serving batch of the decode benchmark over the 8-bit cache
        dict(name="cache8_decode_batch", op="decode8", B=16, H=32, Hkv=32, T=2048, most=2047, least=1024, d=128, block=64, code="int8", io="float16", out="float32", softcap=0.0, alibi=False, weights=False, window=0),
        # one very long sequence with shared K/V heads, capped scores, weights accumulated for a later eviction
        dict(name="cache8_decode_long", op="decode8", B=1, H=32, Hkv=8, T=131072, most=100001, least=100001, d=128, block=64, code="int8", io="float16", out="float16", softcap=50.0, alibi=False, weights=True, window=0),
        # a serving batch that has grown past its budget
        dict(name="evict_batch", op="evict", B=16, Hkv=8, T=4352, most=4350, least=2000, budget=4096, recent=256, sinks=4, d=128, block=64, code="int8"),
        # a long sequence cut down to a quarter
        dict(name="evict_long", op="evict", B=1, Hkv=8, T=65536, most=65536, least=65536, budget=16384, recent=512, sinks=4, d=128, block=64, code="int8"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _heads(rng, most):
    g = rng.choice([1, 1, 2, 4, 5, 8])
    kv = _log_int(rng, 1, max(1, most // g))
    return kv * g, kv


def draw(rng):
    op = rng.choice(["prefill", "prefill", "decode", "append", "decode8", "decode8", "evict"])
    if op == "prefill":
        B, S, d = _log_int(rng, 1, 8), _log_int(rng, 2, 2100), rng.choice([64, 128, 128])
        H, Hkv = _heads(rng, 32)
        while B * H * S * S > 8 * 32 * 1024 * 1024:
            S = max(2, S // 2 + 1)
        io = rng.choice(["float16", "float16", "float32", "int32"])
        return dict(op=op, B=B, H=H, Hkv=Hkv, S=S, d=d, io=io, cache=rng.choice(["float16", "float32"]), softcap=rng.choice([0.0, 20.0, 30.0, 50.0]),
                    alibi=rng.random() < 0.4, mask=rng.choice(["causal", "prefix", "documents", "padded"]))
    if op == "decode":
        B, T, d = _log_int(rng, 1, 16), _log_int(rng, 2, 4096), rng.choice([64, 128, 256])
        H, Hkv = _heads(rng, 32)
        while B * H * T * d > 16 * 32 * 2048 * 128:
            T = max(2, T // 2)
        return dict(op=op, B=B, H=H, Hkv=Hkv, T=T, most=T - 1, least=rng.randrange(0, T), d=d, io=rng.choice(["float16", "float32", "int32"]),
                    cache=rng.choice(["float16", "float32"]), softcap=rng.choice([0.0, 20.0, 50.0]), alibi=rng.random() < 0.5, window=rng.choice([0, 0, 100]))
    if op == "append":
        B, Hkv, d, block = _log_int(rng, 1, 16), _log_int(rng, 1, 32), rng.choice([64, 128, 256]), rng.choice([16, 32, 64, 128])
        S = _log_int(rng, 1, 1500)
        while B * Hkv * S * d > 8 * 32 * 1024 * 128:
            S = max(1, S // 2)
        least = rng.choice([0, 0, rng.randrange(1, 300)])
        most = least + rng.randrange(0, 2 * block)
        T = -(-(most + S) // block) * block + block * rng.randrange(0, 3)
        return dict(op=op, B=B, Hkv=Hkv, S=S, T=T, d=d, block=block, code=rng.choice(["int8", "e4m3"]), io=rng.choice(["float16", "float32", "int32"]),
                    most=most, least=least, ragged=rng.random() < 0.5)
    if op == "decode8":
        B, d, block = _log_int(rng, 1, 16), rng.choice([64, 128, 128, 256]), rng.choice([16, 32, 64, 128])
        H, Hkv = _heads(rng, 32)
        T = _log_int(rng, 1, 65536 // block) * block
        while B * Hkv * T * d > 16 * 32 * 2048 * 128 or B * H * T > 32 * 131072:
            T = max(block, T // (2 * block) * block)
        return dict(op=op, B=B, H=H, Hkv=Hkv, T=T, most=T - 1, least=rng.randrange(0, T), d=d, block=block, code=rng.choice(["int8", "e4m3"]),
                    io=rng.choice(["float16", "float32", "int32"]), out=rng.choice(["float16", "float32"]), softcap=rng.choice([0.0, 0.0, 30.0]),
                    alibi=rng.random() < 0.3, weights=rng.random() < 0.5, window=rng.choice([0, 0, 1000]))
    B, Hkv, d, block = _log_int(rng, 1, 16), _log_int(rng, 1, 16), rng.choice([64, 128, 256]), rng.choice([16, 32, 64, 128])
    T = _log_int(rng, 2, 65536 // block) * block
    while B * Hkv * T * d > 8 * 65536 * 128:
        T = max(block, T // (2 * block) * block)
    budget = rng.randrange(1, T + 1)
    recent = rng.randrange(0, budget + 1)
    return dict(op=op, B=B, Hkv=Hkv, T=T, most=T, least=rng.randrange(0, T + 1), budget=budget, recent=recent, sinks=min(rng.choice([0, 1, 4]), budget - recent),
                d=d, block=block, code=rng.choice(["int8", "e4m3"]))


# ---------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    return g


def _table(rows, d):
    # [2i] = cos, [2i+1] = sin of position * 10000^(-2i/d); the table is an input, as in the decoder layer
    pos = torch.arange(rows, dtype=torch.float64, device=DEV)[:, None]
    theta = pos * torch.pow(torch.tensor(10000.0, dtype=torch.float64, device=DEV), -torch.arange(0, d, 2, dtype=torch.float64, device=DEV) / d)
    return torch.stack([theta.cos(), theta.sin()], dim=-1).reshape(rows, d).float().contiguous()


def _tokens(g, io, B, S, heads, d, std=1.0):
    """Fresh rows of a projection [B,S,heads,d] with what turns them into values: int32 sums with two scales, or values."""
    x = torch.randn(B, S, heads, d, generator=g, device=DEV) * std
    if io == "int32":
        w = torch.rand(heads * d, generator=g, device=DEV) + 0.5
        return torch.round(x * 4096.0).to(torch.int32), (w / 64.0).contiguous()
    return x.to(getattr(torch, io)), None


def _act(g, io, n):
    return (torch.rand(n, generator=g, device=DEV) + 0.5) / 64.0 if io == "int32" else None


def _lens(g, B, least, most):
    n = torch.randint(least, most + 1, (B,), generator=g, device=DEV, dtype=torch.int32)
    n[-1:] = most
    return n


def _slopes(H):
    return torch.pow(torch.tensor(2.0, device=DEV), -8.0 * torch.arange(1, H + 1, device=DEV) / H).float()


def _codes(g, code, shape):
    x = torch.empty(shape, dtype=torch.int8 if code == "int8" else torch.float8_e4m3fn, device=DEV)
    for b in range(shape[0]):  # a sequence at a time: the fp32 draws of a long cache take four times its room
        r = torch.randn(shape[1:], generator=g, device=DEV)
        x[b] = (r * 32.0).round().clamp_(-127, 127).to(torch.int8) if code == "int8" else (r * 112.0).clamp_(-448, 448).to(torch.float8_e4m3fn)
    return x


def _cache8(g, c):
    """A cache in use: codes, one scale per block and head of values of about unit size, positions in row order."""
    B, Hkv, T, d = c["B"], c["Hkv"], c["T"], c["d"]
    top = 127.0 / 4 if c["code"] == "int8" else 448.0 / 4
    s = dict(k_codes=_codes(g, c["code"], (B, Hkv, T, d)), v_codes=_codes(g, c["code"], (B, Hkv, T, d)))
    for n in ("k_scale", "v_scale"):
        s[n] = torch.exp(torch.randn(B, Hkv, T // c["block"], generator=g, device=DEV) * 0.2) / top
    s["row_pos"] = torch.arange(T, dtype=torch.int32, device=DEV).expand(B, Hkv, T).contiguous()
    return s


def prepare(case, seed):
    c, g = dict(case), _gen(seed)
    s = dict(case=c)
    op, B, d = c["op"], c["B"], c["d"]
    if op in ("prefill", "decode"):
        H, Hkv = c["H"], c["Hkv"]
        S = c["S"] if op == "prefill" else 1
        T = S + 5 if op == "prefill" else c["T"]
        # projections of trained models give scores of several units: that is where a cap acts
        s["q"], s["qw"] = _tokens(g, c["io"], B, S, H, d, 2.0)
        s["k"], s["kw"] = _tokens(g, c["io"], B, S, Hkv, d)
        s["v"], s["vw"] = _tokens(g, c["io"], B, S, Hkv, d)
        s["act"] = _act(g, c["io"], B * S)
        dt = getattr(torch, c["cache"])
        s["k_cache"] = torch.randn(B, Hkv, T, d, generator=g, device=DEV).to(dt)
        s["v_cache"] = torch.randn(B, Hkv, T, d, generator=g, device=DEV).to(dt)
        s["slopes"] = _slopes(H) if c["alibi"] else None
        s["table"] = _table(T, d)
        if op == "prefill":
            s["out"] = torch.empty(B, H, S, d, dtype=torch.float16, device=DEV)
            s["begin"] = s["end"] = None
            row = torch.arange(S, dtype=torch.int32, device=DEV)
            if c["mask"] == "prefix":  # every token sees the prefix, the others as usual
                n = _lens(g, B, 1, max(1, S // 3))
                s["end"] = torch.maximum(row[None] + 1, n[:, None]).contiguous()
            elif c["mask"] == "documents":  # a token sees its own document only
                cut = torch.rand(B, S, generator=g, device=DEV) < 4.0 / S
                s["begin"] = torch.cummax(torch.where(cut, row, torch.zeros_like(row)), dim=1).values.to(torch.int32).contiguous()
            elif c["mask"] == "padded":  # prompts padded on the right: rows behind a prompt see nothing
                n = _lens(g, B, 1, S)
                s["end"] = torch.where(row[None] < n[:, None], row[None] + 1, torch.zeros_like(row)).contiguous()
        else:
            s["past"] = _lens(g, B, min(c["least"], c["most"]), c["most"])
            s["out"] = torch.empty(B, H, 1, d, dtype=torch.float32, device=DEV)
            s["begin"] = (s["past"] - c["window"] + 1).clamp_min(0).to(torch.int32) if c["window"] else None
        n = _scratch_bytes(c, T)
        s["scratch"] = torch.zeros(n, dtype=torch.uint8, device=DEV)
        return s
    if op == "append":
        s.update(_cache8(g, c))
        s["k"], s["kw"] = _tokens(g, c["io"], B, c["S"], c["Hkv"], d)
        s["v"], s["vw"] = _tokens(g, c["io"], B, c["S"], c["Hkv"], d)
        s["act"] = _act(g, c["io"], B * c["S"])
        s["past"] = _lens(g, B, c["least"], c["most"])
        s["new"] = _lens(g, B, 0, c["S"]) if c["ragged"] else None
        s["table"] = _table(c["T"], d)
        s["scratch"] = torch.zeros(4096, dtype=torch.uint8, device=DEV)
        return s
    if op == "decode8":
        s.update(_cache8(g, c))
        H, Hkv = c["H"], c["Hkv"]
        s["q"], s["qw"] = _tokens(g, c["io"], B, 1, H, d, 2.0)
        s["k"], s["kw"] = _tokens(g, c["io"], B, 1, Hkv, d)
        s["v"], s["vw"] = _tokens(g, c["io"], B, 1, Hkv, d)
        s["act"] = _act(g, c["io"], B)
        s["past"] = _lens(g, B, min(c["least"], c["most"]), c["most"])
        s["out"] = torch.empty(B, H, 1, d, dtype=getattr(torch, c["out"]), device=DEV)
        s["slopes"] = _slopes(H) if c["alibi"] else None
        s["begin"] = (s["past"] - c["window"] + 1).clamp_min(0).to(torch.int32) if c["window"] else None
        s["table"] = _table(c["T"], d)
        if c["weights"]:
            s["w_in"] = torch.rand(B, Hkv, c["T"], generator=g, device=DEV)
            s["w_out"] = torch.zeros(B, Hkv, c["T"], device=DEV)
        s["scratch"] = torch.zeros(_scratch_bytes(c, c["T"]), dtype=torch.uint8, device=DEV)
        return s
    s.update(_cache8(g, c))
    T = c["T"]
    s["past"] = _lens(g, B, min(c["least"], c["most"]), c["most"])
    # a few rows draw most of the attention, the newest have had none yet: equal weights
    w = torch.exp(torch.randn(B, c["Hkv"], T, generator=g, device=DEV) * 2.0)
    s["w_in"] = torch.where(torch.rand(B, c["Hkv"], T, generator=g, device=DEV) < 0.1, torch.zeros_like(w), w)
    # positions: what earlier evictions left (gaps, and rows that were moved into holes)
    p = torch.arange(T, device=DEV, dtype=torch.int32) * 2
    swap = torch.randint(0, T, (2, max(1, T // 50)), generator=g, device=DEV)
    perm = torch.arange(T, device=DEV)
    a, b = swap[0].unique(), swap[1].unique()
    m = min(len(a), len(b))
    both = torch.isin(b[:m], a[:m])
    a, b = a[:m][~both], b[:m][~both]
    keep_a = ~torch.isin(a, b)
    a, b = a[keep_a], b[keep_a]
    perm[a], perm[b] = perm[b].clone(), perm[a].clone()
    s["row_pos"] = p[perm].expand(B, c["Hkv"], T).contiguous()
    s["next"] = (2 * s["past"]).to(torch.int32)
    s["w_out"] = torch.zeros_like(s["w_in"])
    s["pos_out"] = torch.zeros_like(s["row_pos"])
    s["len_out"] = torch.zeros_like(s["past"])
    s["scratch"] = torch.zeros(B * c["Hkv"] * (8 * T + 64) + 4096, dtype=torch.uint8, device=DEV)
    return s


def _scratch_bytes(c, T):
    """Room that every call of these sizes fits into, with some to spare."""
    B, H, d = c["B"], c["H"], c["d"]
    if c["op"] == "prefill":
        return 3 * (B * H * c["S"] * d * 2 + 256) + B * (c["S"] // 64 + 2) * 16 + 65536
    return B * H * (T // 32 + 2) * (d + 2) * 4 + B * H * T * 4 + B * H * 64 + 65536


# ---------------------------------------------------------------------------------------------------------------
# plain form
# ---------------------------------------------------------------------------------------------------------------
def _values(x, act, w):
    """[B,S,heads,d] in 32 bits."""
    if x.dtype != torch.int32:
        return x.float()
    B, S, h, d = x.shape
    return x.float() * act.view(B, S, 1, 1) * w.view(1, 1, h, d)


def _rotate(x, table, pos):
    """Pairs (2i, 2i+1) of [B,S,heads,d] by the table's rows at pos [B,S]."""
    f = table[pos.long()]
    co, sn = f[..., 0::2].unsqueeze(2), f[..., 1::2].unsqueeze(2)
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack([a * co - b * sn, b * co + a * sn], dim=-1).reshape(x.shape)


def _cap(x, cap):
    return cap * torch.tanh(x / cap) if cap else x


def _attend(q, k, v, visible, distance, slopes, cap):
    """q [B,H,S,d] against k, v [B,Hkv,K,d] in 32 bits; visible [B,S,K] and distance [B,1|Hkv,S,K] or None. Rows without a visible key give 0."""
    B, H, S, d = q.shape
    G = H // k.shape[1]
    x = torch.matmul(q.view(B, -1, G * S, d), k.transpose(-1, -2)).view(B, H, S, -1) * (1.0 / math.sqrt(d))
    x = _cap(x, cap)
    if slopes is not None:
        x = x - slopes.view(1, H, 1, 1) * distance.float().repeat_interleave(H // distance.shape[1], dim=1)
    x = torch.where(visible, x, torch.full_like(x, -torch.inf))
    m = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(torch.isfinite(m), m, torch.zeros_like(m)))
    p = torch.where(visible, p, torch.zeros_like(p))
    n = p.sum(-1, keepdim=True)
    p = torch.where(n > 0, p / n, torch.zeros_like(p))
    return torch.matmul(p.view(B, -1, G * S, p.shape[-1]), v).view(B, H, S, d), p


def _top(code):
    return 127.0 if code == "int8" else 448.0


def _encode(x, scale, code):
    """Codes of x at the scale of its block; a block of zeros has scale 0 and codes 0."""
    y = torch.where(scale > 0, x / scale, torch.zeros_like(x))
    return _round(y, code)


def _round(y, code):
    return y.round().clamp(-127, 127).to(torch.int8) if code == "int8" else y.clamp(-448, 448).to(torch.float8_e4m3fn)


def _merge(codes, scale, x, new, live, fresh, code):
    """Rows x where `new` into blocks: codes, x [B,h,n,block,d], scale, fresh [B,h,n], new, live [B,h,n,block]. The scale of a block
    grows to hold its new rows, and the codes of the live rows it held are brought to the new scale."""
    amax = torch.where(new[..., None], x, torch.zeros_like(x)).abs().amax((-1, -2))
    need = amax / torch.full_like(amax, _top(code))
    old = torch.where(fresh, torch.zeros_like(scale), scale)
    s = torch.maximum(old, need)
    touched = new.any(-1)
    grown = touched & (s > old) & ~fresh
    ratio = torch.where(grown, old / s, torch.ones_like(s))[..., None, None]
    held = torch.where(grown[..., None, None] & live[..., None], _round(codes.float() * ratio, code).float(), codes.float())
    put = torch.where(new[..., None], _encode(x, s[..., None, None], code).float(), held)
    return put.to(codes.dtype), torch.where(touched, s, scale)


def _append_one(codes, scale, x, past, count, block, code):
    """Rows x [B,h,S,d] behind the first `past` of a cache, in place. Only the blocks that the call can reach are looked at."""
    B, h, T, d = codes.shape
    S = x.shape[2]
    W = min(T, (-(-S // block) + 1) * block)
    first = torch.minimum(past.long() // block * block, torch.full_like(past.long(), T - W))
    rows = first[:, None] + torch.arange(W, device=codes.device)
    j = rows - past.long()[:, None]
    new = ((j >= 0) & (j < count.long()[:, None]))[:, None].expand(B, h, W)
    x = torch.gather(x, 2, j.clamp(0, S - 1)[:, None, :, None].expand(B, h, W, d))
    at = rows[:, None, :, None].expand(B, h, W, d)
    sat = (first[:, None] // block + torch.arange(W // block, device=codes.device))[:, None].expand(B, h, W // block)
    window = torch.gather(codes.view(torch.int8), 2, at).view(codes.dtype)
    shape = (B, h, W // block, block)
    fresh = sat * block >= past.long()[:, None, None]
    c, s = _merge(window.view(*shape, d), torch.gather(scale, 2, sat), x.view(*shape, d), new.reshape(shape),
                  (j < 0)[:, None].expand(B, h, W).reshape(shape), fresh, code)
    codes.view(torch.int8).scatter_(2, at, c.view(B, h, W, d).view(torch.int8))
    scale.scatter_(2, sat, s)
    return rows, new


def _decoded(codes, scale, block):
    B, h, T, d = codes.shape
    return (codes.float().view(B, h, T // block, block, d) * scale[..., None, None]).view(B, h, T, d)


def _plain_prefill(s):
    c = s["case"]
    S, Hkv, d = c["S"], c["Hkv"], c["d"]
    pos = torch.arange(S, device=DEV)[None].expand(c["B"], S)
    q = _rotate(_values(s["q"], s["act"], s["qw"]), s["table"], pos).transpose(1, 2)
    k = _rotate(_values(s["k"], s["act"], s["kw"]), s["table"], pos).transpose(1, 2)
    v = _values(s["v"], s["act"], s["vw"]).transpose(1, 2)
    s["k_cache"][:, :, :S] = k
    s["v_cache"][:, :, :S] = v
    row, col = torch.arange(S, device=DEV)[:, None], torch.arange(S, device=DEV)[None]
    see = (col <= row)[None] if s["end"] is None else (col[None] < s["end"][:, :, None])
    if s["begin"] is not None:
        see = see & (col[None] >= s["begin"][:, :, None])
    o, _ = _attend(q.contiguous(), k.contiguous(), v.contiguous(), see[:, None], (row - col).abs()[None, None], s["slopes"], c["softcap"])
    s["out"].copy_(o)
    return s["out"], s["k_cache"], s["v_cache"]


def _plain_decode(s):
    c = s["case"]
    B, T = c["B"], c["T"]
    past = s["past"].long()
    q = _rotate(_values(s["q"], s["act"], s["qw"]), s["table"], past[:, None]).transpose(1, 2)
    k = _rotate(_values(s["k"], s["act"], s["kw"]), s["table"], past[:, None]).transpose(1, 2)
    v = _values(s["v"], s["act"], s["vw"]).transpose(1, 2)
    b = torch.arange(B, device=DEV)
    s["k_cache"][b, :, past] = k[:, :, 0].to(s["k_cache"].dtype)
    s["v_cache"][b, :, past] = v[:, :, 0].to(s["v_cache"].dtype)
    row = torch.arange(T, device=DEV)[None]
    see = row <= past[:, None]
    if s["begin"] is not None:
        see = see & (row >= s["begin"].long()[:, None])
    o, _ = _attend(q.contiguous(), s["k_cache"].float(), torch.where(see[:, None, :, None], s["v_cache"].float(), torch.zeros((), device=DEV)),
                   see[:, None, None], (past[:, None] - row).abs()[:, None, None], s["slopes"], c["softcap"])
    s["out"].copy_(o)
    return s["out"], s["k_cache"], s["v_cache"]


def _plain_append(s):
    c = s["case"]
    B, S = c["B"], c["S"]
    pos = s["past"].long()[:, None] + torch.arange(S, device=DEV)
    count = s["new"] if s["new"] is not None else torch.full((B,), S, device=DEV)
    k = _rotate(_values(s["k"], s["act"], s["kw"]), s["table"], pos.clamp_max(c["T"] - 1)).transpose(1, 2)
    v = _values(s["v"], s["act"], s["vw"]).transpose(1, 2)
    _append_one(s["k_codes"], s["k_scale"], k, s["past"], count, c["block"], c["code"])
    rows, new = _append_one(s["v_codes"], s["v_scale"], v, s["past"], count, c["block"], c["code"])
    at = rows[:, None].expand(new.shape)
    s["row_pos"].scatter_(2, at, torch.where(new, at.to(torch.int32), torch.gather(s["row_pos"], 2, at)))
    return s["k_codes"], s["k_scale"], s["v_codes"], s["v_scale"], s["row_pos"]


def _plain_decode8(s):
    c = s["case"]
    B, T, Hkv, block = c["B"], c["T"], c["Hkv"], c["block"]
    past = s["past"].long()
    q = _rotate(_values(s["q"], s["act"], s["qw"]), s["table"], past[:, None]).transpose(1, 2)
    k = _rotate(_values(s["k"], s["act"], s["kw"]), s["table"], past[:, None]).transpose(1, 2)
    v = _values(s["v"], s["act"], s["vw"]).transpose(1, 2)
    one = torch.ones(B, device=DEV)
    _append_one(s["k_codes"], s["k_scale"], k, past, one, block, c["code"])
    _append_one(s["v_codes"], s["v_scale"], v, past, one, block, c["code"])
    s["row_pos"].scatter_(2, past[:, None, None].expand(B, Hkv, 1), past[:, None, None].expand(B, Hkv, 1).to(torch.int32))
    row = torch.arange(T, device=DEV)[None]
    see = row <= past[:, None]
    if s["begin"] is not None:
        see = see & (row >= s["begin"].long()[:, None])
    o, p = _attend(q.contiguous(), _decoded(s["k_codes"], s["k_scale"], block), _decoded(s["v_codes"], s["v_scale"], block),
                   see[:, None, None], (past[:, None, None] - s["row_pos"]).abs()[:, :, None], s["slopes"], c["softcap"])
    s["out"].copy_(o)
    r = [s["out"], s["k_codes"], s["k_scale"], s["v_codes"], s["v_scale"]]
    if c["weights"]:
        w = torch.where(row[:, None] == past[:, None, None], torch.zeros_like(s["w_in"]), s["w_in"]) + p.view(B, Hkv, -1, T).sum(2)
        s["w_out"].copy_(torch.where(row[:, None] <= past[:, None, None], w, s["w_out"]))
        r.append(s["w_out"])
    return r


def _plain_evict(s):
    c = s["case"]
    B, Hkv, T, d, block = c["B"], c["Hkv"], c["T"], c["d"], c["block"]
    n = s["past"].long()[:, None, None]
    m = n.clamp_max(c["budget"])
    row = torch.arange(T, device=DEV).expand(B, Hkv, T)
    pos, w = s["row_pos"], s["w_in"]
    held = row < n
    first = (pos < c["sinks"]) | (pos >= s["next"][:, None, None] - c["recent"])
    # by weight, then the protected rows in front, then what is held at all: each sort keeps the order of the one before among equals
    order = torch.sort(w, dim=-1, descending=True, stable=True).indices
    order = torch.gather(order, 2, torch.sort(torch.gather(first, 2, order).to(torch.int8), dim=-1, descending=True, stable=True).indices)
    order = torch.gather(order, 2, torch.sort(torch.gather(held, 2, order).to(torch.int8), dim=-1, descending=True, stable=True).indices)
    rank = torch.empty_like(order).scatter_(2, order, row)
    keep = held & (rank < c["budget"])
    hole = (row < m) & ~keep
    source = torch.sort((keep & (row >= m)).to(torch.int8), dim=-1, descending=True, stable=True).indices
    source = torch.gather(source, 2, (hole.long().cumsum(-1) - 1).clamp_min(0))
    source = torch.where(hole, source, row)
    at = source[..., None].expand(B, Hkv, T, d)
    shape = (B, Hkv, T // block, block)
    no = torch.zeros(shape[:3], dtype=torch.bool, device=DEV)
    for which in ("k", "v"):
        codes, scale = s[which + "_codes"], s[which + "_scale"]
        x = torch.gather(_decoded(codes, scale, block), 2, at)
        a, b = _merge(codes.view(*shape, d), scale, x.view(*shape, d), hole.view(shape), (row < m).view(shape), no, c["code"])
        codes.copy_(a.view(B, Hkv, T, d))
        scale.copy_(b)
    s["w_out"].copy_(torch.where(row < m, torch.gather(w, 2, source), s["w_out"]))
    s["pos_out"].copy_(torch.where(row < m, torch.gather(pos, 2, source), s["pos_out"]))
    s["len_out"].copy_(m.view(B))
    return s["k_codes"], s["k_scale"], s["v_codes"], s["v_scale"], s["w_out"], s["pos_out"], s["len_out"]


# ---------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------
def run(state):
    s, c = state, state["case"]
    if not own:
        return {"prefill": _plain_prefill, "decode": _plain_decode, "append": _plain_append, "decode8": _plain_decode8, "evict": _plain_evict}[c["op"]](s)
    from fasterllama_b200 import attention as A
    from fasterllama_b200 import kv8

    if c["op"] in ("prefill", "decode"):
        if c["op"] == "prefill":
            mode = A.FLB_MASK_CAUSAL_INCLUSIVE if s["end"] is None else A.FLB_MASK_NONE
            more = dict(mask_mode=mode, key_end=s["end"])
        else:
            more = dict(past_lens=s["past"], max_past_len=c["most"], rope_add_past=True)
        p, f = A.make_scored_params(
            q=s["q"], k=s["k"], v=s["v"], k_cache=s["k_cache"], v_cache=s["v_cache"], out=s["out"], scratch=s["scratch"], act_scale=s["act"],
            q_w_scale=s["qw"], k_w_scale=s["kw"], v_w_scale=s["vw"], freq_cis=s["table"], softcap=c["softcap"], alibi_slopes=s["slopes"],
            key_begin=s["begin"], scratch_zeroed=c["op"] == "decode", **more)
        A.forward_scored(p, f)
        return s["out"], s["k_cache"], s["v_cache"]
    cache = kv8.Cache(s["k_codes"], s["v_codes"], s["k_scale"], s["v_scale"], row_pos=s["row_pos"])
    if c["op"] == "append":
        kv8.append(cache, s["k"], s["v"], past_lens=s["past"], new_lens=s["new"], act_scale=s["act"], k_w_scale=s["kw"], v_w_scale=s["vw"],
                   freq_cis=s["table"], scratch=s["scratch"])
        return s["k_codes"], s["k_scale"], s["v_codes"], s["v_scale"], s["row_pos"]
    if c["op"] == "decode8":
        kv8.decode(cache, s["q"], s["k"], s["v"], s["out"], past_lens=s["past"], max_past_len=c["most"], act_scale=s["act"], q_w_scale=s["qw"],
                   k_w_scale=s["kw"], v_w_scale=s["vw"], freq_cis=s["table"], softcap=c["softcap"], alibi_slopes=s["slopes"], key_begin=s["begin"],
                   weight_in=s.get("w_in"), weight_out=s.get("w_out"), scratch=s["scratch"], scratch_zeroed=True)
        r = [s["out"], s["k_codes"], s["k_scale"], s["v_codes"], s["v_scale"]]
        return r + [s["w_out"]] if c["weights"] else r
    kv8.evict(cache, past_lens=s["past"], len_out=s["len_out"], budget=c["budget"], recent=c["recent"], sinks=c["sinks"], next_pos=s["next"],
              weight=s["w_in"], weight_out=s["w_out"], pos_out=s["pos_out"], scratch=s["scratch"])
    return s["k_codes"], s["k_scale"], s["v_codes"], s["v_scale"], s["w_out"], s["pos_out"], s["len_out"]


def work(case):
    c = case
    op, B, d = c["op"], c["B"], c["d"]
    size = {"float16": 2, "float32": 4, "int32": 4}
    mean = (min(c["least"], c["most"]) + c["most"]) / 2 if "most" in c else 0
    if op == "prefill":
        H, Hkv, S = c["H"], c["Hkv"], c["S"]
        e = size[c["io"]]
        pairs = S * (S + 1) / 2
        if c["mask"] == "documents":
            n = min(5.0, S / 2.0)  # five documents of about equal length
            pairs = pairs / n
        return {"bytes": B * S * d * ((H + 2 * Hkv) * e + 2 * Hkv * size[c["cache"]] + 2 * H), "flops": 4.0 * B * H * d * pairs}
    if op == "decode":
        H, Hkv = c["H"], c["Hkv"]
        seen = min(mean, c["window"]) if c["window"] else mean
        ec = size[c["cache"]]
        return {"bytes": B * d * (2 * Hkv * (seen + 1) * ec + (H + 2 * Hkv) * size[c["io"]] + 4 * H), "flops": 4.0 * B * H * d * (seen + 1)}
    if op == "append":
        n = c["S"] * (0.5 + 0.5 / B if c["ragged"] else 1.0)
        return {"bytes": B * c["Hkv"] * n * (2 * d * (size[c["io"]] + 1) + 4 + 8.0 / c["block"]), "flops": 8.0 * B * c["Hkv"] * n * d}
    if op == "decode8":
        H, Hkv = c["H"], c["Hkv"]
        seen = min(mean, c["window"]) if c["window"] else mean
        n = B * Hkv * (seen + 1) * (2 * d + 8.0 / c["block"] + (4 if c["alibi"] or c["window"] else 0) + (8 if c["weights"] else 0))
        return {"bytes": n + B * d * ((H + 2 * Hkv) * size[c["io"]] + size[c["out"]] * H), "flops": 4.0 * B * H * d * (seen + 1)}
    n = B * c["Hkv"] * mean
    kept = min(mean, c["budget"])
    moved = B * c["Hkv"] * kept * max(0.0, mean - c["budget"]) / max(mean, 1.0)  # kept rows are spread evenly
    return {"bytes": n * 8 + B * c["Hkv"] * kept * 8 + moved * 4 * d, "flops": n * 4.0}


# ---------------------------------------------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------------------------------------------
def _x_values(x, act, w):
    if x.dtype == torch.int32:
        return x.double() * act.double().reshape(x.shape[0], x.shape[1], 1, 1) * w.double().reshape(x.shape[2], x.shape[3])
    return x.double()


def _x_turn(x, table, at):
    """One sequence [S,heads,d] turned as complex numbers by the rows `at` of the table."""
    z = torch.view_as_complex(x.reshape(*x.shape[:-1], -1, 2).contiguous())
    t = torch.view_as_complex(table.double()[at].reshape(len(at), -1, 2))
    return torch.view_as_real(z * t[:, None]).reshape(x.shape)


def _x_softmax(q, k, v, hide, bias, cap):
    """One head: q [S,d], k, v [K,d], hide [S,K] -> rows and probabilities."""
    x = q @ k.T / math.sqrt(q.shape[-1])
    if cap:
        x = cap * torch.tanh(x / cap)
    if bias is not None:
        x = x + bias
    x = x.masked_fill(hide, -math.inf)
    p = torch.softmax(x, -1)
    p = torch.where(hide.all(-1, keepdim=True), torch.zeros_like(p), p)
    return p @ v, p


def _x_grow(codes, scale, x, rows, start, block, code):
    """Rows x [n,d] at `rows` (rising) of one head's cache of 64-bit codes, by the rule of the operator, in place; `start`: blocks from there on are new."""
    top = 127.0 if code == "int8" else 448.0

    def near(y):
        return y.round().clamp(-127, 127) if code == "int8" else y.clamp(-448, 448).to(torch.float8_e4m3fn).double()

    for j in sorted(set((rows // block).tolist())):
        m = rows // block == j
        was = 0.0 if j * block >= start else float(scale[j])
        now = max(was, float(x[m].abs().max()) / top)
        if now > was:
            if was:
                codes[j * block:(j + 1) * block] = near(codes[j * block:(j + 1) * block] * (was / now))
            scale[j] = now
        elif j * block >= start:
            scale[j] = now
        codes[rows[m]] = near(x[m] / now) if now > 0 else 0.0


def exact(case, seed):
    s = prepare(case, seed)
    c = s["case"]
    op, B = c["op"], c["B"]
    if op in ("prefill", "decode", "decode8"):
        H, Hkv, d = c["H"], c["Hkv"], c["d"]
        G = H // Hkv
        q, k, v = (_x_values(s[n], s["act"], s[n + "w"]) for n in "qkv")
        o = torch.zeros(s["out"].shape, dtype=torch.float64, device=DEV)
        slope = s["slopes"].double() if s["slopes"] is not None else None
    if op == "prefill":
        S = c["S"]
        kc, vc = s["k_cache"].double(), s["v_cache"].double()
        at = torch.arange(S, device=DEV)
        for b in range(B):
            qb, kb = _x_turn(q[b], s["table"], at), _x_turn(k[b], s["table"], at)
            kc[b, :, :S], vc[b, :, :S] = kb.transpose(0, 1), v[b].transpose(0, 1)
            low = s["begin"][b].long() if s["begin"] is not None else torch.zeros_like(at)
            high = s["end"][b].long() if s["end"] is not None else at + 1
            hide = (at[None] < low[:, None]) | (at[None] >= high[:, None])
            for h in range(H):
                bias = -slope[h] * (at[:, None] - at[None]).abs().double() if slope is not None else None
                o[b, h] = _x_softmax(qb[:, h], kb[:, h // G], v[b, :, h // G], hide, bias, c["softcap"])[0]
        return o, kc, vc
    if op == "decode":
        kc, vc = s["k_cache"].double(), s["v_cache"].double()
        for b in range(B):
            n = int(s["past"][b])
            at = torch.tensor([n], device=DEV)
            qb = _x_turn(q[b], s["table"], at)[0]
            kc[b, :, n], vc[b, :, n] = _x_turn(k[b], s["table"], at)[0], v[b, 0]
            low = int(s["begin"][b]) if s["begin"] is not None else 0
            r = torch.arange(n + 1, device=DEV)
            # what the cache holds is what was rounded to its type
            kr, vr = kc[b, :, :n + 1].to(s["k_cache"].dtype).double(), vc[b, :, :n + 1].to(s["v_cache"].dtype).double()
            for h in range(H):
                bias = -slope[h] * (n - r).double()[None] if slope is not None else None
                o[b, h] = _x_softmax(qb[h][None], kr[h // G], vr[h // G], (r < low)[None], bias, c["softcap"])[0]
        return o, kc, vc
    if op == "append":
        if B * c["Hkv"] * (c["S"] // c["block"] + 1) > 20000:
            return None
        k, v = _x_values(s["k"], s["act"], s["kw"]), _x_values(s["v"], s["act"], s["vw"])
        ks, vs = s["k_scale"].double(), s["v_scale"].double()
        for b in range(B):
            n, m = int(s["past"][b]), c["S"] if s["new"] is None else int(s["new"][b])
            at = torch.arange(n, n + m, device=DEV)
            kb = _x_turn(k[b, :m], s["table"], at) if m else k[b, :0]
            for h in range(c["Hkv"]):
                if m:
                    _x_grow(s["k_codes"][b, h].double(), ks[b, h], kb[:, h], at, n, c["block"], c["code"])
                    _x_grow(s["v_codes"][b, h].double(), vs[b, h], v[b, :m, h], at, n, c["block"], c["code"])
                s["row_pos"][b, h, n:n + m] = at.to(torch.int32)
        # the codes are whole values (or their 8-bit floats) of which both sides have to hold the same
        return None, ks, None, vs, s["row_pos"]
    if op == "decode8":
        if B * Hkv > 2000:
            return None
        block = c["block"]
        ks, vs = s["k_scale"].double(), s["v_scale"].double()
        w = s["w_out"].double() if c["weights"] else None
        for b in range(B):
            n = int(s["past"][b])
            at = torch.tensor([n], device=DEV)
            qb, kb = _x_turn(q[b], s["table"], at)[0], _x_turn(k[b], s["table"], at)[0]
            low = int(s["begin"][b]) if s["begin"] is not None else 0
            r = torch.arange(n + 1, device=DEV)
            for j in range(Hkv):
                kc, vc = s["k_codes"][b, j, :(n // block + 1) * block].double(), s["v_codes"][b, j, :(n // block + 1) * block].double()
                _x_grow(kc, ks[b, j], kb[j][None], at, n, block, c["code"])
                _x_grow(vc, vs[b, j], v[b, 0, j][None], at, n, block, c["code"])
                kr, vr = kc[:n + 1] * ks[b, j][r // block][:, None], vc[:n + 1] * vs[b, j][r // block][:, None]
                if w is not None:
                    w[b, j, :n] = s["w_in"][b, j, :n].double()
                    w[b, j, n] = 0.0
                for h in range(j * G, (j + 1) * G):
                    bias = -slope[h] * (n - r).double()[None] if slope is not None else None
                    o[b, h], p = _x_softmax(qb[h][None], kr, vr, (r < low)[None], bias, c["softcap"])
                    if w is not None:
                        w[b, j, :n + 1] += p[0]
        r = [o, None, ks, None, vs]
        return r + [w] if c["weights"] else r
    ks, vs = s["k_scale"].double(), s["v_scale"].double()
    w, pos = s["w_in"].double().cpu().numpy(), s["row_pos"].cpu().numpy()
    w_out, pos_out = s["w_out"].double().cpu().numpy(), s["pos_out"].cpu().numpy().copy()
    lens, nxt = s["past"].cpu().numpy(), s["next"].cpu().numpy()
    if B * c["Hkv"] * (c["T"] // c["block"]) > 20000:
        return None
    for b in range(B):
        n = int(lens[b])
        m = min(n, c["budget"])
        for h in range(c["Hkv"]):
            weight, place = w[b, h, :n], pos[b, h, :n]
            safe = (place < c["sinks"]) | (place >= nxt[b] - c["recent"])
            kept = np.lexsort((np.arange(n), -weight, ~safe))[:m]
            stay = np.zeros(n, dtype=bool)
            stay[kept] = True
            holes, moved = np.flatnonzero(~stay[:m]), m + np.flatnonzero(stay[m:])
            w_out[b, h, :m], pos_out[b, h, :m] = weight[:m], place[:m]
            w_out[b, h, holes], pos_out[b, h, holes] = weight[moved], place[moved]
            if len(holes):
                to, of = torch.from_numpy(holes).to(DEV), torch.from_numpy(moved).to(DEV)
                for codes, scale in ((s["k_codes"], ks), (s["v_codes"], vs)):
                    x = codes[b, h][of].double() * scale[b, h][of // c["block"]][:, None]
                    _x_grow(codes[b, h].double(), scale[b, h], x, to, c["T"], c["block"], c["code"])
    return None, ks, None, vs, torch.from_numpy(w_out).to(DEV), torch.from_numpy(pos_out).to(DEV), torch.from_numpy(np.minimum(lens, c["budget"])).to(DEV)
