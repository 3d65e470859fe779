"""Plain implementations in 64 bits of the score forms, the 8-bit cache and eviction, for the tests of those calls.

The coding rule of the 8-bit cache is defined by IEEE fp32 operations (include/flb_kv8.h); it is restated with them, so codes
and scales have to be equal bit for bit.  Everything behind the codes is in 64 bits."""
from __future__ import annotations

import numpy as np
import torch

TOP = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}


def values(x, act=None, w=None):
    """[B,S,heads,d] as the projections leave them -> fp32 (the order of the products is part of the interface)."""
    if x.dtype != torch.int32:
        return x.float()
    B, S, h, d = x.shape
    return (x.float() * act.view(B, S, 1, 1)) * w.view(h, d)


def rotate(x, table, pos):
    """fp32 rotation of the pairs (2i, 2i+1), every product rounded on its own; x [B,S,heads,d], pos [B,S]."""
    if table is None:
        return x
    f = table[pos.long()].unsqueeze(2)
    co, sn, a, b = f[..., 0::2], f[..., 1::2], x[..., 0::2], x[..., 1::2]
    return torch.stack([a * co - b * sn, b * co + a * sn], -1).reshape(x.shape)


def attend(q, k, v, see, scale, *, cap=0.0, bias=None, mask=None):
    """One head in 64 bits: q [S,d], k, v [K,d], see [S,K] -> (out [S,d], weights [S,K], log2-domain magnitude of the scores)."""
    q, k, v = q.double(), k.double(), v.double()
    x = q @ k.T * scale
    if cap:
        x = cap * torch.tanh(x / cap)
    if bias is not None:
        x = x + bias
    if mask is not None:
        x = x + mask.double()
    x = torch.where(see, x, torch.full_like(x, -torch.inf))
    m = x.amax(-1, keepdim=True)
    p = torch.where(see, torch.exp(x - torch.where(torch.isfinite(m), m, torch.zeros_like(m))), torch.zeros_like(x))
    n = p.sum(-1, keepdim=True)
    p = torch.where(n > 0, p / n, torch.zeros_like(p))
    return torch.where(see.any(-1, keepdim=True), torch.where(p == 0, torch.zeros_like(p), p) @ torch.where(see.any(0)[:, None], v, torch.zeros_like(v)),
                       torch.zeros_like(q)), p


def code(y, dtype):
    if dtype == torch.int8:
        return y.round().clamp(-127, 127).to(torch.int8)
    return y.clamp(-448, 448).to(dtype)


def put_rows(codes, scale, x, rows, live, fresh_from, block):
    """Rows x [n,d] (fp32) at `rows` of one head's cache, in place: codes [T,d], scale [T/block]; rows below `live` are held, blocks from
    row `fresh_from` on start with the new rows."""
    dt = codes.dtype
    top = torch.tensor(TOP[dt], device=codes.device)
    for j in sorted({int(r) // block for r in rows}):
        m = torch.tensor([i for i, r in enumerate(rows) if int(r) // block == j], device=codes.device)
        new = torch.tensor([int(r) for r in rows if int(r) // block == j], device=codes.device)
        need = x[m].abs().amax() / top
        old = torch.zeros((), device=codes.device) if j * block >= fresh_from else scale[j].clone()
        s = torch.maximum(old, need)
        if bool(s > old) and bool(old > 0):
            a, b = j * block, min((j + 1) * block, live)
            if b > a:
                codes[a:b] = code(codes[a:b].float() * (old / s), dt)
        ok = bool(torch.isfinite(s)) and float(s) > 0
        codes[new] = code(x[m] / s, dt) if ok else torch.zeros_like(x[m]).to(dt)
        scale[j] = s


def dequant(codes, scale, block):
    return codes.double() * scale.double().repeat_interleave(block)[:, None]


def evict_plan(weight, pos, n, budget, recent, sinks, next_pos):
    """(kept rows below m that stay, holes, sources) of one head; numpy arrays."""
    m = min(n, budget)
    w, p = weight[:n].astype(np.float64), pos[:n].astype(np.int64)
    safe = p < sinks
    if next_pos is not None:
        safe = safe | (p >= int(next_pos) - recent)
    w = np.where(np.isnan(w), np.inf, w)
    nan = np.isnan(weight[:n])
    order = np.lexsort((np.arange(n), -w, ~nan, ~safe))
    keep = np.zeros(n, bool)
    keep[order[:m]] = True
    return m, np.flatnonzero(~keep[:m]), m + np.flatnonzero(keep[m:])
