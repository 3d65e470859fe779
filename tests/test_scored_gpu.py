"""Score forms of the prefill and decode calls against the plain implementation in 64 bits."""
import math

import numpy as np
import pytest
import torch

from fasterllama_b200 import _lib
from fasterllama_b200 import attention as A
from fasterllama_b200 import workloads as W

import forms_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def rnd(g, *shape, std=1.0, dtype=torch.float16):
    return (torch.randn(*shape, generator=g, device=DEV) * std).to(dtype)


def slopes_of(H):
    return torch.pow(2.0, -8.0 * torch.arange(1, H + 1, device=DEV) / H)


def bounds(kind, B, S, g):
    """(key_begin, key_end, mask mode) of the masks that real prompts bring."""
    row = torch.arange(S, dtype=torch.int32, device=DEV).expand(B, S)
    if kind == "causal":
        return None, None, A.FLB_MASK_CAUSAL_INCLUSIVE
    if kind == "strict":
        return None, None, A.FLB_MASK_CAUSAL_STRICT
    if kind == "none":
        return None, None, A.FLB_MASK_NONE
    if kind == "documents":
        cut = torch.rand(B, S, generator=g, device=DEV) < 5.0 / S
        return torch.cummax(torch.where(cut, row, torch.zeros_like(row)), 1).values.to(torch.int32).contiguous(), None, A.FLB_MASK_CAUSAL_INCLUSIVE
    if kind == "window":
        return (row - 40).contiguous(), None, A.FLB_MASK_CAUSAL_INCLUSIVE  # negative bounds in front
    if kind == "prefix":
        return None, torch.maximum(row + 1, torch.full_like(row, S // 3 + 1)).contiguous(), A.FLB_MASK_NONE
    if kind == "padded":
        n = torch.randint(0, S + 1, (B, 1), generator=g, device=DEV)
        return None, torch.where(row < n, row + 1, torch.zeros_like(row)).contiguous(), A.FLB_MASK_NONE
    if kind == "holes":  # any bounds: rows that see nothing, bounds outside the prompt, crossed bounds
        a = torch.randint(-5, S + 5, (B, S), generator=g, device=DEV, dtype=torch.int32)
        b = torch.randint(-5, S + 5, (B, S), generator=g, device=DEV, dtype=torch.int32)
        b[:, ::3] = 2147483647
        a[:, 1::5] = -2147483648
        return a, b, A.FLB_MASK_NONE
    if kind == "ends":
        low, high = (torch.full((B, S), x, dtype=torch.int32, device=DEV) for x in (-2147483648, 2147483647))
        a, b = low.clone(), high.clone()
        b[:, 1::4] = -2147483648
        a[:, 2::4] = 2147483647
        b[:, 3::4] = -1
        return a, b, A.FLB_MASK_NONE
    raise AssertionError(kind)


def run_prefill(seed, *, B, H, Hkv, S, d, kind="causal", cap=0.0, alibi=False, cache="float16", out="float32", io="float16", rope=False, std=1.0, generic=False, T=None):
    """Without rotation fp16 inputs are the tensor cores' operands as they are: what is left is the weights' fp16 rounding (half a step,
    2^-11 relative to each), the fp32 sums and the cap's fit.  With rotation the plain form takes operands rounded to fp16 as the kernel does; a rotation
    may round to the neighbouring fp16 value where a product was fused, a step of 2^-10 in single elements."""
    g = gen(seed)
    T = T or S + 3
    q, k, v = rnd(g, B, S, H, d, std=std), rnd(g, B, S, Hkv, d), rnd(g, B, S, Hkv, d)
    if io == "float32":
        q, k, v = q.float(), k.float(), v.float()
    kc, vc = (torch.full((B, Hkv, T, d), 7.0, dtype=getattr(torch, cache), device=DEV) for _ in range(2))
    o = torch.full((B, H, S, d), math.nan, dtype=getattr(torch, out), device=DEV)
    begin, end, mode = bounds(kind, B, S, g)
    tab = torch.from_numpy(W.freq_cis_table(T, d)).to(DEV) if rope else None
    mask = None
    if generic:
        mask = torch.where(torch.rand(S, S, generator=g, device=DEV) < 0.1, -torch.finfo(torch.float32).max, -torch.rand(S, S, generator=g, device=DEV)).contiguous()
        mode = A.FLB_MASK_GENERIC
    sl = slopes_of(H) if alibi else None
    scratch = torch.full((A.workspace_bytes(B, H, T, S, size_per_head=d) + 65536,), 0xA5, dtype=torch.uint8, device=DEV)
    p, f = A.make_scored_params(q=q, k=k, v=v, k_cache=kc, v_cache=vc, out=o, scratch=scratch, freq_cis=tab, mask_mode=mode, attn_mask=mask, softcap=cap,
                                alibi_slopes=sl, key_begin=begin, key_end=end)
    p.scratch_bytes = A.scored_workspace_bytes(p, f)  # no byte more than it asks for
    A.forward_scored(p, f)
    torch.cuda.synchronize()
    assert A.scratch_status(scratch) == 0
    pos = torch.arange(S, device=DEV).expand(B, S)
    kr = R.rotate(k.float(), tab, pos)
    assert torch.allclose(kc[:, :, :S].float(), kr.transpose(1, 2).to(kc.dtype).float(), rtol=2.0 ** -10 if cache == "float16" else 1e-5, atol=1e-6)
    assert torch.equal(vc[:, :, :S], v.transpose(1, 2).to(vc.dtype))
    assert bool((kc[:, :, S:] == 7).all()) and bool((vc[:, :, S:] == 7).all())
    qh, kh = R.rotate(q.float(), tab, pos).half().double(), kr.half().double()
    row = torch.arange(S, device=DEV)
    lo = begin.long() if begin is not None else torch.zeros(B, S, dtype=torch.long, device=DEV)
    hi = end.long() if end is not None else torch.full((B, S), S, device=DEV)
    if mode == A.FLB_MASK_CAUSAL_INCLUSIVE:
        hi = torch.minimum(hi, row + 1)
    if mode == A.FLB_MASK_CAUSAL_STRICT:
        hi = torch.minimum(hi, row)
    scale = 1.0 / math.sqrt(d)
    vmax, qk = float(v.float().abs().max()), float(qh.abs().max() * kh.abs().max()) * scale
    # log-domain error of a score: the products' fp32 sum, the finished score's roundings, the cap's fit (2.8e-6 of the cap), the bias
    size = float(qh.norm(dim=-1).max() * kh.norm(dim=-1).max()) * scale
    ds = size * (d / 16 + 16) * 2.0 ** -23 + (3e-6 + 2.0 ** -21) * cap + (S * 2.0 ** -22 if alibi else 0.0) + (4 * 2.0 ** -10 * qk if rope else 0.0)
    tol = vmax * (2 * ds + 2 * 2.0 ** -11 + (S / 16 + 64) * 2.0 ** -23)
    for b in range(B):
        see = (row[None] >= lo[b][:, None]) & (row[None] < hi[b][:, None])
        seen = see & (mask > -1e30) if generic else see
        for h in range(H):
            bias = -sl[h].double() * (row[:, None] - row[None]).abs().double() if alibi else None
            want, _ = R.attend(qh[b, :, h], kh[b, :, h // (H // Hkv)], v[b, :, h // (H // Hkv)].half(), seen, scale, cap=cap, bias=bias, mask=mask)
            err = (o[b, h].double() - want).abs()
            lim = tol + torch.finfo(o.dtype).eps / 2 * want.abs()
            assert bool((err <= lim).all()), (b, h, float(err.max()), tol, (err > lim).nonzero()[0].tolist())
            assert float(o[b, h][~seen.any(-1)].float().abs().sum()) == 0
    return q, k, v, o


@pytest.mark.parametrize("S", [2, 63, 64, 65, 127, 128, 129, 191, 256, 257, 300, 513])
@pytest.mark.parametrize("kind", ["documents", "prefix", "padded", "holes", "window"])
def test_prefill_bounds(cuda_device, S, kind):
    run_prefill(S, B=2, H=2, Hkv=2, S=S, d=128 if S % 2 else 64, kind=kind)


@pytest.mark.parametrize("S", [130, 300])
def test_prefill_bounds_at_the_ends_of_their_type(cuda_device, S):
    """Rows whose bounds are the type's lowest and highest values, among rows that see every key."""
    run_prefill(28, B=2, H=2, Hkv=2, S=S, d=64, kind="ends")


@pytest.mark.parametrize("kind", ["causal", "strict", "none", "documents", "prefix", "holes"])
@pytest.mark.parametrize("H,Hkv,d", [(4, 4, 128), (8, 2, 128), (5, 1, 64), (6, 3, 64)])
@pytest.mark.parametrize("cap,alibi,std", [(0.0, False, 1.0), (15.0, False, 2.0), (2.0, False, 4.0), (0.0, True, 1.0), (30.0, True, 1.0)])
def test_prefill_forms(cuda_device, kind, H, Hkv, d, cap, alibi, std):
    run_prefill(H + d, B=2, H=H, Hkv=Hkv, S=201, d=d, kind=kind, cap=cap, alibi=alibi, std=std)


@pytest.mark.parametrize("cap", [2.0 ** -10, 2.0 ** 40])
def test_prefill_caps_at_the_ends_of_their_range(cuda_device, cap):
    """The smallest leaves nearly even weights, the largest leaves the scores (its fit is off by 2.1e-5 of a score there, scores are below 8)."""
    S, d = 200, 64
    g = gen(29)
    q, k, v = rnd(g, 1, S, 2, d), rnd(g, 1, S, 2, d), rnd(g, 1, S, 2, d)
    outs = []
    for c in (cap, 0.0):
        kc, vc = (torch.zeros(1, 2, S, d, dtype=torch.float16, device=DEV) for _ in range(2))
        o = torch.empty(1, 2, S, d, device=DEV)
        scratch = torch.zeros(A.workspace_bytes(1, 2, S, S, size_per_head=d) + 65536, dtype=torch.uint8, device=DEV)
        p, f = A.make_scored_params(q=q, k=k, v=v, k_cache=kc, v_cache=vc, out=o, scratch=scratch, softcap=c, mask_mode=A.FLB_MASK_NONE,
                                    softmax_scale=0.125 if c else 0.125 if cap > 1 else 1e-30)
        A.forward_scored(p, f)
        outs.append(o)
    # weights: both sides in fp16 (2^-11 each), log-domain difference 2 * cap or 2 * 8 * 2.1e-5
    tol = float(v.float().abs().max()) * (2 * 2.0 ** -11 + (2 * cap if cap < 1 else 4e-4))
    assert float((outs[0] - outs[1]).abs().max()) <= tol


@pytest.mark.parametrize("cache", ["float16", "float32"])
@pytest.mark.parametrize("out", ["float16", "float32"])
@pytest.mark.parametrize("io", ["float16", "float32"])
@pytest.mark.parametrize("rope", [True, False])
def test_prefill_types(cuda_device, cache, out, io, rope):
    run_prefill(3, B=1, H=4, Hkv=2, S=130, d=128, kind="prefix", cap=20.0, cache=cache, out=out, io=io, rope=rope)
    run_prefill(4, B=1, H=4, Hkv=2, S=130, d=64, kind="causal", alibi=True, cache=cache, out=out, io=io, rope=rope)


@pytest.mark.parametrize("kind", ["none", "documents", "holes"])
def test_prefill_with_the_callers_additive_mask(cuda_device, kind):
    run_prefill(5, B=2, H=2, Hkv=1, S=140, d=128, kind=kind, cap=10.0, alibi=True, generic=True)


def test_prefill_many_items_per_block(cuda_device):
    """More work items than SMs: the rings and phases run on from item to item, of different lengths and first tiles."""
    run_prefill(6, B=5, H=16, Hkv=8, S=700, d=64, kind="documents", cap=30.0)
    run_prefill(7, B=3, H=32, Hkv=32, S=520, d=128, kind="holes", alibi=True)


def test_prefill_int32_inputs_share_heads(cuda_device):
    """int32 sums with their scales against the same values handed over as fp32."""
    g = gen(8)
    B, H, Hkv, S, d = 2, 4, 2, 77, 128
    act = (torch.rand(B * S, generator=g, device=DEV) + 0.5) / 64
    outs = []
    raw = {n: (rnd(g, B, S, h, d, dtype=torch.float32) * 4096).round().int() for n, h in (("q", H), ("k", Hkv), ("v", Hkv))}
    ws = {n: (torch.rand(h * d, generator=g, device=DEV) + 0.5) / 64 for n, h in (("q", H), ("k", Hkv), ("v", Hkv))}
    for form in ("int32", "float32"):
        x = raw if form == "int32" else {n: R.values(t, act, ws[n]) for n, t in raw.items()}
        kc, vc = (torch.zeros(B, Hkv, S, d, device=DEV) for _ in range(2))
        o = torch.empty(B, H, S, d, device=DEV)
        scratch = torch.zeros(A.workspace_bytes(B, H, S, S) + 65536, dtype=torch.uint8, device=DEV)
        scales = dict(act_scale=act, q_w_scale=ws["q"], k_w_scale=ws["k"], v_w_scale=ws["v"]) if form == "int32" else {}
        p, f = A.make_scored_params(**x, k_cache=kc, v_cache=vc, out=o, scratch=scratch, softcap=20.0, **scales)
        A.prefill_scored(p, f)
        outs.append((o, kc, vc))
    for a, b in zip(*outs):
        assert torch.equal(a, b)


# ------------------------------------------------------------------------------------------------ decode
def run_decode(seed, *, B, H, Hkv, T, d, past, cap=0.0, alibi=False, begin=None, cache="float16", out="float32", io="float16", rope=True, std=2.0, split=0, generic=False,
               early=0, poison=True):
    g = gen(seed)
    dt = getattr(torch, cache)
    kc, vc = rnd(g, B, Hkv, T, d, dtype=dt), rnd(g, B, Hkv, T, d, dtype=dt)
    if poison:  # what a sequence does not see may hold anything
        for b in range(B):
            kc[b, :, past[b] + 1:], vc[b, :, past[b] + 1:] = math.nan, math.inf
            if begin is not None:
                kc[b, :, :max(0, min(begin[b], past[b]))], vc[b, :, :max(0, min(begin[b], past[b]))] = math.nan, math.inf
    q, k, v = (rnd(g, B, 1, h, d, std=s, dtype=getattr(torch, io)) for h, s in ((H, std), (Hkv, 1.0), (Hkv, 1.0)))
    tab = torch.from_numpy(W.freq_cis_table(T, d)).to(DEV) if rope else None
    sl = slopes_of(H) if alibi else None
    mask = -torch.rand(T, T, generator=g, device=DEV) if generic else None
    o = torch.full((B, H, 1, d), math.nan, dtype=getattr(torch, out), device=DEV)
    scratch = torch.zeros(A.workspace_bytes(B, H, T, split_len=split, size_per_head=d), dtype=torch.uint8, device=DEV)
    k0, v0 = kc.clone(), vc.clone()
    p, f = A.make_scored_params(q=q, k=k, v=v, k_cache=kc, v_cache=vc, out=o, scratch=scratch, past_lens=torch.tensor(past, dtype=torch.int32, device=DEV),
                                max_past_len=max(past), freq_cis=tab, rope_add_past=True, softcap=cap, alibi_slopes=sl, split_len=split, scratch_zeroed=True, early_start=early,
                                key_begin=None if begin is None else torch.tensor(begin, dtype=torch.int32, device=DEV),
                                mask_mode=A.FLB_MASK_GENERIC if generic else A.FLB_MASK_CAUSAL_INCLUSIVE, attn_mask=mask)
    A.forward_scored(p, f)
    torch.cuda.synchronize()
    assert A.scratch_status(scratch) == 0
    pt = torch.tensor(past, device=DEV)[:, None]
    qr, kr = R.rotate(q.float(), tab, pt), R.rotate(k.float(), tab, pt)
    for b in range(B):
        n = past[b] + 1
        # the row of this token was stored (a fused product may round it to the neighbouring value), no other was touched
        assert torch.allclose(kc[b, :, n - 1].float(), kr[b, 0].to(dt).float(), rtol=torch.finfo(dt).eps, atol=1e-6)
        assert torch.equal(vc[b, :, n - 1], v[b, 0].to(dt))
        for a, c in ((kc, k0), (vc, v0)):
            x, y = (t[b].clone().view(torch.int16 if dt == torch.float16 else torch.int32) for t in (a, c))
            x[:, n - 1] = y[:, n - 1]
            assert torch.equal(x, y)
        rows = torch.arange(n, device=DEV)
        see = (rows >= (begin[b] if begin is not None else 0))[None]
        for h in range(H):
            kd, vd = torch.nan_to_num(kc[b, h // (H // Hkv), :n].double(), 0, 0, 0), vc[b, h // (H // Hkv), :n].double()
            dist = (past[b] - rows).double()
            bias = -sl[h].double() * dist[None] if alibi else None
            want, _ = R.attend(qr[b, 0, h][None], kd, vd, see, 1 / math.sqrt(d), cap=cap, bias=bias, mask=mask[past[b], :n][None] if generic else None)
            if not see.any():
                assert float(o[b, h].float().abs().max()) == 0
                continue
            # fp32 sums of d products and of the weights, the score's roundings, tanhf (2 ulp of the cap); q is rotated with fused products
            size = float((kd[see[0]].abs() @ qr[b, 0, h].double().abs()).max()) / math.sqrt(d)
            ds = size * (d / 16 + 16) * 2.0 ** -23 + (cap + (float(bias[see].abs().max()) if alibi else 0.0) + 1) * 2.0 ** -20
            vmax = float(vd[see[0]].abs().max())
            err = (o[b, h].double() - want).abs()
            assert bool((err <= vmax * (2 * ds + (n / 16 + 64) * 2.0 ** -23) + torch.finfo(o.dtype).eps / 2 * want.abs()).all()), (b, h, float(err.max()))
    return (q, k, v, kc, vc), o


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("cache,io", [("float16", "float16"), ("float32", "float32"), ("float16", "float32")])
@pytest.mark.parametrize("H,Hkv", [(4, 4), (6, 2), (8, 1)])
def test_decode_forms(cuda_device, d, cache, io, H, Hkv):
    past = [0, 1, 31, 255, 256, 511]
    for kw in (dict(cap=10.0), dict(alibi=True), dict(begin=[0, 1, 5, 200, 257, 500]), dict(cap=30.0, alibi=True, begin=[-3, 2, 31, 17, 256, 32])):
        run_decode(d + H, B=6, H=H, Hkv=Hkv, T=512, d=d, past=past, cache=cache, io=io, split=128, **kw)


def test_decode_additive_mask_and_early_start(cuda_device):
    run_decode(50, B=2, H=4, Hkv=2, T=300, d=128, past=[299, 100], generic=True, cap=10.0, alibi=True, begin=[7, 64])
    for level in (1, 2):
        run_decode(51, B=2, H=4, Hkv=4, T=1100, d=128, past=[1099, 600], cap=10.0, begin=[0, 599], early=level)
        run_decode(52, B=2, H=4, Hkv=2, T=1100, d=128, past=[1099, 600], alibi=True, early=level, out="float16")


def test_decode_quantised_output_and_static_shapes(cuda_device):
    """The fused output quantisation reads the scored result."""
    g = gen(53)
    B, H, Hkv, T, d = 2, 4, 2, 256, 128
    kc, vc = rnd(g, B, Hkv, T, d), rnd(g, B, Hkv, T, d)
    q, k, v = rnd(g, B, 1, H, d), rnd(g, B, 1, Hkv, d), rnd(g, B, 1, Hkv, d)
    o = torch.empty(B, H, 1, d, device=DEV)
    q8, qs = torch.empty(B, H * d, dtype=torch.int8, device=DEV), torch.empty(B, device=DEV)
    s = torch.zeros(A.workspace_bytes(B, H, T), dtype=torch.uint8, device=DEV)
    p, f = A.make_scored_params(q=q, k=k, v=v, k_cache=kc, v_cache=vc, out=o, scratch=s, start_pos=255, softcap=5.0, out_q8=q8, out_q8_scale=qs)
    A.decode_scored(p, f)
    want8, wants = torch.empty(B, 1, H * d, dtype=torch.int8, device=DEV), torch.empty(B, device=DEV)
    A.quantize(o, want8, wants)
    assert torch.equal(q8, want8.view(B, H * d)) and torch.equal(qs, wants)


@pytest.mark.parametrize("S", [1, 150])
def test_no_form_is_the_plain_call(cuda_device, S):
    """Bit for bit: a form of zeros, no form, and the plain entry point."""
    g = gen(54)
    B, H, T, d = 2, 4, 256, 128
    q, k, v = (rnd(g, B, S, H, d) for _ in range(3))
    outs = []
    for how in ("plain", "null", "zeros"):
        kc, vc = (torch.ones(B, H, T, d, dtype=torch.float16, device=DEV) for _ in range(2))
        o = torch.empty(B, H, S, d, device=DEV)
        s = torch.zeros(A.workspace_bytes(B, H, T, S), dtype=torch.uint8, device=DEV)
        kw = dict(q=q, k=k, v=v, k_cache=kc, v_cache=vc, out=o, scratch=s, start_pos=0 if S > 1 else 99)
        if how == "plain":
            A.forward(A.make_params(**kw))
        else:
            p, f = A.make_scored_params(**kw)
            A.forward_scored(p, _lib.FlbScoreForm() if how == "zeros" else None)
        outs.append((o, kc, vc))
    for x in outs[1:]:
        for a, b in zip(outs[0], x):
            assert torch.equal(a, b)


@pytest.mark.parametrize("S", [1, 140])
def test_merged_projection_with_shared_heads(cuda_device, S):
    """q, k and v as columns of one [B, S, (H + 2 Hkv) d] projection."""
    g = gen(55)
    B, H, Hkv, T, d = 2, 6, 2, 256, 128
    buf = rnd(g, B, S, (H + 2 * Hkv) * d)
    q, k, v = (buf[:, :, a * d:(a + n) * d].unflatten(2, (n, d)) for a, n in ((0, H), (H, Hkv), (H + Hkv, Hkv)))
    outs = []
    for x in ((q, k, v), tuple(t.contiguous() for t in (q, k, v))):
        kc, vc = (torch.ones(B, Hkv, T, d, dtype=torch.float16, device=DEV) for _ in range(2))
        o = torch.empty(B, H, S, d, device=DEV)
        s = torch.zeros(A.workspace_bytes(B, H, T, S) + 65536, dtype=torch.uint8, device=DEV)
        p, f = A.make_scored_params(q=x[0], k=x[1], v=x[2], k_cache=kc, v_cache=vc, out=o, scratch=s, start_pos=0 if S > 1 else 50, alibi_slopes=slopes_of(H))
        A.forward_scored(p, f)
        outs.append((o, kc, vc))
    for a, b in zip(*outs):
        assert torch.equal(a, b)


def test_scored_prefill_and_decode_in_a_graph(cuda_device):
    g = gen(56)
    B, H, Hkv, S, T, d = 1, 4, 2, 130, 256, 128
    q, k, v = rnd(g, B, S, H, d), rnd(g, B, S, Hkv, d), rnd(g, B, S, Hkv, d)
    q1, k1, v1 = rnd(g, B, 1, H, d), rnd(g, B, 1, Hkv, d), rnd(g, B, 1, Hkv, d)
    kc, vc = (torch.zeros(B, Hkv, T, d, dtype=torch.float16, device=DEV) for _ in range(2))
    o, o1 = torch.empty(B, H, S, d, device=DEV), torch.empty(B, H, 1, d, device=DEV)
    s = torch.zeros(A.workspace_bytes(B, H, T, S) + 65536, dtype=torch.uint8, device=DEV)
    s1 = torch.zeros(A.workspace_bytes(B, H, T), dtype=torch.uint8, device=DEV)
    begin = torch.zeros(B, S, dtype=torch.int32, device=DEV)
    a = A.make_scored_params(q=q, k=k, v=v, k_cache=kc, v_cache=vc, out=o, scratch=s, softcap=10.0, key_begin=begin)
    b = A.make_scored_params(q=q1, k=k1, v=v1, k_cache=kc, v_cache=vc, out=o1, scratch=s1, start_pos=S, scratch_zeroed=True, softcap=10.0)

    def both():
        A.forward_scored(*a)
        A.forward_scored(*b)

    both()
    begin.add_(3)  # the next pass reads other bounds from the same buffer
    both()
    want = o.clone(), o1.clone(), kc.clone()
    begin.sub_(3)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        both()
        begin.add_(3)
    graph.replay()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(want, (o, o1, kc)))


# ------------------------------------------------------------------------------------------------ large caps and scores
def two_keys(less, *, cap, scale, mask_b=0.0, alibi=False, d=64):
    """One query row whose keys have raw scores of 0 but for key 3 (2^30) and key 9 (2^30 - less * 181; less = None: 0); the other rows see
    nothing -> the weight of key 9.  mask_b: an additive mask lets the row see these two only and adds this to the second's score."""
    S, row = 70, 66
    q, k, v = (torch.zeros(1, S, 1, d, dtype=torch.float16, device=DEV) for _ in range(3))
    q[0, row, 0, 0], q[0, row, 0, 1] = 32768.0, 181.0
    k[0, 3, 0, 0] = 32768.0
    if less is not None:
        k[0, 9, 0, 0], k[0, 9, 0, 1] = 32768.0, -float(less)
    v[0, 9] = 1.0
    begin = torch.full((1, S), S, dtype=torch.int32, device=DEV)
    begin[0, row] = 0
    mask = None
    if mask_b:
        mask = torch.full((S, S), -torch.finfo(torch.float32).max, device=DEV)
        mask[row, 3], mask[row, 9] = 0.0, mask_b
    kc, vc = (torch.zeros(1, 1, S, d, dtype=torch.float16, device=DEV) for _ in range(2))
    o = torch.empty(1, 1, S, d, device=DEV)
    scratch = torch.zeros(A.workspace_bytes(1, 1, S, S, size_per_head=d) + 65536, dtype=torch.uint8, device=DEV)
    p, f = A.make_scored_params(q=q, k=k, v=v, k_cache=kc, v_cache=vc, out=o, scratch=scratch, softcap=cap, softmax_scale=scale, key_begin=begin,
                                mask_mode=A.FLB_MASK_NONE if mask is None else A.FLB_MASK_GENERIC, attn_mask=mask,
                                alibi_slopes=torch.full((1,), 2.0 ** -20, device=DEV) if alibi else None)
    A.forward_scored(p, f)
    torch.cuda.synchronize()
    assert A.scratch_status(scratch) == 0
    assert float(o[0, 0, :row].abs().max()) == 0
    return float(o[0, 0, row, 5])


@pytest.mark.parametrize("alibi", [False, True])
@pytest.mark.parametrize("log_cap", [18, 20, 24, 25, 28, 30, 40])
def test_prefill_large_caps_keep_the_distance_of_large_scores(cuda_device, log_cap, alibi):
    """Raw scores of 2^30 and 181^2 less, 65536 and 2 less after the scale, below a quarter of the cap.  Tolerance: a score of 2^16.5 in units of log2 is rounded to 2^-8
    at each of five operations on either side and the fit's error changes the difference by less than 2^-10 of it, so the exponent is off by at most 0.03."""
    raw, scale, cap = 2.0 ** 30, 2.0 ** -14, 2.0 ** log_cap
    gap = cap * (math.tanh(raw * scale / cap) - math.tanh((raw - 181.0 ** 2) * scale / cap)) - (6 * 2.0 ** -20 if alibi else 0.0)
    got = two_keys(181, cap=cap, scale=scale, alibi=alibi)
    assert 0 < got < 1
    assert abs(math.log(got / (1 - got)) + gap) <= 0.03 + 2.0 ** -9, (got, gap)  # (weights are fp16)


@pytest.mark.parametrize("log_cap", [28, 30, 35, 40])
def test_prefill_large_capped_scores_against_a_mask(cuda_device, log_cap):
    """A raw score of 2^30 comes to 8.7e7 (or what the cap leaves of it), and loses to a mask that lifts the other key 4 % above it."""
    scale, cap = 0.08125, 2.0 ** log_cap
    x = cap * math.tanh(2.0 ** 30 * scale / cap)
    assert two_keys(None, cap=cap, scale=scale, mask_b=1.04 * x) == 1.0
    assert two_keys(None, cap=cap, scale=scale, mask_b=0.96 * x) == 0.0


@pytest.mark.parametrize("log_cap", [20, 28, 40])
def test_prefill_saturated_caps_share_the_weight(cuda_device, log_cap):
    """Two scores far beyond the cap are both the cap."""
    assert two_keys(0, cap=2.0 ** log_cap, scale=2.0 ** (log_cap - 26)) == pytest.approx(0.5, abs=2.0 ** -11)


# ------------------------------------------------------------------------------------------------ devices
@pytest.mark.parametrize("S", [1, 5])
def test_tensors_in_host_memory_are_refused(cuda_device, S):
    """Refused while the blocks are filled, so no kernel sees their addresses; a decode call may read pinned ones."""
    B, H, Hkv, T, d = 2, 8, 4, 64, 128
    good = dict(q=torch.zeros(B, S, H, d).half(), k=torch.zeros(B, S, Hkv, d).half(), v=torch.zeros(B, S, Hkv, d).half(), k_cache=torch.zeros(B, Hkv, T, d), v_cache=torch.zeros(B, Hkv, T, d),
                out=torch.zeros(B, H, S, d), scratch=torch.zeros(A.workspace_bytes(B, H, T, S) + 65536, dtype=torch.uint8), alibi_slopes=torch.zeros(H),
                key_begin=torch.zeros((B,) if S == 1 else (B, S), dtype=torch.int32), freq_cis=torch.zeros(T, d), out_q8=torch.zeros(B, S, H * d, dtype=torch.int8),
                out_q8_scale=torch.zeros(B * S))
    dev = {n: t.to(DEV) for n, t in good.items()}
    A.make_scored_params(**dev)
    for name, t in good.items():
        with pytest.raises(ValueError, match="another device"):
            A.make_scored_params(**{**dev, name: t})
        pinned = {**dev, name: t.pin_memory()}
        if S == 1 and name not in ("k_cache", "v_cache", "scratch"):
            A.make_scored_params(**pinned)
        else:
            with pytest.raises(ValueError, match="another device"):
                A.make_scored_params(**pinned)


def test_decode_reads_and_writes_pinned_memory(cuda_device):
    (q, k, v, kc, vc), o = run_decode(60, B=2, H=4, Hkv=2, T=256, d=128, past=[255, 17], cap=10.0, rope=False)
    host = {n: t.cpu().pin_memory() for n, t in (("q", q), ("k", k), ("v", v), ("out", torch.zeros_like(o)), ("past_lens", torch.tensor([255, 17], dtype=torch.int32)))}
    scratch = torch.zeros(A.workspace_bytes(2, 4, 256), dtype=torch.uint8, device=DEV)
    A.forward_scored(*A.make_scored_params(**host, k_cache=kc, v_cache=vc, scratch=scratch, max_past_len=255, softcap=10.0))
    torch.cuda.synchronize()
    assert torch.equal(host["out"], o.cpu())
