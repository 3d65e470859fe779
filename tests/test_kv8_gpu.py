"""The 8-bit cache on the GPU against the plain implementation in 64 bits (codes and scales bit for bit: their rule is defined
by IEEE fp32 operations)."""
import math

import numpy as np
import pytest
import torch

from fasterllama_b200 import attention as A
from fasterllama_b200 import kv8
from fasterllama_b200 import workloads as W

import forms_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
I8, E4 = torch.int8, torch.float8_e4m3fn


def gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def tokens(g, io, B, S, h, d, std=1.0):
    x = torch.randn(B, S, h, d, generator=g, device=DEV) * std
    if io == "int32":
        return (x * 4096).round().to(torch.int32), (torch.rand(h * d, generator=g, device=DEV) + 0.5) / 64
    return x.to(getattr(torch, io)), None


def table(rows, d):
    return torch.from_numpy(W.freq_cis_table(rows, d)).to(DEV)


def used_cache(g, B, H, T, d, block, dtype, row_pos=False):
    """A cache whose every byte is set: codes of live values, NaN patterns included nowhere a live row may be read from."""
    c = kv8.empty_cache(B, H, T, d, block_len=block, dtype=dtype, row_pos=row_pos, device=DEV)
    for t in (c.k, c.v):
        x = torch.randn(B, H, T, d, generator=g, device=DEV)
        t.copy_((x * 30).round().clamp(-127, 127).to(I8) if dtype == I8 else (x * 100).clamp(-448, 448).to(E4))
    for t in (c.k_scale, c.v_scale):
        t.copy_(torch.exp(torch.randn(t.shape, generator=g, device=DEV)) * (0.03 if dtype == I8 else 0.01))
    if row_pos:
        c.row_pos.copy_(torch.arange(T, dtype=torch.int32, device=DEV).expand(B, H, T))
    return c


def clone(c):
    return kv8.Cache(*(t.clone() for t in (c.k, c.v, c.k_scale, c.v_scale)), row_pos=None if c.row_pos is None else c.row_pos.clone())


def same(a, b):
    """Equal bits."""
    for n, t in a.tensors().items():
        u = b.tensors()[n]
        x, y = (z.view(torch.int8) if z.dtype == E4 else z.view(torch.int32) if z.dtype == torch.float32 else z for z in (t, u))
        if not torch.equal(x, y):
            bad = (x != y).nonzero()
            raise AssertionError(f"{n}: {len(bad)} differ, first at {bad[0].tolist()}: {t[tuple(bad[0])]} and {u[tuple(bad[0])]}")


def ref_append(c, k, v, past, counts, pos0, tab, act=None, kw=None, vw=None):
    """The plain append on a clone."""
    c = clone(c)
    B, S = k.shape[:2]
    pos = torch.tensor(pos0, device=DEV)[:, None] + torch.arange(S, device=DEV)
    kr = R.rotate(R.values(k, act, kw), tab, pos.clamp_max(tab.shape[0] - 1) if tab is not None else pos)
    vr = R.values(v, act, vw)
    for b in range(B):
        n = counts[b]
        if n == 0:
            continue
        rows = list(range(past[b], past[b] + n))
        for h in range(c.k.shape[1]):
            R.put_rows(c.k[b, h], c.k_scale[b, h], kr[b, :n, h], rows, past[b], past[b], c.block_len)
            R.put_rows(c.v[b, h], c.v_scale[b, h], vr[b, :n, h], rows, past[b], past[b], c.block_len)
            if c.row_pos is not None:
                c.row_pos[b, h, past[b]:past[b] + n] = pos[b, :n].to(torch.int32)
    return c


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


# ------------------------------------------------------------------------------------------------ append
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("block", [16, 32, 64, 128])
@pytest.mark.parametrize("dtype,io,S,past,counts", [
    (I8, "float16", 70, [0, 3, 127], None), (E4, "int32", 33, [0, 15, 16], [33, 0, 7]), (I8, "float32", 1, [0, 31, 64], None),
    (E4, "float16", 129, [0, 1, 100], [129, 128, 1]), (I8, "int32", 16, [16, 128, 5], [0, 16, 11])])
def test_append(cuda_device, d, block, dtype, io, S, past, counts):
    g = gen(S + d + block)
    B, H, T = 3, 2, 384
    c = used_cache(g, B, H, T, d, block, dtype, row_pos=(S % 2 == 1))
    k, kw = tokens(g, io, B, S, H, d)
    v, vw = tokens(g, io, B, S, H, d)
    act = (torch.rand(B * S, generator=g, device=DEV) + 0.5) / 64 if io == "int32" else None
    tab = table(T, d)
    want = ref_append(c, k, v, past, counts or [S] * B, past, tab, act, kw, vw)
    st = torch.zeros(4, dtype=torch.int32, device=DEV)
    kv8.append(c, k, v, past_lens=i32(past), new_lens=None if counts is None else i32(counts), act_scale=act, k_w_scale=kw, v_w_scale=vw, freq_cis=tab, scratch=st)
    torch.cuda.synchronize()
    assert int(st[0]) == 0
    same(c, want)


def test_append_uniform_start_positions_and_no_rotation(cuda_device):
    g = gen(1)
    c = used_cache(g, 2, 3, 128, 64, 32, I8, row_pos=True)
    k, _ = tokens(g, "float16", 2, 5, 3, 64)
    v, _ = tokens(g, "float16", 2, 5, 3, 64)
    want = ref_append(c, k, v, [30, 30], [5, 5], [1000, 7], None)
    kv8.append(c, k, v, start_pos=30, token_pos=i32([1000, 7]))
    same(c, want)


def test_append_strided_rows(cuda_device):
    """k and v as columns of one merged projection."""
    g = gen(2)
    B, S, H, d = 2, 9, 4, 128
    buf = torch.randn(B, S, 3 * H * d, generator=g, device=DEV).half()
    k, v = (buf[:, :, i * H * d:(i + 1) * H * d].unflatten(2, (H, d)) for i in (1, 2))
    a = used_cache(g, B, H, 64, d, 16, E4)
    b = clone(a)
    kv8.append(a, k, v, start_pos=3)
    kv8.append(b, k.contiguous(), v.contiguous(), start_pos=3)
    same(a, b)


def test_append_in_steps_grows_scales_and_recodes(cuda_device):
    """Token by token with rising magnitude: the block's scale grows at each, the held codes follow each time."""
    g = gen(3)
    d, block = 128, 16
    for dtype in (I8, E4):
        c = kv8.empty_cache(1, 2, 48, d, block_len=block, dtype=dtype, device=DEV)
        want = clone(c)
        for r in range(40):
            k = (torch.randn(1, 1, 2, d, generator=g, device=DEV) * (1.3 ** (r % 17))).half()
            v = (torch.randn(1, 1, 2, d, generator=g, device=DEV) * (0.7 ** (r % 17))).half()
            want = ref_append(want, k, v, [r], [1], [r], None)
            kv8.append(c, k, v, start_pos=r)
        same(c, want)


def test_append_zero_rows_denormals_and_values_that_are_not_finite(cuda_device):
    d = 64
    c = kv8.empty_cache(1, 4, 32, d, block_len=16, device=DEV)
    k = torch.zeros(1, 2, 4, d, device=DEV)
    v = torch.zeros(1, 2, 4, d, device=DEV)
    v[0, :, 0] = 1e-40           # a subnormal block: its scale is subnormal too
    v[0, 1, 1, 5] = math.inf
    v[0, 0, 2, 7] = math.nan
    v[0, 0, 3, 1] = 65504.0
    kv8.append(c, k, v)
    _, out = c.dequantize()
    assert float(c.k_scale[0, :, 0].abs().max()) == 0 and int(c.k.abs().max()) == 0
    want = ref_append(kv8.empty_cache(1, 4, 32, d, block_len=16, device=DEV), k, v, [0], [2], [0], None)
    assert torch.equal(c.v[0, 0], want.v[0, 0]) and torch.equal(c.v_scale[0, 0], want.v_scale[0, 0])
    assert math.isinf(float(c.v_scale[0, 1, 0])) and math.isnan(float(c.v_scale[0, 2, 0]))
    assert out[0, 1, :2].isnan().all() and out[0, 2, :2].isnan().all()  # never silently a number
    assert float(out[0, 3, 0, 1]) == pytest.approx(65504.0, rel=1e-6)
    # a later finite token does not make the block finite again; the next block is its own
    kv8.append(c, torch.ones(1, 15, 4, d, device=DEV), torch.ones(1, 15, 4, d, device=DEV), start_pos=2)
    assert math.isnan(float(c.v_scale[0, 2, 0])) and float(c.v_scale[0, 2, 1]) == pytest.approx(1 / 127, rel=1e-6)


@pytest.mark.parametrize("dtype", [I8, E4])
def test_subnormal_rows_keep_their_signs(cuda_device, dtype):
    """A scale of a few units of the smallest subnormal number is rounded coarsely: quotients pass the largest code and are held to it."""
    d, tiny = 64, 2.0 ** -149
    for top in (1, 63, 64, 127, 128, 190, 191, 500, 671, 672, 5000):
        x = torch.linspace(-1, 1, d, dtype=torch.float64, device=DEV).mul(top).round().mul(tiny).float().expand(1, 3, 1, d).contiguous()
        c = kv8.empty_cache(1, 1, 32, d, block_len=16, dtype=dtype, device=DEV)
        want = ref_append(c, x, x, [0], [3], [0], None)
        kv8.append(c, x, x)
        same(c, want)
        one = kv8.empty_cache(1, 1, 32, d, block_len=16, dtype=dtype, device=DEV)
        s = torch.zeros(kv8.decode_workspace_bytes(1, 1, 1, 32, d, block_len=16), dtype=torch.uint8, device=DEV)
        for r in range(3):
            kv8.decode(one, x[:, :1], x[:, :1], x[:, :1], torch.empty(1, 1, 1, d, device=DEV), start_pos=r, scratch=s)
        same(one, want)


def test_append_bad_lengths_are_flagged_and_touch_nothing(cuda_device):
    g = gen(4)
    c = used_cache(g, 5, 1, 64, 64, 32, I8, row_pos=True)
    before = clone(c)
    k, _ = tokens(g, "float16", 5, 8, 1, 64)
    st = torch.zeros(4, dtype=torch.int32, device=DEV)
    kv8.append(c, k, k, past_lens=i32([-1, 57, 64, 10, 2147483647]), new_lens=i32([8, 8, 8, 9, 8]), scratch=st)
    torch.cuda.synchronize()
    assert int(st[0]) == kv8.STATUS_BAD_LEN
    same(c, before)
    st.zero_()
    kv8.append(c, k, k, start_pos=0, token_pos=i32([0, 0, 60, 0, -3]), freq_cis=table(64, 64), scratch=st)
    torch.cuda.synchronize()
    assert int(st[0]) == kv8.STATUS_BAD_POS


# ------------------------------------------------------------------------------------------------ decode
def run_decode(seed, *, B, Hq, Hkv, T, d, block, dtype, io="float16", out="float32", past, cap=0.0, alibi=False, begin=None, weights=None, shuffled=False,
               token_pos=None, split=0, rope=True, std=1.5, zeroed=True):
    g = gen(seed)
    c = used_cache(g, B, Hkv, T, d, block, dtype, row_pos=shuffled)
    if shuffled:
        for b in range(B):
            for h in range(Hkv):
                n = past[b]
                c.row_pos[b, h, :n] = torch.randperm(2 * n + 1, generator=g, device=DEV)[:n].to(torch.int32)
    # behind the sequences: codes that read as NaN in e4m3, and scales that are NaN
    for b in range(B):
        for t in (c.k, c.v):
            t.view(I8)[b, :, past[b]:] = 127
        first = -(-past[b] // block)
        for t in (c.k_scale, c.v_scale):
            t[b, :, first:] = math.nan
    pos = token_pos or past
    q, qw = tokens(g, io, B, 1, Hq, d, std)
    k, kw = tokens(g, io, B, 1, Hkv, d)
    v, vw = tokens(g, io, B, 1, Hkv, d)
    act = (torch.rand(B, generator=g, device=DEV) + 0.5) / 64 if io == "int32" else None
    tab = table(max(2 * T + 2, 8), d) if rope else None
    slopes = torch.pow(2.0, -8.0 * torch.arange(1, Hq + 1, device=DEV) / Hq) if alibi else None
    w_in = torch.rand(B, Hkv, T, generator=g, device=DEV) if weights else None
    w_out = w_in if weights == "in place" else torch.full((B, Hkv, T), 9.0, device=DEV) if weights else None
    w_was = None if w_in is None else w_in.clone()
    after = ref_append(c, k, v, past, [1] * B, pos, tab, act, kw, vw)
    o = torch.full((B, Hq, 1, d), math.nan, dtype=getattr(torch, out), device=DEV)
    scratch = torch.zeros(kv8.decode_workspace_bytes(B, Hq, Hkv, T, d, block_len=block, weights=bool(weights), split_len=split), dtype=torch.uint8, device=DEV)
    if not zeroed:
        scratch.fill_(0xA5)
    args = dict(past_lens=i32(past), max_past_len=max(past), act_scale=act, q_w_scale=qw, k_w_scale=kw, v_w_scale=vw, freq_cis=tab, softcap=cap, alibi_slopes=slopes,
                key_begin=None if begin is None else i32(begin), weight_in=w_in, weight_out=w_out, token_pos=None if token_pos is None else i32(token_pos),
                scratch=scratch, scratch_zeroed=zeroed, split_len=split)
    kv8.decode(c, q, k, v, o, **args)
    torch.cuda.synchronize()
    assert A.scratch_status(scratch) == 0
    same(c, after)
    check_decode(after, R.rotate(R.values(q, act, qw), tab, torch.tensor(pos, device=DEV)[:, None]), o, past, pos, cap, slopes, begin, w_was, w_out)
    return c, (q, k, v, o), args


def check_decode(c, qr, o, past, pos, cap, slopes, begin, w_was, w_out):
    """Against 64 bits.  Tolerance of a score (natural units): q reaches the products in two fp16 parts, off by at most 2^-22 of each
    element's row maximum; products are exact, their fp32 sum over d dims off by at most (d / 16 + 8) 2^-23 of the sum of magnitudes (the
    matrix instruction adds 16 products at a time, and may cut instead of round), a few more roundings of the finished score: 2^-21 of its size, 2^-20 of the cap
    for tanhf (2 ulp).  A weight is off by that relatively, the result by it times the largest |v| on both sides of the fraction; sums
    over n rows in four warps of 16-row steps add (n / 64 + 64) 2^-22; p in two fp16 parts 2^-21 of the largest."""
    B, Hq, _, d = o.shape
    Hkv, block = c.k.shape[1], c.block_len
    G, scale = Hq // Hkv, 1.0 / math.sqrt(d)
    for b in range(B):
        n = past[b] + 1
        rows = torch.arange(n, device=DEV)
        for h in range(Hkv):
            kd, vd = R.dequant(c.k[b, h, :-(-n // block) * block], c.k_scale[b, h, :-(-n // block)], block)[:n], \
                R.dequant(c.v[b, h, :-(-n // block) * block], c.v_scale[b, h, :-(-n // block)], block)[:n]
            rp = rows if c.row_pos is None else c.row_pos[b, h, :n].long()
            see = torch.ones(1, n, dtype=torch.bool, device=DEV) if begin is None else (rp >= begin[b])[None]
            total = torch.zeros(n, dtype=torch.float64, device=DEV)
            werr = 0.0
            for j in range(G):
                hq = h * G + j
                q = qr[b, 0, hq].double()
                dist = (pos[b] - rp).abs().double()
                bias = -slopes[hq].double() * dist if slopes is not None else None
                want, p = R.attend(q[None], kd, vd, see, scale, cap=cap, bias=None if bias is None else bias[None])
                if not see.any():
                    assert float(o[b, hq].float().abs().max()) == 0
                    continue
                mag = float((kd.abs() @ q.abs()).max()) * scale
                qmax = float(q.abs().max()) * float(kd.abs().sum(1).max()) * scale
                size = mag + (cap or 0.0) + (float(bias[see[0]].abs().max()) if bias is not None else 0.0)
                ds = qmax * 2.0 ** -22 + mag * (d / 16 + 8) * 2.0 ** -23 + size * 2.0 ** -20
                vmax = float(vd[see[0]].abs().max())
                tol = vmax * (2 * ds + (n / 64 + 64) * 2.0 ** -22)
                rnd = torch.finfo(o.dtype).eps / 2
                err = (o[b, hq].double() - want).abs()
                assert bool((err <= tol + rnd * want.abs() + 2.0 ** -24).all()), (b, hq, float(err.max()), tol)
                total += p[0]
                werr += (ds * 2 + (n / 64 + 64) * 2.0 ** -22)
            if w_out is not None:
                base = w_was[b, h, :n].double().clone()
                base[n - 1] = 0
                got = w_out[b, h, :n].double()
                assert bool(((got - base - total).abs() <= werr * total + 2.0 ** -22 * (base + total) + 1e-30).all())


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("G", [1, 2, 4, 5, 8, 9, 16])
@pytest.mark.parametrize("dtype", [I8, E4])
def test_decode_heads(cuda_device, d, G, dtype):
    """Every split of the q heads over column tiles and CTAs, lengths around the 16-row steps, 128-row splits and blocks."""
    run_decode(10 * G + d, B=5, Hq=2 * G, Hkv=2, T=384, d=d, block=16 if G % 2 else 64, dtype=dtype, past=[0, 1, 127, 128, 383], split=128)


@pytest.mark.parametrize("past", [[0], [14], [15], [16], [63], [64], [65], [255], [256], [700]])
@pytest.mark.parametrize("block", [16, 32, 64, 128])
def test_decode_lengths(cuda_device, past, block):
    run_decode(past[0] + block, B=1, Hq=4, Hkv=2, T=768, d=128, block=block, dtype=I8, past=past, io="int32", weights="apart")


@pytest.mark.parametrize("form", ["cap", "alibi", "begin", "all", "nothing seen", "shuffled", "positions"])
@pytest.mark.parametrize("dtype,d,G", [(I8, 128, 1), (E4, 128, 8), (I8, 64, 3), (E4, 256, 4)])
def test_decode_forms(cuda_device, form, dtype, d, G):
    past = [300, 17, 0, 511]
    kw = {"cap": dict(cap=10.0, std=6.0), "alibi": dict(alibi=True), "begin": dict(begin=[0, 17, 0, 300]), "all": dict(cap=30.0, alibi=True, begin=[290, 3, -5, 511]),
          "nothing seen": dict(begin=[301, 18, 2147483647, 600]), "shuffled": dict(shuffled=True, alibi=True, begin=[200, 9, 0, 1000], cap=20.0),
          "positions": dict(token_pos=[900, 17, 5, 1023], alibi=True)}[form]
    if form == "shuffled":
        kw["token_pos"] = [601, 40, 1, 1023]
    run_decode(5, B=4, Hq=2 * G, Hkv=2, T=512, d=d, block=32, dtype=dtype, past=past, weights="in place", split=128, **kw)


@pytest.mark.parametrize("io", ["float16", "float32", "int32"])
@pytest.mark.parametrize("out", ["float16", "float32"])
@pytest.mark.parametrize("rope", [True, False])
def test_decode_types_and_a_scratch_that_is_not_zeroed(cuda_device, io, out, rope):
    run_decode(6, B=3, Hq=4, Hkv=4, T=256, d=128, block=64, dtype=I8, io=io, out=out, past=[255, 130, 7], rope=rope, zeroed=False)


def test_decode_default_splits_of_long_slabs(cuda_device):
    run_decode(7, B=1, Hq=8, Hkv=2, T=16384, d=128, block=128, dtype=I8, past=[16383], weights="apart", cap=50.0)
    run_decode(8, B=2, Hq=4, Hkv=1, T=4096, d=64, block=16, dtype=E4, past=[4095, 2000])


def test_decode_very_large_and_very_small_values(cuda_device):
    """Powers of two are moved out of q and the scales before fp16 sees them: results are relative to the values."""
    for up in (2.0 ** -60, 2.0 ** 40, 2.0 ** 112):
        g = gen(9)
        B, H, T, d, block, past = 1, 2, 128, 128, 32, [100]
        c = used_cache(g, B, H, T, d, block, I8)
        small = clone(c)
        c.v_scale.mul_(up)
        q, _ = tokens(g, "float32", B, 1, H, d)
        k, _ = tokens(g, "float32", B, 1, H, d)
        v, _ = tokens(g, "float32", B, 1, H, d)
        outs = []
        for cache, qq, vv, sc in ((small, q, v, 0.1), (c, q * up, v * up, 0.1 / up)):
            o = torch.empty(B, H, 1, d, device=DEV)
            s = torch.zeros(kv8.decode_workspace_bytes(B, H, H, T, d, block_len=block), dtype=torch.uint8, device=DEV)
            kv8.decode(cache, qq, k, vv, o, past_lens=i32(past), softmax_scale=sc, scratch=s)
            outs.append(o)
        assert torch.equal(outs[0] * up, outs[1])


@pytest.mark.parametrize("dtype,d,G", [(I8, 128, 1), (E4, 64, 4), (I8, 256, 2), (E4, 128, 8), (I8, 128, 9)])
@pytest.mark.parametrize("what", [math.nan, math.inf, 1e37])
@pytest.mark.parametrize("positions", [False, True])
def test_decode_rows_before_key_begin_may_hold_anything(cuda_device, dtype, d, G, what, positions):
    """The block in front of key_begin reads as infinity, NaN or a huge number: results are those of a clean cache."""
    g = gen(17)
    T, block, n = 512, 16, 300
    c = used_cache(g, 1, 2, T, d, block, dtype, row_pos=positions)
    bad = clone(c)
    for t in (bad.k_scale, bad.v_scale):
        t[:, :, 0] = what
        t[:, :, 2] = what
    q, _ = tokens(g, "float16", 1, 1, 2 * G, d)
    k, _ = tokens(g, "float16", 1, 1, 2, d)
    w = torch.zeros(1, 2, T, device=DEV)
    outs = []
    for cache in (c, bad):
        o, wo = torch.empty(1, 2 * G, 1, d, device=DEV), torch.zeros_like(w)
        s = torch.zeros(kv8.decode_workspace_bytes(1, 2 * G, 2, T, d, block_len=block, weights=True, split_len=128), dtype=torch.uint8, device=DEV)
        kv8.decode(cache, q, k, k, o, past_lens=i32([n]), key_begin=i32([51]), weight_in=w, weight_out=wo, scratch=s, split_len=128)
        outs.append((o, wo))
    assert bool(outs[0][0].isfinite().all())
    assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1])


def test_decode_is_deterministic_and_independent_of_the_batch(cuda_device):
    c, (q, k, v, o), args = run_decode(11, B=4, Hq=8, Hkv=2, T=1024, d=128, block=64, dtype=I8, past=[1000, 513, 128, 40])
    again = torch.empty_like(o)
    kv8.decode(c, q, k, v, again, **args)
    assert torch.equal(o, again)
    one = kv8.Cache(c.k[1:2].contiguous(), c.v[1:2].contiguous(), c.k_scale[1:2].contiguous(), c.v_scale[1:2].contiguous())
    alone = torch.empty_like(o[1:2])
    kv8.decode(one, q[1:2], k[1:2], v[1:2], alone, **{**args, "past_lens": args["past_lens"][1:2], "max_past_len": 513})
    assert torch.equal(o[1:2], alone)


def test_decode_bad_length_is_flagged_and_gives_zeros(cuda_device):
    g = gen(12)
    c = used_cache(g, 3, 2, 64, 64, 16, I8)
    before = clone(c)
    q, _ = tokens(g, "float16", 3, 1, 2, 64)
    o = torch.full((3, 2, 1, 64), math.nan, device=DEV)
    s = torch.zeros(kv8.decode_workspace_bytes(3, 2, 2, 64, 64, block_len=16), dtype=torch.uint8, device=DEV)
    kv8.decode(c, q, q, q, o, past_lens=i32([64, -1, 2147483647]), scratch=s)
    torch.cuda.synchronize()
    assert A.scratch_status(s) == kv8.STATUS_BAD_LEN
    assert float(o.abs().max()) == 0
    same(c, before)


@pytest.mark.parametrize("Hq", [2, 20])
def test_decode_length_one_above_the_promised_bound(cuda_device, Hq):
    """Flagged too where the bound is no whole number of splits."""
    g = gen(18)
    c = used_cache(g, 2, 2, 512, 64, 16, I8)
    before = clone(c)
    q, _ = tokens(g, "float16", 2, 1, Hq, 64)
    k, _ = tokens(g, "float16", 2, 1, 2, 64)
    o = torch.full((2, Hq, 1, 64), math.nan, device=DEV)
    w, wo = torch.ones(2, 2, 512, device=DEV), torch.full((2, 2, 512), 7.0, device=DEV)
    s = torch.zeros(kv8.decode_workspace_bytes(2, Hq, 2, 512, 64, block_len=16, weights=True), dtype=torch.uint8, device=DEV)
    kv8.decode(c, q, k, k, o, past_lens=i32([121, 120]), max_past_len=120, weight_in=w, weight_out=wo, scratch=s)
    torch.cuda.synchronize()
    assert A.scratch_status(s) == kv8.STATUS_BAD_LEN
    assert float(o[0].abs().max()) == 0 and bool(o[1].isfinite().all())
    assert torch.equal(c.k[0], before.k[0]) and not torch.equal(c.k[1], before.k[1])
    assert bool((wo[0] == 7).all()) and bool((wo[1, :, 121:] == 7).all()) and not bool((wo[1, :, :121] == 7).any())


@pytest.mark.parametrize("Hq", [2, 20])  # the attention kernel stores the token itself, or a launch in front does
def test_decode_length_above_the_promised_bound(cuda_device, Hq):
    g = gen(15)
    c = used_cache(g, 2, 2, 512, 64, 16, I8)
    before = clone(c)
    q, _ = tokens(g, "float16", 2, 1, Hq, 64)
    k, _ = tokens(g, "float16", 2, 1, 2, 64)
    o = torch.full((2, Hq, 1, 64), math.nan, device=DEV)
    s = torch.zeros(kv8.decode_workspace_bytes(2, Hq, 2, 512, 64, block_len=16), dtype=torch.uint8, device=DEV)
    kv8.decode(c, q, k, k, o, past_lens=i32([400, 100]), max_past_len=120, scratch=s)
    torch.cuda.synchronize()
    assert A.scratch_status(s) == kv8.STATUS_BAD_LEN
    assert float(o[0].abs().max()) == 0 and bool(o[1].isfinite().all())
    assert torch.equal(c.k[0], before.k[0]) and torch.equal(c.v_scale[0], before.v_scale[0]) and not torch.equal(c.k[1], before.k[1])


def test_decode_q_that_is_not_finite_reaches_its_own_rows_only(cuda_device):
    for dtype in (I8, E4):
        g = gen(16)
        c = used_cache(g, 1, 2, 256, 128, 32, dtype)
        q, _ = tokens(g, "float32", 1, 1, 8, 128)
        k, _ = tokens(g, "float32", 1, 1, 2, 128)
        s = torch.zeros(kv8.decode_workspace_bytes(1, 8, 2, 256, 128, block_len=32), dtype=torch.uint8, device=DEV)
        a, b = torch.empty(1, 8, 1, 128, device=DEV), torch.empty(1, 8, 1, 128, device=DEV)
        kv8.decode(c, q, k, k, a, past_lens=i32([200]), scratch=s)
        q[0, 0, 2, 7], q[0, 0, 5, 100] = math.nan, math.inf
        kv8.decode(c, q, k, k, b, past_lens=i32([200]), scratch=s)
        bad = [2, 5]
        assert bool(b[0, bad].isnan().all())
        rest = [h for h in range(8) if h not in bad]
        assert torch.equal(a[0, rest], b[0, rest])


def test_decode_on_another_stream_and_in_a_replayed_graph(cuda_device):
    g = gen(13)
    B, H, T, d = 2, 4, 512, 128
    c = used_cache(g, B, H, T, d, 64, I8, row_pos=True)
    start = clone(c)
    q, _ = tokens(g, "float16", B, 1, 2 * H, d)
    k, _ = tokens(g, "float16", B, 1, H, d)
    v, _ = tokens(g, "float16", B, 1, H, d)
    past = i32([300, 140])
    w = torch.zeros(B, H, T, device=DEV)
    o = torch.empty(B, 2 * H, 1, d, device=DEV)
    s = torch.zeros(kv8.decode_workspace_bytes(B, 2 * H, H, T, d, weights=True), dtype=torch.uint8, device=DEV)

    def step(cache, out, weight, stream=None):
        kv8.decode(cache, q, k, v, out, past_lens=past, weight_in=weight, weight_out=weight, scratch=s, scratch_zeroed=True, stream=stream)

    # eager: three steps, the lengths grown on the device in between
    for _ in range(3):
        step(c, o, w)
        past.add_(1)
    want, ww, cc = o.clone(), w.clone(), clone(c)
    side = torch.cuda.Stream()
    past.sub_(3)
    w.zero_()
    for n, t in c.tensors().items():
        t.copy_(start.tensors()[n])
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            step(c, o, w)
            past.add_(1)
        for _ in range(3):
            graph.replay()
    side.synchronize()
    assert torch.equal(o, want) and torch.equal(w, ww)
    same(c, cc)


def test_codes_behind_2_31_bytes(cuda_device):
    """The last sequence of a cache whose codes and scores lie behind 2^31 bytes."""
    g = gen(14)
    B, H, T, d, block = 9, 1, 1 << 20, 256, 128
    c = kv8.empty_cache(B, H, T, d, block_len=block, device=DEV)
    small = used_cache(g, 1, H, 1024, d, block, I8)
    for n in ("k", "v", "k_scale", "v_scale"):
        t = getattr(small, n)
        getattr(c, n)[B - 1, :, :t.shape[2]] = t[0]
    q, _ = tokens(g, "float16", B, 1, 4, d)
    k, _ = tokens(g, "float16", B, 1, H, d)
    v, _ = tokens(g, "float16", B, 1, H, d)
    past = [0] * (B - 1) + [1000]
    o = torch.empty(B, 4, 1, d, device=DEV)
    s = torch.zeros(kv8.decode_workspace_bytes(B, 4, H, T, d, block_len=block, split_len=128), dtype=torch.uint8, device=DEV)
    kv8.decode(c, q, k, v, o, past_lens=i32(past), max_past_len=1000, scratch=s, split_len=128)
    o1 = torch.empty(1, 4, 1, d, device=DEV)
    kv8.decode(small, q[B - 1:], k[B - 1:], v[B - 1:], o1, past_lens=i32([1000]), scratch=s, split_len=128)
    assert torch.equal(o[B - 1:], o1)
    assert torch.equal(c.k[B - 1, :, :1024], small.k[0])


# ------------------------------------------------------------------------------------------------ evict
def ref_evict(c, weight, lens, budget, recent, sinks, nxt, w_out, p_out):
    c, w_out, p_out, out = clone(c), w_out.clone(), p_out.clone(), []
    pos = c.row_pos.cpu().numpy()
    w = weight.cpu().numpy()
    for b, n in enumerate(lens):
        m = min(n, budget)
        out.append(m)
        for h in range(c.k.shape[1]):
            _, holes, src = R.evict_plan(w[b, h], pos[b, h], n, budget, recent, sinks, None if nxt is None else nxt[b])
            new_w, new_p = weight[b, h, :m].clone(), c.row_pos[b, h, :m].clone()
            if len(holes):
                ht, stt = torch.from_numpy(holes).to(DEV), torch.from_numpy(src).to(DEV)
                new_w[ht], new_p[ht] = weight[b, h][stt], c.row_pos[b, h][stt]
                for codes, scale in ((c.k, c.k_scale), (c.v, c.v_scale)):
                    x = codes[b, h][stt].float() * scale[b, h][stt // c.block_len][:, None]
                    R.put_rows(codes[b, h], scale[b, h], x, holes, m, 1 << 30, c.block_len)
            w_out[b, h, :m], p_out[b, h, :m] = new_w, new_p
    return c, w_out, p_out, out


def run_evict(seed, *, lens, T, budget, recent=0, sinks=0, H=2, d=64, block=16, dtype=I8, in_place=False, weight=None, pos=None, nxt="default"):
    g = gen(seed)
    B = len(lens)
    c = used_cache(g, B, H, T, d, block, dtype, row_pos=True)
    if pos is not None:
        c.row_pos.copy_(pos)
    w = weight if weight is not None else torch.exp(2 * torch.randn(B, H, T, generator=g, device=DEV))
    nx = [n for n in lens] if nxt == "default" else nxt
    w_out = w if in_place else torch.full_like(w, -7.0)
    p_out = c.row_pos if in_place else torch.full_like(c.row_pos, -7)
    want = ref_evict(c, w, lens, budget, recent, sinks, nx, w_out, p_out)
    lt = i32(lens)
    len_out = lt if in_place else i32([-1] * B)
    s = torch.full((kv8.evict_workspace_bytes(B, H, T, d, block_len=block),), 0xA5, dtype=torch.uint8, device=DEV)
    kv8.evict(c, past_lens=lt, len_out=len_out, budget=budget, recent=recent, sinks=sinks, next_pos=None if nx is None else i32(nx), weight=w,
              weight_out=None if in_place else w_out, pos_out=None if in_place else p_out, scratch=s)
    torch.cuda.synchronize()
    assert A.scratch_status(s) == 0
    wc, ww, wp, wl = want
    if in_place:
        wc.row_pos.copy_(wp)
    assert len_out.tolist() == wl
    assert torch.equal(w_out.view(torch.int32), ww.view(torch.int32)) and torch.equal(p_out, wp)
    same(c, wc)
    return c, w_out, p_out


@pytest.mark.parametrize("d,block,dtype", [(64, 16, I8), (128, 64, I8), (256, 32, E4), (128, 128, E4), (64, 128, I8)])
@pytest.mark.parametrize("lens,budget,recent,sinks", [
    ([384, 200, 130, 0], 128, 16, 4), ([384, 383, 1, 2], 1, 0, 0), ([384, 100, 99, 98], 99, 99, 0), ([384, 300, 250, 17], 250, 0, 250), ([384, 370, 360, 350], 384, 8, 8),
    ([384, 200, 201, 7], 200, 0, 0)])
def test_evict(cuda_device, d, block, dtype, lens, budget, recent, sinks):
    run_evict(budget + d, lens=lens, T=384, budget=budget, recent=recent, sinks=sinks, d=d, block=block, dtype=dtype, in_place=(budget % 2 == 0))


def test_evict_ties_zeros_nan_infinities_and_signs(cuda_device):
    g = gen(20)
    T = 512
    w = torch.randint(0, 3, (2, 2, T), generator=g, device=DEV).float()      # long runs of equal weights
    run_evict(21, lens=[512, 301], T=T, budget=200, recent=5, sinks=1, weight=w.clone())
    run_evict(22, lens=[512, 301], T=T, budget=100, weight=torch.zeros(2, 2, T, device=DEV), nxt=None)
    w = torch.randn(2, 2, T, generator=g, device=DEV)                         # negative ones, -0 and 0, all the special values
    w[:, :, ::7], w[:, :, 1::11], w[:, :, 2::13], w[:, :, 3::17], w[:, :, 4::19] = math.nan, math.inf, -math.inf, 0.0, -0.0
    for budget in (10, 60, 150, 290):
        run_evict(23, lens=[512, 301], T=T, budget=budget, recent=3, sinks=2, weight=w.clone())


def test_evict_positions_out_of_order_and_given_twice(cuda_device):
    g = gen(24)
    T = 256
    pos = torch.stack([torch.randperm(2 * T, generator=g, device=DEV)[:T] for _ in range(4)]).view(2, 2, T).to(torch.int32)
    run_evict(25, lens=[256, 200], T=T, budget=64, recent=40, sinks=10, pos=pos, nxt=[512, 500])
    # more protected rows than room: the selection is among them
    run_evict(26, lens=[256, 200], T=T, budget=30, recent=20, sinks=5, pos=torch.zeros(2, 2, T, dtype=torch.int32, device=DEV) + 3, nxt=[10, 10])
    run_evict(27, lens=[256, 200], T=T, budget=30, recent=20, sinks=5, pos=pos, nxt=[-2147483648, 2147483647])


def test_evict_long_slabs(cuda_device):
    """Several passes of the selecting block over the rows, more blocks than a block has threads."""
    run_evict(28, lens=[20000], T=20000 // 16 * 16 + 16, budget=7001, recent=100, sinks=4, d=64, block=16)
    run_evict(29, lens=[40001], T=40064, budget=40000, recent=100, sinks=4, d=64, block=32, H=1)


@pytest.mark.parametrize("T", [4096, 16384, 81920])  # a CTA, a cluster with 8 and one with 16 rows per thread
@pytest.mark.parametrize("kind", ["random", "few values", "near", "zeros", "special", "protected"])
def test_evict_selections(cuda_device, T, kind):
    """Few and many weights that share their leading digit with the one looked for, all equal, all protected."""
    g = gen(T + len(kind))
    n, B = T - 7, 1
    w = torch.rand(B, 1, T, generator=g, device=DEV)
    more = dict(recent=50, sinks=4)
    if kind == "few values":
        w = torch.randint(0, 3, (B, 1, T), generator=g, device=DEV).float()
    elif kind == "near":  # one leading digit, all different and some not
        w = 1 + torch.randint(0, T // 2, (B, 1, T), generator=g, device=DEV).float() * 2.0 ** -20
    elif kind == "zeros":
        w.zero_()
    elif kind == "special":
        w[:, :, ::3], w[:, :, 1::3] = math.nan, math.inf
    pos = None
    if kind == "protected":
        pos = torch.arange(T, dtype=torch.int32, device=DEV).flip(0).expand(B, 1, T) // 4
        more = dict(recent=100, sinks=40)
    for budget in (150, T // 3, n - 1):
        run_evict(45, lens=[n], T=T, budget=budget, H=1, weight=w.clone(), pos=pos, nxt=[T // 4] if kind == "protected" else [n], **more)


def test_evict_slabs_beyond_the_registers(cuda_device):
    """More rows than a cluster's threads keep in registers: the keys are read again at every pass."""
    run_evict(31, lens=[150001], T=150016, budget=3000, recent=100, sinks=4, d=64, block=16, H=1)
    w = torch.randint(0, 5, (2, 1, 140000), generator=gen(32), device=DEV).float()
    run_evict(33, lens=[140000, 2500], T=140000, budget=2000, recent=10, sinks=0, d=64, block=32, H=1, weight=w, in_place=True)


def test_evict_bad_length_is_flagged_and_left_alone(cuda_device):
    g = gen(30)
    c = used_cache(g, 3, 1, 64, 64, 16, I8, row_pos=True)
    before = clone(c)
    w = torch.rand(3, 1, 64, generator=g, device=DEV)
    w0, out = w.clone(), i32([0, 0, 0])
    s = torch.zeros(kv8.evict_workspace_bytes(3, 1, 64, 64, block_len=16), dtype=torch.uint8, device=DEV)
    kv8.evict(c, past_lens=i32([65, -1, 64]), len_out=out, budget=64, weight=w, scratch=s)
    torch.cuda.synchronize()
    assert A.scratch_status(s) == kv8.STATUS_BAD_LEN
    assert out.tolist() == [65, -1, 64] and torch.equal(w, w0)
    same(c, before)


# ------------------------------------------------------------------------------------------------ as a server uses them
def test_prompt_decode_evict_decode(cuda_device):
    """A capped prefill, its rows into the 8-bit cache, decode steps that accumulate weights, an eviction, more steps: every step against
    64 bits on the cache as it stands."""
    g = gen(40)
    B, Hq, Hkv, S, T, d, block = 2, 8, 4, 150, 256, 128, 32
    tab = table(T, d)
    cap = 20.0
    n = [150, 97]
    q, _ = tokens(g, "float16", B, S, Hq, d)
    k, _ = tokens(g, "float16", B, S, Hkv, d)
    v, _ = tokens(g, "float16", B, S, Hkv, d)
    slab = [torch.zeros(B, Hkv, S, d, dtype=torch.float16, device=DEV) for _ in range(2)]
    out = torch.empty(B, Hq, S, d, dtype=torch.float16, device=DEV)
    row = torch.arange(S, dtype=torch.int32, device=DEV)
    end = torch.stack([torch.where(row < x, row + 1, torch.zeros_like(row)) for x in n]).contiguous()
    scratch = torch.zeros(A.workspace_bytes(B, Hq, S, S) + 65536, dtype=torch.uint8, device=DEV)
    p, f = A.make_scored_params(q=q, k=k, v=v, k_cache=slab[0], v_cache=slab[1], out=out, scratch=scratch, freq_cis=tab, softcap=cap, key_end=end)
    A.prefill_scored(p, f)
    c = kv8.empty_cache(B, Hkv, T, d, block_len=block, row_pos=True, device=DEV)
    # the slab's rows are rotated already: stored as they are
    want = ref_append(c, slab[0].transpose(1, 2).contiguous(), slab[1].transpose(1, 2).contiguous(), [0, 0], n, [0, 0], None)
    kv8.append(c, slab[0].transpose(1, 2).contiguous(), slab[1].transpose(1, 2).contiguous(), new_lens=i32(n))
    same(c, want)
    w = torch.zeros(B, Hkv, T, device=DEV)
    past, pos = i32(n), i32(n)
    ds = torch.zeros(kv8.decode_workspace_bytes(B, Hq, Hkv, T, d, block_len=block, weights=True), dtype=torch.uint8, device=DEV)
    es = torch.zeros(kv8.evict_workspace_bytes(B, Hkv, T, d, block_len=block), dtype=torch.uint8, device=DEV)
    for step in range(12):
        q1, _ = tokens(g, "float16", B, 1, Hq, d, 2.0)
        k1, _ = tokens(g, "float16", B, 1, Hkv, d)
        v1, _ = tokens(g, "float16", B, 1, Hkv, d)
        o = torch.empty(B, Hq, 1, d, device=DEV)
        was, hp, hq = w.clone(), past.tolist(), pos.tolist()
        after = ref_append(c, k1, v1, hp, [1] * B, hq, tab)
        kv8.decode(c, q1, k1, v1, o, past_lens=past, token_pos=pos, freq_cis=tab, softcap=cap, weight_in=w, weight_out=w, scratch=ds, scratch_zeroed=True)
        same(c, after)
        check_decode(after, R.rotate(R.values(q1), tab, pos[:, None]), o, hp, hq, cap, None, None, was, w)
        past.add_(1)
        pos.add_(1)
        if step in (4, 8):
            kept = [min(x, 90) for x in past.tolist()]
            wc, ww, wp, wl = ref_evict(c, w, past.tolist(), 90, 16, 4, pos.tolist(), w, c.row_pos)
            wc.row_pos.copy_(wp)
            kv8.evict(c, past_lens=past, len_out=past, budget=90, recent=16, sinks=4, next_pos=pos, weight=w, scratch=es)
            assert past.tolist() == kept == wl
            assert torch.equal(w, ww)
            same(c, wc)
            assert sorted(c.row_pos[0, 0, :90].tolist())[:4] == [0, 1, 2, 3]
            assert set(range(int(pos[0]) - 16, int(pos[0]))) <= set(c.row_pos[0, 0, :90].tolist())


def _server(seed, B=2, Hq=8, Hkv=2, T=512, d=128, block=32, long=False):
    """State of a sequence of calls, and the calls: a chunk appended, three tokens, an eviction, a token; lengths and positions stay on the device."""
    g = gen(seed)
    T = 16384 if long else T
    c = kv8.empty_cache(B, Hkv, T, d, block_len=block, row_pos=True, device=DEV)
    big = T - 200
    first = big - 40
    ins = [tokens(g, "float16", B, S, h, d)[0] for S, h in ((first, Hkv), (first, Hkv), (40, Hkv), (40, Hkv))]
    steps = [[tokens(g, "float16", B, 1, h, d)[0] for h in (Hq, Hkv, Hkv)] for _ in range(4)]
    st = dict(c=c, w=torch.zeros(B, Hkv, T, device=DEV), past=i32([0] * B), pos=i32([0] * B), outs=[torch.empty(B, Hq, 1, d, device=DEV) for _ in steps],
              tab=table(T, d), ds=torch.zeros(kv8.decode_workspace_bytes(B, Hq, Hkv, T, d, block_len=block, weights=True), dtype=torch.uint8, device=DEV),
              es=torch.zeros(kv8.evict_workspace_bytes(B, Hkv, T, d, block_len=block), dtype=torch.uint8, device=DEV))

    def reset():
        for t in (*c.tensors().values(), st["w"]):
            t.zero_() if t.dtype != E4 else t.view(I8).zero_()
        st["past"].zero_()
        st["pos"].zero_()

    def run():
        past, pos, w = st["past"], st["pos"], st["w"]
        for k, v in (ins[:2], ins[2:]):
            kv8.append(c, k, v, past_lens=past, token_pos=pos, freq_cis=st["tab"])
            past.add_(k.shape[1])
            pos.add_(k.shape[1])
        for i, (q, k, v) in enumerate(steps):
            kv8.decode(c, q, k, v, st["outs"][i], past_lens=past, token_pos=pos, freq_cis=st["tab"], softcap=20.0, weight_in=w, weight_out=w,
                       scratch=st["ds"], scratch_zeroed=i % 2 == 0)  # both with and without a memset in front
            past.add_(1)
            pos.add_(1)
            if i == 2:
                kv8.evict(c, past_lens=past, len_out=past, budget=big // 2, recent=16, sinks=4, next_pos=pos, weight=w, scratch=st["es"])

    def result():
        return [t.clone() for t in (*st["outs"], st["w"], st["past"], st["pos"])], clone(c)

    return reset, run, result


@pytest.mark.parametrize("long", [False, True])  # an eviction by one CTA per head, and by clusters
def test_captured_calls_replay_as_they_run(cuda_device, long):
    reset, run, result = _server(42, long=long)
    reset()
    run()
    want, cache = result()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for _ in range(3):
        reset()
        graph.replay()
        got, now = result()
        assert all(torch.equal(a, b) for a, b in zip(want, got))
        same(now, cache)


def test_two_streams_at_once(cuda_device):
    """Two servers with caches and scratch of their own, their calls interleaved on two streams."""
    servers = [_server(43), _server(44, long=True)]
    want = []
    for reset, run, result in servers:
        reset()
        run()
        want.append(result())
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in servers]
    for _ in range(5):
        for (reset, run, _r), s in zip(servers, streams):
            with torch.cuda.stream(s):
                reset()
                run()
    torch.cuda.synchronize()
    for (_a, _b, result), (outs, cache) in zip(servers, want):
        got, now = result()
        assert all(torch.equal(a, b) for a, b in zip(outs, got))
        same(now, cache)


def test_empty_cache_and_dequantize(cuda_device):
    c = kv8.empty_cache(1, 2, 100, 64, block_len=64, device=DEV)
    assert tuple(c.k.shape) == (1, 2, 128, 64) and c.block_len == 64 and c.row_pos is None
    g = gen(41)
    k, _ = tokens(g, "float32", 1, 100, 2, 64)
    kv8.append(c, k, k)
    kd, vd = c.dequantize()
    # a code is off by half a step at most, a step being the block's largest magnitude / 127 (and a few roundings)
    step = c.k_scale.repeat_interleave(64, 2)[:, :, :100, None]
    assert bool(((kd[:, :, :100] - k.transpose(1, 2)).abs() <= step * (0.5 + 127 * 2.0 ** -22)).all())
    assert torch.equal(kd, vd)


# ------------------------------------------------------------------------------------------------ positions at the ends of their type
def test_append_positions_at_the_ends_of_int(cuda_device):
    """Positions outside the table are flagged and take the nearest row of it, however far outside; those that pass INT_MAX are kept as that."""
    g = gen(90)
    top, d, S = 2147483647, 64, 20
    tab = table(50, d)
    k, _ = tokens(g, "float32", 1, S, 2, d)
    for first, past in ((top, 0), (top - 1, 3), (top - 18, 5), (-top - 1, 7), (-top - 1, 0), (-3, 9), (45, 2)):
        c = kv8.empty_cache(1, 2, 48, d, block_len=16, row_pos=True, device=DEV)
        st = torch.zeros(4, dtype=torch.int32, device=DEV)
        want = clone(c)
        pos = [min(first + i, top) for i in range(S)]
        kr = R.rotate(k, tab, torch.tensor([[min(max(p, 0), 49) for p in pos]], device=DEV))
        for h in range(2):
            R.put_rows(want.k[0, h], want.k_scale[0, h], kr[0, :, h], list(range(past, past + S)), past, past, 16)
            R.put_rows(want.v[0, h], want.v_scale[0, h], k[0, :, h], list(range(past, past + S)), past, past, 16)
            want.row_pos[0, h, past:past + S] = i32(pos)
        kv8.append(c, k, k, start_pos=past, token_pos=i32([first]), freq_cis=tab, scratch=st)
        torch.cuda.synchronize()
        assert int(st[0]) == kv8.STATUS_BAD_POS
        same(c, want)


def test_decode_distances_beyond_31_bits(cuda_device):
    """Rows and token at opposite ends of int: the distance is 2^32 - 1 and not 1.  k = 0, so the weights are those of the bias."""
    d, top = 64, 2147483647
    for token, row in ((top, -top - 1), (-top - 1, top), (5, -top), (top, top - 7)):
        c = kv8.empty_cache(1, 1, 16, d, block_len=16, row_pos=True, device=DEV)
        one, zero = torch.ones(1, 1, 1, d, device=DEV), torch.zeros(1, 1, 1, d, device=DEV)
        kv8.append(c, zero, zero, token_pos=i32([row]))
        o = torch.empty(1, 1, 1, d, device=DEV)
        s = torch.zeros(kv8.decode_workspace_bytes(1, 1, 1, 16, d, block_len=16), dtype=torch.uint8, device=DEV)
        kv8.decode(c, zero, zero, one, o, start_pos=1, token_pos=i32([token]), alibi_slopes=torch.full((1,), 2.0 ** -32, device=DEV), scratch=s)
        want = 1.0 / (1.0 + math.exp(-abs(token - row) * 2.0 ** -32))
        assert float((o - want).abs().max()) <= 2.0 ** -20  # v = 1 is coded as 127 * fp32(1 / 127); exponent and quotient a few roundings of 2^-23


# ------------------------------------------------------------------------------------------------ joins of many splits
@pytest.mark.parametrize("past", [[8191], [8192], [20000, 8200]])
@pytest.mark.parametrize("dtype,d,G", [(I8, 64, 1), (E4, 64, 3), (I8, 128, 8), (E4, 128, 1), (I8, 256, 4), (I8, 128, 9)])
@pytest.mark.parametrize("weights", [None, "apart"])
def test_decode_joins_more_than_64_splits(cuda_device, past, dtype, d, G, weights):
    """64, 65 and 157 splits of 128 rows: the join's weights are worked out 64 splits at a time; with few heads its threads share a column's splits, with many they take
    several columns each."""
    run_decode(21 + G + d, B=len(past), Hq=G, Hkv=1, T=20096, d=d, block=32, dtype=dtype, past=past, split=128, weights=weights, cap=30.0 if G == 8 else 0.0)


def test_decode_of_many_splits_is_repeatable(cuda_device):
    c, (q, k, v, o), args = run_decode(22, B=1, Hq=16, Hkv=2, T=20096, d=128, block=64, dtype=I8, past=[20000], split=128)
    for _ in range(5):
        again = torch.empty_like(o)
        kv8.decode(c, q, k, v, again, **args)
        assert torch.equal(o, again)


# ------------------------------------------------------------------------------------------------ captures with several branches
def test_captured_calls_wait_for_every_branch(cuda_device):
    """Inputs and lengths are made on two other streams, by kernels of this family and by others, and the results are used on a third: as graph nodes
    the calls have several predecessors and successors."""
    g = gen(95)
    B, Hq, Hkv, T, d, block, S = 2, 8, 2, 4096, 128, 32, 1500
    raw = [tokens(g, "float16", B, n, h, d)[0] for n, h in ((S, Hkv), (S, Hkv), (1, Hq), (1, Hkv), (1, Hkv))]
    tab = table(T, d)
    c, other = (kv8.empty_cache(B, Hkv, T, d, block_len=block, row_pos=True, device=DEV) for _ in range(2))
    src = [torch.empty_like(t) for t in raw]
    ins = [torch.empty_like(t) for t in raw]
    past, nxt, w = i32([0] * B), i32([S + 1] * B), torch.zeros(B, Hkv, T, device=DEV)
    out, twice = torch.empty(B, Hq, 1, d, device=DEV), torch.empty(B, Hq, 1, d, device=DEV)
    ds, es = (torch.zeros(n, dtype=torch.uint8, device=DEV) for n in (kv8.decode_workspace_bytes(B, Hq, Hkv, T, d, block_len=block, weights=True),
                                                                      kv8.evict_workspace_bytes(B, Hkv, T, d, block_len=block)))
    left, right = torch.cuda.Stream(), torch.cuda.Stream()

    def run():
        main = torch.cuda.current_stream()
        past.zero_()
        w.zero_()
        left.wait_stream(main)
        right.wait_stream(main)
        with torch.cuda.stream(left):  # k, q: other kernels, with some work in front of them
            for _ in range(8):
                ins[0].copy_(src[0])
                ins[2].copy_(src[2])
                ins[3].copy_(src[3])
        with torch.cuda.stream(right):  # v: behind a call of this family on another cache
            for _ in range(8):
                ins[1].copy_(src[1])
                ins[4].copy_(src[4])
            kv8.append(other, ins[1], ins[1])
        main.wait_stream(left)
        main.wait_stream(right)
        kv8.append(c, ins[0], ins[1], past_lens=past, freq_cis=tab)
        right.wait_stream(main)
        with torch.cuda.stream(right):
            past.add_(S)
        main.wait_stream(right)
        kv8.decode(c, ins[2], ins[3], ins[4], out, past_lens=past, freq_cis=tab, weight_in=w, weight_out=w, scratch=ds)
        past.add_(1)
        left.wait_stream(main)
        with torch.cuda.stream(left):
            torch.mul(out, 2, out=twice)
        kv8.evict(c, past_lens=past, len_out=past, budget=1000, recent=16, sinks=4, next_pos=nxt, weight=w, scratch=es)
        main.wait_stream(left)

    def result():
        torch.cuda.synchronize()
        return [t.clone() for t in (out, twice, past, w[..., :1000], c.k.view(I8)[:, :, :1000], c.v.view(I8)[:, :, :1000], c.row_pos[:, :, :1000], other.v.view(I8))]

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for turn in range(4):
        for t, r in zip(src, raw):
            t.copy_(r * (1 + 0.25 * turn))
        torch.cuda.synchronize()
        run()
        want = result()
        for t in (*ins, out, twice):
            t.fill_(7)
        for x in (c.k, c.v, c.k_scale, c.v_scale, c.row_pos):
            x.zero_()
        torch.cuda.synchronize()
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(want, result())), turn
    assert torch.equal(out * 2, twice)


# ------------------------------------------------------------------------------------------------ accumulated weights
@pytest.mark.parametrize("G", [1, 6, 8, 11])
def test_accumulated_weights_are_rounded_once_per_step(cuda_device, G):
    """Weights of 2^-11 or less join accumulated ones between 1/2 and 1: the group's sum is below 2^-7 and off by 2^-20 of itself at most, so the result is off
    by its own rounding, 2^-25, and 2^-27."""
    g = gen(96)
    T, d, n = 4096, 64, 4095
    c = used_cache(g, 1, 1, T, d, 64, I8)
    q, _ = tokens(g, "float32", 1, 1, G, d, 0.01)
    k, _ = tokens(g, "float32", 1, 1, 1, d)
    w = torch.rand(1, 1, T, generator=g, device=DEV) * 0.49 + 0.5
    w_out, o = torch.empty_like(w), torch.empty(1, G, 1, d, device=DEV)
    s = torch.zeros(kv8.decode_workspace_bytes(1, G, 1, T, d, weights=True), dtype=torch.uint8, device=DEV)
    kv8.decode(c, q, k, k, o, start_pos=n, weight_in=w, weight_out=w_out, scratch=s)
    kd = R.dequant(c.k[0, 0], c.k_scale[0, 0], 64)
    p = torch.softmax(q[0, 0].double() @ kd.T / math.sqrt(d), -1)
    assert float(p.max()) < 2.0 ** -11
    want = w[0, 0].double() + p.sum(0)
    want[n] -= w[0, 0, n].double()
    assert float((w_out[0, 0].double() - want).abs().max()) <= 2.0 ** -25 + 2.0 ** -27
