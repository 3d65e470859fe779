"""Host side of the score forms: refusals and the parameter blocks, without a GPU."""
import ctypes as C

import numpy as np
import pytest
import torch

from fasterllama_b200 import _lib
from fasterllama_b200 import attention as A


def _call(S=1, H=8, Hkv=4, d=128, T=64, **kw):
    B = 2
    a = dict(q=np.zeros((B, S, H, d), np.float16), k=np.zeros((B, S, Hkv, d), np.float16), v=np.zeros((B, S, Hkv, d), np.float16),
             k_cache=np.zeros((B, Hkv, T, d), np.float16), v_cache=np.zeros((B, Hkv, T, d), np.float16), out=np.zeros((B, H, S, d), np.float16),
             scratch=np.zeros(A.workspace_bytes(B, H, T, S, size_per_head=d) + 65536, np.uint8))
    a.update(kw)
    p, f = A.make_scored_params(**a)
    return p, f, a


def test_a_good_call_passes_and_names_heads_and_strides():
    p, f, keep = _call()
    assert A.validate_scored(p, f) == _lib.FLB_OK
    assert (p.head_num, f.kv_head_num, f.kv_row_stride, p.qkv_row_stride) == (8, 4, 512, 0)
    assert p.k == keep["k"].ctypes.data and p.k_cache == keep["k_cache"].ctypes.data
    assert A.validate_scored(p, None) == _lib.FLB_OK


@pytest.mark.parametrize("S,field,value,status", [
    (1, "kv_head_num", 3, _lib.FLB_ERR_BAD_SHAPE), (1, "kv_head_num", 16, _lib.FLB_ERR_BAD_SHAPE), (1, "kv_head_num", -1, _lib.FLB_ERR_BAD_SHAPE),
    (5, "kv_row_stride", 8, _lib.FLB_ERR_BAD_SHAPE), (5, "kv_row_stride", 513, _lib.FLB_ERR_MISALIGNED), (1, "softcap", -2.0, _lib.FLB_ERR_BAD_SHAPE),
    (1, "softcap", float("nan"), _lib.FLB_ERR_BAD_SHAPE), (5, "softcap", float("inf"), _lib.FLB_ERR_BAD_SHAPE), (1, "key_end", 4096, _lib.FLB_ERR_UNSUPPORTED)])
def test_refusals(S, field, value, status):
    p, f, keep = _call(S=S)
    setattr(f, field, value)
    assert A.validate_scored(p, f) == status
    lib = _lib.load_library()
    assert lib.flb_attn_forward_scored(C.byref(p), C.byref(f), None) == status  # refused before any CUDA call


@pytest.mark.parametrize("S", [1, 5])
@pytest.mark.parametrize("cap", [1e-30, 2.0 ** -11, 2.0 ** 41, 3.4e38])
def test_caps_that_arithmetic_cannot_hold_are_refused(S, cap):
    p, f, keep = _call(S=S)
    f.softcap = cap
    assert A.validate_scored(p, f) == _lib.FLB_ERR_BAD_SHAPE
    for good in (2.0 ** -10, 30.0, 2.0 ** 40):
        f.softcap = good
        assert A.validate_scored(p, f) == _lib.FLB_OK
    f.softcap, p.softmax_scale = 2.0 ** -10, 65.0
    assert A.validate_scored(p, f) == (_lib.FLB_OK if S == 1 else _lib.FLB_ERR_BAD_SHAPE)


def test_the_wrong_entry_point_and_null_blocks_are_refused():
    lib = _lib.load_library()
    p, f, keep = _call(S=5)
    assert lib.flb_attn_decode_scored(C.byref(p), C.byref(f), None) == _lib.FLB_ERR_BAD_SHAPE
    p, f, keep = _call(S=1)
    assert lib.flb_attn_prefill_scored(C.byref(p), C.byref(f), None) == _lib.FLB_ERR_BAD_SHAPE
    assert lib.flb_attn_forward_scored(None, None, None) == _lib.FLB_ERR_NULL_POINTER
    p.q = None
    assert lib.flb_attn_decode_scored(C.byref(p), C.byref(f), None) == _lib.FLB_ERR_NULL_POINTER


def test_key_bounds_of_a_prefill_need_their_scratch():
    S = 300
    begin = np.zeros((2, S), np.int32)
    p, f, keep = _call(S=S, T=512, key_begin=begin)
    need = A.scored_workspace_bytes(p, f)
    assert need > A.scored_workspace_bytes(p, None)
    p.scratch_bytes = need
    assert A.validate_scored(p, f) == _lib.FLB_OK
    p.scratch_bytes = A.scored_workspace_bytes(p, None)
    assert A.validate_scored(p, f) == _lib.FLB_ERR_SCRATCH_TOO_SMALL


@pytest.mark.parametrize("S", [1, 6])
def test_tensors_and_arrays_fill_the_same_blocks(S):
    B, H, T, d = 2, 8, 64, 128
    kw = dict(alibi_slopes=np.ones(H, np.float32), key_begin=np.zeros((B,) if S == 1 else (B, S), np.int32), freq_cis=np.zeros((T, d), np.float32), softcap=7.5,
              past_lens=np.zeros(B, np.int32), max_past_len=33, rope_pos0=2, rope_add_past=True, mask_mode=A.FLB_MASK_GENERIC, attn_mask=np.zeros((T, T), np.float32),
              scratch_zeroed=True, split_len=256, early_start=1, start_pos=3, act_scale=np.ones(B * S, np.float32), out_q8=np.zeros((B, S, H * d), np.int8),
              out_q8_scale=np.zeros(B * S, np.float32))
    merged = np.zeros((B, S, (H + 4 + 4) * d), np.float16)  # q, k and v as columns of one projection
    for name, at, heads in (("q", 0, H), ("k", H, 4), ("v", H + 4, 4)):
        kw[name] = np.lib.stride_tricks.as_strided(merged[:, :, at * d:], (B, S, heads, d), (merged.strides[0], merged.strides[1], 2 * d, 2))
    p, f, arrays = _call(S=S, T=T, **kw)
    pt, ft = A.make_scored_params(**{n: torch.from_numpy(x) if isinstance(x, np.ndarray) else x for n, x in arrays.items()})
    assert bytes(p) == bytes(pt) and bytes(f) == bytes(ft)
    assert p.qkv_row_stride == 16 * d == f.kv_row_stride and f.kv_head_num == 4


def test_tensors_are_refused_like_arrays():
    def t(**kw):
        a = dict(q=torch.zeros(2, 1, 8, 128), k=torch.zeros(2, 1, 4, 128), v=torch.zeros(2, 1, 4, 128), k_cache=torch.zeros(2, 4, 64, 128), v_cache=torch.zeros(2, 4, 64, 128),
                 out=torch.zeros(2, 8, 1, 128), scratch=torch.zeros(1 << 20, dtype=torch.uint8))
        return A.make_scored_params(**{**a, **kw})

    assert A.validate_scored(*t()) == _lib.FLB_OK
    for bad in (dict(alibi_slopes=torch.zeros(7)), dict(key_begin=torch.zeros(3, dtype=torch.int32)), dict(key_begin=torch.zeros(2, dtype=torch.int64)), dict(k=torch.zeros(2, 1, 3, 128)),
                dict(v=torch.zeros(2, 1, 4, 128).half()), dict(k_cache=torch.zeros(2, 8, 64, 128)), dict(k_cache=torch.zeros(2, 4, 64, 256)[..., ::2]), dict(q=torch.zeros(2, 8, 128)),
                dict(out=torch.zeros(2, 8, 1, 128, dtype=torch.bfloat16)), dict(freq_cis=torch.zeros(64, 128).double()), dict(freq_cis=torch.zeros(128, 64).T), dict(q=np.zeros(3)),
                dict(start_pos=1 << 40), dict(act_scale="x")):
        with pytest.raises((ValueError, AttributeError, IndexError)):
            t(**bad)


def test_binding_refuses_shapes_and_types():
    for bad in (dict(alibi_slopes=np.zeros(7, np.float32)), dict(key_begin=np.zeros(3, np.int32)), dict(key_begin=np.zeros(2, np.int64)),
                dict(k=np.zeros((2, 1, 3, 128), np.float16)), dict(v=np.zeros((2, 1, 4, 128), np.float32)),
                dict(k_cache=np.zeros((2, 8, 64, 128), np.float16)), dict(k_cache=np.zeros((2, 4, 64, 128), np.float16)[:, :, ::2], v_cache=np.zeros((2, 4, 32, 128), np.float16))):
        with pytest.raises(ValueError):
            _call(**bad)


def _tensors(S=1, dtype=torch.float16, **kw):
    B, H, Hkv, T, d = 2, 8, 4, 64, 128
    a = dict(q=torch.zeros(B, S, H, d, dtype=dtype), k=torch.zeros(B, S, Hkv, d, dtype=dtype), v=torch.zeros(B, S, Hkv, d, dtype=dtype),
             k_cache=torch.zeros(B, Hkv, T, d, dtype=torch.float16), v_cache=torch.zeros(B, Hkv, T, d, dtype=torch.float16), out=torch.zeros(B, H, S, d),
             scratch=torch.zeros(A.workspace_bytes(B, H, T, S, size_per_head=d) + 65536, dtype=torch.uint8))
    return A.make_scored_params(**{**a, **kw})


SCALES = dict(act_scale=2 * 5, q_w_scale=8 * 128, k_w_scale=4 * 128, v_w_scale=4 * 128)


@pytest.mark.parametrize("name", list(SCALES))
def test_scales_of_int32_inputs_have_their_lengths(name):
    good = {n: torch.ones(k) for n, k in SCALES.items()}
    assert A.validate_scored(*_tensors(5, torch.int32, **good)) == _lib.FLB_OK
    for n in (SCALES[name] - 1, SCALES[name] + 1, 0):
        with pytest.raises(ValueError, match=name):
            _tensors(5, torch.int32, **{**good, name: torch.ones(n)})


@pytest.mark.parametrize("kw,rows", [
    (dict(S=5), 5), (dict(S=5, rope_pos0=3), 8), (dict(start_pos=9, rope_add_past=True), 10), (dict(start_pos=9), 1), (dict(start_pos=9, rope_pos0=7), 8),
    (dict(past_lens=torch.zeros(2, dtype=torch.int32), max_past_len=20, rope_add_past=True), 21),
    (dict(past_lens=torch.zeros(2, dtype=torch.int32), rope_add_past=True, rope_pos0=2), 66)])
def test_rope_tables_reach_every_position(kw, rows):
    assert A.validate_scored(*_tensors(freq_cis=torch.zeros(rows, 128), **kw)) == _lib.FLB_OK
    with pytest.raises(ValueError, match="freq_cis"):
        _tensors(freq_cis=torch.zeros(rows - 1, 128), **kw)
    if rows > 1:
        with pytest.raises(ValueError, match="freq_cis"):
            _tensors(freq_cis=torch.zeros(rows, 64), **kw)


@pytest.mark.parametrize("kw,n", [(dict(S=5), 5), (dict(start_pos=9), 10), (dict(past_lens=torch.zeros(2, dtype=torch.int32), max_past_len=20), 21),
                                  (dict(past_lens=torch.zeros(2, dtype=torch.int32)), 64)])
def test_additive_masks_reach_every_position(kw, n):
    kw = dict(kw, mask_mode=A.FLB_MASK_GENERIC)
    assert A.validate_scored(*_tensors(attn_mask=torch.zeros(n, n), **kw)) == _lib.FLB_OK
    assert A.validate_scored(*_tensors(attn_mask=torch.zeros(n, n + 3), **kw)) == _lib.FLB_OK
    assert A.validate_scored(*_tensors(attn_mask=torch.zeros(n * n), mask_row_stride=n, **kw)) == _lib.FLB_OK
    for bad in (dict(attn_mask=torch.zeros(n - 1, n)), dict(attn_mask=torch.zeros(n, n), mask_row_stride=n + 1)):
        with pytest.raises(ValueError, match="attn_mask"):
            _tensors(**bad, **kw)


@pytest.mark.parametrize("S", [1, 5])
def test_quantised_outputs_have_their_sizes(S):
    good = dict(out_q8=torch.zeros(2, S, 1024, dtype=torch.int8), out_q8_scale=torch.zeros(2 * S))
    assert A.validate_scored(*_tensors(S, **good)) == _lib.FLB_OK
    for bad in (dict(out_q8=torch.zeros(2, S, 1023, dtype=torch.int8)), dict(out_q8_scale=torch.zeros(2 * S - 1))):
        with pytest.raises(ValueError, match="out_q8"):
            _tensors(S, **{**good, **bad})


@pytest.mark.parametrize("S", [1, 5])
def test_host_memory_is_not_launched_on(S):
    p, f = _tensors(S)
    for call in (A.forward_scored, A.decode_scored if S == 1 else A.prefill_scored):
        with pytest.raises(ValueError, match="CUDA device"):
            call(p, f)
    with pytest.raises(ValueError, match="memory"):
        _tensors(S, alibi_slopes=torch.zeros(8, device="meta"))


@pytest.mark.parametrize("S,field", [(1, "alibi_slopes"), (1, "key_begin"), (5, "alibi_slopes"), (5, "key_begin"), (5, "key_end")])
def test_words_at_odd_addresses_are_refused(S, field):
    p, f, keep = _call(S=S)
    setattr(f, field, 4098)
    assert A.validate_scored(p, f) == _lib.FLB_ERR_MISALIGNED
