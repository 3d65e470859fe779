"""Host side of the score forms: refusals and the parameter blocks, without a GPU."""
import ctypes as C

import numpy as np
import pytest

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


def test_binding_refuses_shapes_and_types():
    for bad in (dict(alibi_slopes=np.zeros(7, np.float32)), dict(key_begin=np.zeros(3, np.int32)), dict(key_begin=np.zeros(2, np.int64)),
                dict(k=np.zeros((2, 1, 3, 128), np.float16)), dict(v=np.zeros((2, 1, 4, 128), np.float32)),
                dict(k_cache=np.zeros((2, 8, 64, 128), np.float16)), dict(k_cache=np.zeros((2, 4, 64, 128), np.float16)[:, :, ::2], v_cache=np.zeros((2, 4, 32, 128), np.float16))):
        with pytest.raises(ValueError):
            _call(**bad)
