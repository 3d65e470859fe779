"""Host side of the 8-bit cache: the library exports what the header declares, the structs match, and every refusal answers
with its status before anything touches a GPU."""
import ctypes as C
import os
import re
import subprocess

import pytest
import torch

from fasterllama_b200 import _lib, kv8

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_library_exports_every_declared_symbol():
    lib = kv8.load_library()
    header = open(os.path.join(ROOT, "include", "flb_kv8.h")).read()
    declared = set(re.findall(r"^int\s+(flb_\w+)\s*\(", header, flags=re.M))
    assert declared == set(kv8.EXPORTS)
    for name in declared:
        assert hasattr(lib, name)


def test_struct_layouts_match_the_headers(tmp_path):
    structs = {"flb_kv8_cache": kv8.FlbKv8Cache, "flb_kv8_append_params": kv8.FlbKv8Append, "flb_kv8_decode_params": kv8.FlbKv8Decode,
               "flb_kv8_evict_params": kv8.FlbKv8Evict, "flb_score_form": _lib.FlbScoreForm}
    want, lines = [], []
    for name, cls in structs.items():
        lines.append(f'printf("%zu\\n", sizeof({name}));')
        want.append(C.sizeof(cls))
        for field, _ in cls._fields_:
            lines.append(f'printf("%zu\\n", offsetof({name}, {field}));')
            want.append(getattr(cls, field).offset)
    probe, exe = tmp_path / "probe.c", tmp_path / "probe"
    probe.write_text('#include <stdio.h>\n#include "flb_kv8.h"\nint main(void){' + "".join(lines) + "return 0;}\n")
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(probe), "-o", str(exe)], check=True)
    assert [int(x) for x in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()] == want


def _cache(**over):
    c = dict(B=2, H=4, T=128, d=128, block_len=32, dtype=torch.int8, row_pos=True)
    c.update(over)
    return kv8.empty_cache(c["B"], c["H"], c["T"], c["d"], block_len=c["block_len"], dtype=c["dtype"], row_pos=c["row_pos"], device="cpu")


def _append(S=3, start_pos=5, **kw):
    c = _cache()
    k = torch.zeros(2, S, 4, 128, dtype=torch.float16)
    return kv8.append_params(c, k, k.clone(), start_pos=start_pos, **kw), c


def _decode(Hq=8, start_pos=5, **kw):
    c = _cache()
    k = torch.zeros(2, 1, 4, 128, dtype=torch.float16)
    scratch = torch.zeros(kv8.decode_workspace_bytes(2, Hq, 4, 128, 128, block_len=32, weights=True), dtype=torch.uint8)
    out = torch.zeros(2, Hq, 1, 128)
    w = torch.zeros(2, 4, 128)
    return kv8.decode_params(c, torch.zeros(2, 1, Hq, 128, dtype=torch.float16), k, k.clone(), out, start_pos=start_pos, scratch=scratch,
                             weight_in=w, weight_out=w, **kw), (c, scratch, out, w, k)


def _evict(**kw):
    c = _cache()
    scratch = torch.zeros(kv8.evict_workspace_bytes(2, 4, 128, 128, block_len=32), dtype=torch.uint8)
    a = dict(len_out=torch.zeros(2, dtype=torch.int32), budget=64, recent=8, sinks=2, next_pos=torch.zeros(2, dtype=torch.int32),
             weight=torch.zeros(2, 4, 128), start_pos=100, scratch=scratch)
    a.update(kw)
    return kv8.evict_params(c, **a), (c, a)


def _refused(p, field, value, status):
    obj, name = (p.cache, field[6:]) if field.startswith("cache.") else (p, field)
    old = getattr(obj, name)
    setattr(obj, name, value)
    assert kv8.validate(p) == status, (field, value)
    setattr(obj, name, old)
    assert kv8.validate(p) == _lib.FLB_OK


CACHE_REFUSALS = [
    ("cache.batch_size", 0, _lib.FLB_ERR_BAD_SHAPE), ("cache.kv_head_num", -1, _lib.FLB_ERR_BAD_SHAPE), ("cache.size_per_head", 96, _lib.FLB_ERR_UNSUPPORTED),
    ("cache.block_len", 24, _lib.FLB_ERR_UNSUPPORTED), ("cache.block_len", 256, _lib.FLB_ERR_UNSUPPORTED), ("cache.total_len", 100, _lib.FLB_ERR_BAD_SHAPE),
    ("cache.code_type", 2, _lib.FLB_ERR_BAD_ENUM), ("cache.k_codes", None, _lib.FLB_ERR_NULL_POINTER), ("cache.v_scale", None, _lib.FLB_ERR_NULL_POINTER),
    ("cache.v_codes", 4100, _lib.FLB_ERR_MISALIGNED), ("cache.batch_size", 1 << 24, _lib.FLB_ERR_TOO_LARGE),
]


@pytest.mark.parametrize("field,value,status", CACHE_REFUSALS + [
    ("seq_len", 0, _lib.FLB_ERR_BAD_SHAPE), ("seq_len", 129, _lib.FLB_ERR_BAD_SHAPE), ("start_pos", 126, _lib.FLB_ERR_BAD_SHAPE),
    ("start_pos", -1, _lib.FLB_ERR_BAD_SHAPE), ("start_pos", 2147483647, _lib.FLB_ERR_BAD_SHAPE), ("input_mode", 3, _lib.FLB_ERR_BAD_ENUM),
    ("input_mode", 0, _lib.FLB_ERR_NULL_POINTER), ("k", None, _lib.FLB_ERR_NULL_POINTER), ("v", 4098, _lib.FLB_ERR_MISALIGNED),
    ("kv_row_stride", 511, _lib.FLB_ERR_BAD_SHAPE), ("kv_row_stride", 513, _lib.FLB_ERR_MISALIGNED), ("freq_cis", 4096, _lib.FLB_ERR_BAD_SHAPE)])
def test_append_refusals(field, value, status):
    p, keep = _append()
    _refused(p, field, value, status)


@pytest.mark.parametrize("field,value,status", CACHE_REFUSALS + [
    ("head_num", 6, _lib.FLB_ERR_BAD_SHAPE), ("head_num", 0, _lib.FLB_ERR_BAD_SHAPE), ("start_pos", 128, _lib.FLB_ERR_BAD_SHAPE), ("start_pos", -1, _lib.FLB_ERR_BAD_SHAPE),
    ("split_len", 64, _lib.FLB_ERR_BAD_SHAPE), ("split_len", 8320, _lib.FLB_ERR_BAD_SHAPE), ("softcap", -1.0, _lib.FLB_ERR_BAD_SHAPE),
    ("softcap", float("nan"), _lib.FLB_ERR_BAD_SHAPE), ("softcap", float("inf"), _lib.FLB_ERR_BAD_SHAPE), ("weight_in", None, _lib.FLB_ERR_NULL_POINTER),
    ("weight_out", None, _lib.FLB_ERR_NULL_POINTER), ("out", None, _lib.FLB_ERR_NULL_POINTER), ("out_dtype", 2, _lib.FLB_ERR_BAD_ENUM), ("scratch", None, _lib.FLB_ERR_NULL_POINTER),
    ("scratch", 4104, _lib.FLB_ERR_MISALIGNED), ("scratch_bytes", 64, _lib.FLB_ERR_SCRATCH_TOO_SMALL), ("q", 4100, _lib.FLB_ERR_MISALIGNED),
    ("q_row_stride", 8, _lib.FLB_ERR_BAD_SHAPE), ("input_mode", -1, _lib.FLB_ERR_BAD_ENUM)])
def test_decode_refusals(field, value, status):
    p, keep = _decode()
    _refused(p, field, value, status)


def test_decode_length_bound_is_checked_against_the_slab():
    p, keep = _decode()
    p.past_lens, p.max_past_len = 4096, 128
    assert kv8.validate(p) == _lib.FLB_ERR_BAD_SHAPE
    p.max_past_len = 0  # the whole slab
    assert kv8.validate(p) == _lib.FLB_OK


@pytest.mark.parametrize("field,value,status", CACHE_REFUSALS + [
    ("cache.row_pos", None, _lib.FLB_ERR_NULL_POINTER), ("budget", 0, _lib.FLB_ERR_BAD_SHAPE), ("recent", 63, _lib.FLB_ERR_BAD_SHAPE),
    ("recent", -1, _lib.FLB_ERR_BAD_SHAPE), ("sinks", 57, _lib.FLB_ERR_BAD_SHAPE), ("sinks", 2147483647, _lib.FLB_ERR_BAD_SHAPE), ("next_pos", None, _lib.FLB_ERR_NULL_POINTER),
    ("weight", None, _lib.FLB_ERR_NULL_POINTER), ("weight_out", None, _lib.FLB_ERR_NULL_POINTER), ("pos_out", None, _lib.FLB_ERR_NULL_POINTER),
    ("len_out", None, _lib.FLB_ERR_NULL_POINTER), ("start_pos", 129, _lib.FLB_ERR_BAD_SHAPE), ("scratch_bytes", 16, _lib.FLB_ERR_SCRATCH_TOO_SMALL),
    ("scratch", None, _lib.FLB_ERR_NULL_POINTER)])
def test_evict_refusals(field, value, status):
    p, keep = _evict()
    _refused(p, field, value, status)


@pytest.mark.parametrize("cap", [1e-30, 2.0 ** -11, 2.0 ** 41, 3.4e38, -0.5])
def test_caps_that_arithmetic_cannot_hold_are_refused(cap):
    p, keep = _decode()
    _refused(p, "softcap", cap, _lib.FLB_ERR_BAD_SHAPE)
    for good in (0.0, 2.0 ** -10, 30.0, 2.0 ** 40):
        p.softcap = good
        assert kv8.validate(p) == _lib.FLB_OK


def test_rows_of_more_than_2_31_elements_are_refused():
    p, keep = _append()
    p.cache.batch_size, p.cache.kv_head_num = 1, 1 << 24  # times 128
    assert kv8.validate(p) == _lib.FLB_ERR_TOO_LARGE
    p, keep = _decode()
    p.cache.batch_size, p.head_num = 1, 1 << 24
    assert kv8.validate(p) == _lib.FLB_ERR_TOO_LARGE


def test_binding_refuses_a_table_without_rows_and_a_scratch_without_a_word():
    c = _cache()
    k = torch.zeros(2, 1, 4, 128, dtype=torch.float16)
    with pytest.raises(ValueError, match="freq_cis"):
        kv8.append_params(c, k, k.clone(), freq_cis=torch.zeros(0, 128))
    with pytest.raises(ValueError, match="scratch"):
        kv8.append_params(c, k, k.clone(), scratch=torch.zeros(3, dtype=torch.uint8))


def test_null_blocks_and_launches_without_a_launch():
    lib = kv8.load_library()
    for name in ("append", "decode", "evict"):
        assert getattr(lib, f"flb_kv8_validate_{name}")(None) == _lib.FLB_ERR_NULL_POINTER
        assert getattr(lib, f"flb_kv8_{name}")(None, None) == _lib.FLB_ERR_NULL_POINTER
    p, keep = _append()
    p.k = None
    assert lib.flb_kv8_append(C.byref(p), None) == _lib.FLB_ERR_NULL_POINTER


def test_binding_refuses_shapes_types_and_hosts():
    c = _cache()
    k = torch.zeros(2, 1, 4, 128, dtype=torch.float16)
    with pytest.raises(ValueError, match="CUDA device"):
        kv8.append(c, k, k.clone())
    with pytest.raises(ValueError):
        kv8.append_params(c, k, torch.zeros(2, 1, 3, 128, dtype=torch.float16))
    with pytest.raises(ValueError):
        kv8.append_params(c, k.double(), k.double())
    with pytest.raises(ValueError):
        kv8.append_params(c, k.int(), k.int())  # scales missing
    with pytest.raises(ValueError):
        kv8.append_params(c, k.transpose(2, 3).contiguous().transpose(2, 3), k)
    with pytest.raises(ValueError):
        kv8.append_params(c, k, k.clone(), past_lens=torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError, match="row_pos"):
        kv8.evict_params(_cache(row_pos=False), len_out=torch.zeros(2, dtype=torch.int32), budget=1, weight=torch.zeros(2, 4, 128))
    bad = kv8.Cache(c.k, c.v.float(), c.k_scale, c.v_scale)
    with pytest.raises(ValueError):
        kv8.append_params(bad, k, k.clone())


def test_binding_passes_on_what_python_raises():
    c = _cache()
    q = torch.zeros(2, 1, 4, 128, dtype=torch.float16)
    out = torch.zeros(2, 4, 1, 128)
    for bad in (dict(scratch_zeroed=torch.zeros(2)), dict(softcap="1"), dict(split_len=1.5), dict(start_pos=1 << 40), dict(max_past_len=None), dict(past_lens=[1, 2])):
        with pytest.raises((TypeError, ValueError, RuntimeError)):
            kv8.decode_params(c, q, q.clone(), q.clone(), out, **bad)
    kv8.decode_params(c, q, q.clone(), q.clone(), out)  # and nothing of it stays behind


def test_merged_projection_columns_share_a_stride():
    c = _cache()
    buf = torch.zeros(2, 3, (8 + 4 + 4) * 128, dtype=torch.float16)
    k, v = (buf[:, :, a * 128:(a + 4) * 128].unflatten(2, (4, 128)) for a in (8, 12))
    p = kv8.append_params(c, k, v)
    assert p.kv_row_stride == 16 * 128 and p.k == buf.data_ptr() + 8 * 256
    assert kv8.validate(p) == _lib.FLB_OK


def test_workspaces_cover_shorter_calls_and_grow():
    a = kv8.decode_workspace_bytes(2, 8, 4, 1024)
    assert kv8.decode_workspace_bytes(2, 8, 4, 4096) > a >= kv8.counter_bytes(2, 8, 4)
    assert kv8.decode_workspace_bytes(2, 8, 4, 1024, weights=True) >= a + 2 * 8 * 1024 * 4
    assert kv8.evict_workspace_bytes(2, 4, 2048) > kv8.evict_workspace_bytes(2, 4, 1024)


def test_words_at_odd_addresses_are_refused():
    p, keep = _append()
    for field in ("past_lens", "new_lens", "token_pos", "act_scale", "status"):
        _refused(p, field, 4098, _lib.FLB_ERR_MISALIGNED)
    p, keep = _decode()
    for field in ("past_lens", "token_pos", "act_scale", "alibi_slopes", "key_begin"):
        _refused(p, field, 4097, _lib.FLB_ERR_MISALIGNED)
    p, keep = _evict()
    for field in ("past_lens", "len_out", "next_pos"):
        _refused(p, field, 4099, _lib.FLB_ERR_MISALIGNED)
    c = _cache()
    k = torch.zeros(2, 1, 4, 128, dtype=torch.float16)
    assert kv8.validate(kv8.append_params(c, k, k.clone(), scratch=torch.zeros(9, dtype=torch.uint8)[1:])) == _lib.FLB_ERR_MISALIGNED


def test_kernels_of_the_cache_use_no_read_only_loads():
    """They are resident while the kernel in front still writes what they read."""
    src = os.path.join(ROOT, "fasterllama_b200", "csrc")
    for name in sorted(os.listdir(src)):
        if name.startswith("kv8"):
            text = open(os.path.join(src, name)).read()
            assert "__ldg(" not in text and "global.nc" not in text and "__restrict__" not in text, name
