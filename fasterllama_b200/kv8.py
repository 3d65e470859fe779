"""The 8-bit K/V cache: host-side entry to include/flb_kv8.h.

A `Cache` names the tensors of one layer's cache.  `append` stores tokens (a prompt, a chunk, one), `decode` stores one
token per sequence and attends over everything cached, `evict` cuts sequences down to a budget of rows by the attention weight
that `decode` accumulated.  Everything is stream-ordered and works in the caller's tensors; scratch comes from the caller
as in `attention` (`decode_workspace_bytes`, `evict_workspace_bytes`).  Calls run on the device of the cache, on its
current stream unless one is given."""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass
from typing import Any

import torch

from . import _lib, _tensor_args

FLB_KV8_I8, FLB_KV8_E4M3 = 0, 1
STATUS_BAD_LEN, STATUS_BAD_POS = 4, 32


class FlbKv8Cache(C.Structure):
    """struct flb_kv8_cache, field for field."""

    _fields_ = [(n, C.c_int) for n in ("batch_size", "kv_head_num", "size_per_head", "total_len", "block_len", "code_type")] + [
        (n, C.c_void_p) for n in ("k_codes", "v_codes", "k_scale", "v_scale", "row_pos")]


class FlbKv8Append(C.Structure):
    """struct flb_kv8_append_params, field for field."""

    _fields_ = [
        ("cache", FlbKv8Cache), ("seq_len", C.c_int), ("start_pos", C.c_int), ("past_lens", C.c_void_p), ("new_lens", C.c_void_p),
        ("token_pos", C.c_void_p), ("input_mode", C.c_int), ("k", C.c_void_p), ("v", C.c_void_p), ("kv_row_stride", C.c_int),
        ("act_scale", C.c_void_p), ("k_w_scale", C.c_void_p), ("v_w_scale", C.c_void_p), ("freq_cis", C.c_void_p), ("freq_rows", C.c_int),
        ("status", C.c_void_p),
    ]


class FlbKv8Decode(C.Structure):
    """struct flb_kv8_decode_params, field for field."""

    _fields_ = [
        ("cache", FlbKv8Cache), ("head_num", C.c_int), ("start_pos", C.c_int), ("past_lens", C.c_void_p), ("max_past_len", C.c_int),
        ("token_pos", C.c_void_p), ("input_mode", C.c_int), ("q", C.c_void_p), ("k", C.c_void_p), ("v", C.c_void_p), ("q_row_stride", C.c_int),
        ("kv_row_stride", C.c_int), ("act_scale", C.c_void_p), ("q_w_scale", C.c_void_p), ("k_w_scale", C.c_void_p), ("v_w_scale", C.c_void_p),
        ("freq_cis", C.c_void_p), ("freq_rows", C.c_int), ("softmax_scale", C.c_float), ("softcap", C.c_float), ("alibi_slopes", C.c_void_p),
        ("key_begin", C.c_void_p), ("weight_in", C.c_void_p), ("weight_out", C.c_void_p), ("out", C.c_void_p), ("out_dtype", C.c_int),
        ("scratch", C.c_void_p), ("scratch_bytes", C.c_size_t), ("scratch_zeroed", C.c_int), ("split_len", C.c_int),
    ]


class FlbKv8Evict(C.Structure):
    """struct flb_kv8_evict_params, field for field."""

    _fields_ = [
        ("cache", FlbKv8Cache), ("start_pos", C.c_int), ("past_lens", C.c_void_p), ("len_out", C.c_void_p), ("budget", C.c_int),
        ("recent", C.c_int), ("sinks", C.c_int), ("next_pos", C.c_void_p), ("weight", C.c_void_p), ("weight_out", C.c_void_p),
        ("pos_out", C.c_void_p), ("scratch", C.c_void_p), ("scratch_bytes", C.c_size_t),
    ]


# every symbol include/flb_kv8.h declares: name -> (restype, argtypes)
_SIZE = C.POINTER(C.c_size_t)
EXPORTS = {
    "flb_kv8_validate_append": (C.c_int, [C.POINTER(FlbKv8Append)]),
    "flb_kv8_validate_decode": (C.c_int, [C.POINTER(FlbKv8Decode)]),
    "flb_kv8_validate_evict": (C.c_int, [C.POINTER(FlbKv8Evict)]),
    "flb_kv8_decode_workspace_bytes": (C.c_int, [C.POINTER(FlbKv8Decode), _SIZE]),
    "flb_kv8_counter_bytes": (C.c_int, [C.POINTER(FlbKv8Decode), _SIZE]),
    "flb_kv8_evict_workspace_bytes": (C.c_int, [C.POINTER(FlbKv8Evict), _SIZE]),
    "flb_kv8_append": (C.c_int, [C.c_void_p, C.c_void_p]),  # a parameter block, by reference or as its bytes
    "flb_kv8_decode": (C.c_int, [C.c_void_p, C.c_void_p]),
    "flb_kv8_evict": (C.c_int, [C.c_void_p, C.c_void_p]),
}

_typed: C.CDLL | None = None


def load_library() -> C.CDLL:
    """The library with the entry points of flb_kv8.h typed.  Raises if it is absent or lacks one: there is no fallback."""
    global _typed
    lib = _lib.load_library()
    if _typed is not lib:
        for name, (res, args) in EXPORTS.items():
            fn = getattr(lib, name)
            fn.restype, fn.argtypes = res, args
        _typed = lib
    return lib


@dataclass
class Cache:
    """One layer's cache.  k, v: codes [B,Hkv,T,d], int8 or float8_e4m3fn; k_scale, v_scale: float32 [B,Hkv,T/block_len]; row_pos:
    int32 [B,Hkv,T] or None (row r is at position r)."""

    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor
    row_pos: torch.Tensor | None = None

    @property
    def block_len(self) -> int:
        return self.k.shape[2] // self.k_scale.shape[2]

    def tensors(self) -> dict[str, torch.Tensor]:
        t = {"k": self.k, "v": self.v, "k_scale": self.k_scale, "v_scale": self.v_scale}
        if self.row_pos is not None:
            t["row_pos"] = self.row_pos
        return t

    def dequantize(self) -> tuple[torch.Tensor, torch.Tensor]:
        """What the codes stand for, float32 [B,Hkv,T,d] twice (a look at the cache, not a step of the path)."""
        def one(codes, scale):
            B, H, T, d = codes.shape
            n = scale.shape[2]
            return (codes.float().view(B, H, n, T // n, d) * scale[..., None, None]).view(B, H, T, d)

        return one(self.k, self.k_scale), one(self.v, self.v_scale)


def empty_cache(batch_size: int, kv_head_num: int, total_len: int, size_per_head: int, *, block_len: int = 64, dtype=torch.int8,
                row_pos: bool = False, device="cuda") -> Cache:
    """An empty cache; total_len is rounded up to whole blocks.  `row_pos`: keep positions, which eviction needs."""
    n = -(-total_len // block_len)
    shape = (batch_size, kv_head_num, n * block_len, size_per_head)
    codes = [torch.zeros(shape, dtype=torch.int8, device=device).view(dtype) for _ in range(2)]
    scales = [torch.zeros(batch_size, kv_head_num, n, device=device) for _ in range(2)]
    pos = torch.zeros(batch_size, kv_head_num, n * block_len, dtype=torch.int32, device=device) if row_pos else None
    return Cache(*codes, *scales, row_pos=pos)


def _call(fn, block: bytes, dev: int, stream) -> None:
    if dev < 0:
        raise ValueError("the 8-bit cache lives on a CUDA device")
    if torch.cuda.current_device() != dev:
        with torch.cuda.device(dev):
            return _call(fn, block, dev, stream)
    if stream is None:
        h = torch._C._cuda_getCurrentRawStream(dev)
    else:
        h = getattr(stream, "cuda_stream", stream)
    st = fn(block, h)
    if st:
        _lib.check(st)


def _append_block(c: Cache, k, v, *, start_pos: int = 0, past_lens=None, new_lens=None, token_pos=None, act_scale=None, k_w_scale=None,
                  v_w_scale=None, freq_cis=None, scratch=None) -> tuple[bytes, int]:
    """The parameter block as bytes, and the index of the device (-1: host memory, for the checks alone)."""
    return _tensor_args.kv8_append(c.k, c.v, c.k_scale, c.v_scale, c.row_pos, k, v, start_pos, past_lens, new_lens, token_pos, act_scale, k_w_scale,
                                   v_w_scale, freq_cis, scratch)


def append_params(cache: Cache, k, v, **kw) -> FlbKv8Append:
    """The parameter block of `append`."""
    return FlbKv8Append.from_buffer_copy(_append_block(cache, k, v, **kw)[0])


def append(cache: Cache, k, v, *, stream=None, **kw) -> None:
    """Stores the tokens k, v [B,S,Hkv,d] (int32 sums with their scales, float32 or float16) behind the rows each sequence has:
    `past_lens` int32 [B], or `start_pos` for all.  `new_lens` int32 [B]: how many of the S tokens of a padded batch count.
    `token_pos` int32 [B]: position of the first new token, where it is not the cached length.  `freq_cis`: RoPE table, row = position.
    `scratch`: its first word collects error bits (`attention.scratch_status`); may be None."""
    _call(load_library().flb_kv8_append, *_append_block(cache, k, v, **kw), stream)


def _decode_block(c: Cache, q, k, v, out, *, start_pos: int = 0, past_lens=None, max_past_len: int = 0, token_pos=None, act_scale=None,
                  q_w_scale=None, k_w_scale=None, v_w_scale=None, freq_cis=None, softmax_scale: float | None = None, softcap: float = 0.0,
                  alibi_slopes=None, key_begin=None, weight_in=None, weight_out=None, scratch=None, scratch_zeroed: bool = False,
                  split_len: int = 0) -> tuple[bytes, int]:
    return _tensor_args.kv8_decode(c.k, c.v, c.k_scale, c.v_scale, c.row_pos, q, k, v, out, start_pos, past_lens, max_past_len, token_pos, act_scale,
                                   q_w_scale, k_w_scale, v_w_scale, freq_cis, softmax_scale, softcap, alibi_slopes, key_begin, weight_in, weight_out,
                                   scratch, scratch_zeroed, split_len)


def decode_params(cache: Cache, q, k, v, out, **kw) -> FlbKv8Decode:
    """The parameter block of `decode`."""
    return FlbKv8Decode.from_buffer_copy(_decode_block(cache, q, k, v, out, **kw)[0])


def decode(cache: Cache, q, k, v, out, *, stream=None, **kw) -> None:
    """One token per sequence: k, v [B,1,Hkv,d] are stored as by `append`, then q [B,1,H,d] attends over the rows 0..past into out [B,H,1,d].
    H is a multiple of Hkv.  `max_past_len`: host's bound on past_lens (0 = T - 1).  `softcap`: scores become
    softcap * tanh(score / softcap); `alibi_slopes` float32 [H]: minus slope times distance; `key_begin` int32 [B]: rows at an earlier
    position are not seen.  `weight_in`, `weight_out` float32 [B,Hkv,T]: attention weights accumulated over the group (for `evict`), in place
    when both are the same tensor.  `scratch_zeroed`: the first `counter_bytes` bytes of scratch are zero (each call leaves them so)."""
    _call(load_library().flb_kv8_decode, *_decode_block(cache, q, k, v, out, **kw), stream)


def _evict_block(c: Cache, *, len_out, budget: int, weight, start_pos: int = 0, past_lens=None, recent: int = 0, sinks: int = 0, next_pos=None,
                 weight_out=None, pos_out=None, scratch=None) -> tuple[bytes, int]:
    if c.row_pos is None:
        raise ValueError("eviction needs a cache with row_pos")
    return _tensor_args.kv8_evict(c.k, c.v, c.k_scale, c.v_scale, c.row_pos, start_pos, past_lens, len_out, budget, recent, sinks, next_pos, weight,
                                  weight if weight_out is None else weight_out, c.row_pos if pos_out is None else pos_out, scratch)


def evict_params(cache: Cache, **kw) -> FlbKv8Evict:
    """The parameter block of `evict`."""
    return FlbKv8Evict.from_buffer_copy(_evict_block(cache, **kw)[0])


def evict(cache: Cache, *, stream=None, **kw) -> None:
    """Keeps `budget` rows per head of every sequence: those at a position below `sinks` or at or behind next_pos - `recent`, then those of the
    largest accumulated `weight`.  Rows move within the cache, weights and positions along (into weight_out and pos_out, or in place);
    len_out int32 [B] gets min(cached rows, budget) and may be past_lens.  The order of rows is no longer that of positions afterwards."""
    _call(load_library().flb_kv8_evict, *_evict_block(cache, **kw), stream)


def decode_workspace_bytes(batch_size: int, head_num: int, kv_head_num: int, total_len: int, size_per_head: int = 128, *, block_len: int = 64,
                           weights: bool = False, split_len: int = 0) -> int:
    """Scratch of a `decode` call on a full cache of these sizes."""
    p = _sized(batch_size, head_num, kv_head_num, total_len, size_per_head, block_len, weights, split_len)
    n = C.c_size_t(0)
    _lib.check(load_library().flb_kv8_decode_workspace_bytes(C.byref(p), C.byref(n)))
    return n.value


def counter_bytes(batch_size: int, head_num: int, kv_head_num: int, size_per_head: int = 128, *, block_len: int = 64) -> int:
    """Bytes at the start of a `decode` scratch that `scratch_zeroed` speaks of."""
    p = _sized(batch_size, head_num, kv_head_num, block_len, size_per_head, block_len, False, 0)
    n = C.c_size_t(0)
    _lib.check(load_library().flb_kv8_counter_bytes(C.byref(p), C.byref(n)))
    return n.value


def evict_workspace_bytes(batch_size: int, kv_head_num: int, total_len: int, size_per_head: int = 128, *, block_len: int = 64) -> int:
    p = FlbKv8Evict()
    p.cache = FlbKv8Cache(batch_size, kv_head_num, size_per_head, -(-total_len // block_len) * block_len, block_len)
    n = C.c_size_t(0)
    _lib.check(load_library().flb_kv8_evict_workspace_bytes(C.byref(p), C.byref(n)))
    return n.value


def _sized(B, Hq, Hkv, T, d, block_len, weights, split_len) -> FlbKv8Decode:
    p = FlbKv8Decode()
    p.cache = FlbKv8Cache(B, Hkv, d, -(-T // block_len) * block_len, block_len)
    p.head_num, p.split_len, p.weight_out = Hq, split_len, (16 if weights else None)
    return p


def validate(p: Any) -> int:
    """Status of the host-side checks of a parameter block (no CUDA call)."""
    lib = load_library()
    fn = {FlbKv8Append: lib.flb_kv8_validate_append, FlbKv8Decode: lib.flb_kv8_validate_decode, FlbKv8Evict: lib.flb_kv8_validate_evict}[type(p)]
    return int(fn(C.byref(p)))
