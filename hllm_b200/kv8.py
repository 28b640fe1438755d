"""The 8-bit paged KV cache on torch tensors: a cache of half the F16 pages'
bytes, its write, its read-back and the attention that reads it.

The calls are those of include/hllm_b200.h (``hllm_b200_kv8_*``), checked
against the tensors they are given, on the tensors' device and its current
torch stream.  A step of a decoder layer is

    q = kv8.write(cache, qkv, positions, slots, rope, q_norm=..., k_norm=...)
    o = kv8.attention(cache, q, cu_seqlens, lengths, block_tables, max_tokens=...)

with positions, slots, cu_seqlens, lengths and block tables as the packer
(``hllm_b200_pack``) makes them; ``kv8.read`` gives cached rows back.  Nothing
waits for the GPU: slots, blocks or rows out of range are skipped and set bits
in ``cache.status``, which ``cache.check()`` reads.  The calls can be captured
into CUDA graphs.  Calls that run at the same time (on several streams, or in
graphs replayed side by side) each need a workspace of their own.
"""
from __future__ import annotations

import ctypes as C
import math
from typing import Optional

import torch

from . import _lib
from ._lib import StageError, lib

__all__ = ["Cache", "Rope", "write", "read", "attention", "attention_workspace", "PAGE"]

PAGE = 16
_TYPES = {torch.float32: _lib.F32, torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}
_SCALINGS = {"none": 0, "linear": 1, "llama3": 2, "yarn": 3}
#: Status bits of the device word (DeviceStatus in csrc/common.cuh).
_BITS = {1: "a device wait ran out", 4: "a slot, block or row out of range"}


def _refuse(message: str):
    raise StageError(_lib.INVALID_REQUEST, message)


def _need(tensor, name: str, dtype, index: int, shape=None, optional=False):
    """Checks one tensor and returns its address (None for a missing optional one)."""
    if tensor is None and optional:
        return None
    if (isinstance(tensor, torch.Tensor) and tensor.dtype is dtype and tensor.get_device() == index
            and tensor.is_contiguous() and (shape is None or tensor.shape == shape)):
        return tensor.data_ptr()
    if not isinstance(tensor, torch.Tensor):
        _refuse(f"{name} must be a tensor")
    if tensor.dtype != dtype:
        _refuse(f"{name} must be {dtype}, not {tensor.dtype}")
    if tensor.get_device() != index:
        _refuse(f"{name} is on {tensor.device}, the cache on cuda:{index}")
    if shape is not None and tensor.shape != shape:
        _refuse(f"{name} must have shape {tuple(shape)}, not {tuple(tensor.shape)}")
    _refuse(f"{name} must be contiguous")


# The device and stream that torch has current, without the objects around them
# (3 us less host time a call).
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
_current_stream = getattr(torch._C, "_cuda_getCurrentRawStream",
                          lambda index: torch.cuda.current_stream(index).cuda_stream)


def _call(name: str, index: int, *args) -> None:
    """One library call with device `index` current, on its current stream (the last argument)."""
    function = _functions.get(name)
    if function is None:
        function = _functions[name] = getattr(lib(), name)
    if _current_device() == index:
        status = function(*args, _current_stream(index))
    else:
        with torch.cuda.device(index):
            status = function(*args, _current_stream(index))
    if status:
        _lib.check(status)


_functions: dict = {}


class Cache:
    """Codes (float8_e4m3fn [blocks, kv_heads, 16, head_dim]) and scales
    (float8_e8m0fnu [blocks, kv_heads, 16]) of K and V: ``k``, ``k_scale``,
    ``v``, ``v_scale``; ``status`` is the device word that calls report to."""

    def __init__(self, blocks: int, kv_heads: int, head_dim: int, device="cuda"):
        def codes():
            return torch.zeros((blocks, kv_heads, PAGE, head_dim), dtype=torch.uint8, device=device)

        def scales():
            return torch.full((blocks, kv_heads, PAGE), 127, dtype=torch.uint8, device=device)
        self._take(codes(), scales(), codes(), scales())

    @classmethod
    def wrap(cls, k, k_scale, v, v_scale) -> "Cache":
        """A cache on four tensors that the caller keeps (8-bit types, contiguous)."""
        self = cls.__new__(cls)
        self._take(k, k_scale, v, v_scale)
        return self

    def _take(self, k, k_scale, v, v_scale):
        if not all(isinstance(t, torch.Tensor) for t in (k, k_scale, v, v_scale)):
            _refuse("a cache is made of four tensors")
        if k.dim() != 4 or k.shape[2] != PAGE:
            _refuse(f"codes must be [blocks, kv_heads, {PAGE}, head_dim], not {tuple(k.shape)}")
        if not k.is_cuda:
            _refuse(f"the cache must be on a CUDA device, not {k.device}")
        for t, name, kinds, shape in (
                (k, "k", (torch.uint8, torch.float8_e4m3fn), k.shape),
                (v, "v", (torch.uint8, torch.float8_e4m3fn), k.shape),
                (k_scale, "k_scale", (torch.uint8, torch.float8_e8m0fnu), k.shape[:3]),
                (v_scale, "v_scale", (torch.uint8, torch.float8_e8m0fnu), k.shape[:3])):
            if t.dtype not in kinds:
                _refuse(f"{name} must be one of {kinds}, not {t.dtype}")
            _need(t, name, t.dtype, k.get_device(), shape)
        self.k, self.v = k.view(torch.float8_e4m3fn), v.view(torch.float8_e4m3fn)
        self.k_scale = k_scale.view(torch.float8_e8m0fnu)
        self.v_scale = v_scale.view(torch.float8_e8m0fnu)
        self.blocks, self.kv_heads, _, self.head_dim = k.shape
        self.device, self._index = k.device, k.get_device()
        self.status = torch.zeros(1, dtype=torch.int32, device=k.device)
        self._status = self.status.data_ptr()
        self._c = _lib.KV8(k.data_ptr(), k_scale.data_ptr(), v.data_ptr(), v_scale.data_ptr(),
                           self.blocks, self.kv_heads, self.head_dim)
        self._ref = C.byref(self._c)

    def check(self) -> None:
        """Waits for the device word on the current stream, clears it, and raises
        what it reports of the calls that this stream has waited for."""
        bits = int(self.status.item())
        if bits:
            self.status.zero_()
            what = [text for bit, text in _BITS.items() if bits & bit] or [f"status {bits:#x}"]
            raise StageError(_lib.INTERNAL, "8-bit KV cache: " + ", ".join(what))


class Rope:
    """How positions turn a head's pairs (``hllm_b200_rope``), with its table
    on a device.  ``scaling`` is None or a dict with "type" ("linear",
    "llama3" or "yarn"), "factor", and what the type takes: "low_freq_factor",
    "high_freq_factor"; "beta_fast", "beta_slow"; "original_max_position".
    ``attention_factor`` scales cos and sin (default: the scaling's own)."""

    def __init__(self, head_dim: int, theta: float, rotary_dim: Optional[int] = None,
                 interleaved: bool = False, scaling: Optional[dict] = None,
                 attention_factor: Optional[float] = None, device="cuda"):
        self.rotary_dim = head_dim if rotary_dim is None else int(rotary_dim)
        if not 0 < self.rotary_dim <= head_dim or self.rotary_dim % 2:
            _refuse(f"rotary_dim must be even and 2 to {head_dim}")
        s = dict(scaling or {"type": "none"})
        kind = s.pop("type", None)
        if kind not in _SCALINGS:
            _refuse(f"unknown rope scaling {kind!r}")
        known = {"factor": 1.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
                 "beta_fast": 32.0, "beta_slow": 1.0, "original_max_position": 0.0}
        if set(s) - set(known):
            _refuse(f"unknown rope scaling options {sorted(set(s) - set(known))}")
        v = {**known, **s}
        self.interleaved = bool(interleaved)
        desc = _lib.Rope(self.rotary_dim, int(self.interleaved), theta, _SCALINGS[kind], v["factor"],
                         v["low_freq_factor"], v["high_freq_factor"], v["beta_fast"],
                         v["beta_slow"], v["original_max_position"],
                         0.0 if attention_factor is None else attention_factor)
        turns = (C.c_double * (self.rotary_dim // 2))()
        factor = C.c_float()
        _lib.check(lib().hllm_b200_rope_turns(C.byref(desc), turns, C.byref(factor)))
        self.factor = factor.value
        self.turns = torch.tensor(list(turns), dtype=torch.float64).to(device)
        self._index, self._turns = self.turns.get_device(), self.turns.data_ptr()


def write(cache: Cache, qkv, positions, slots, rope: Rope, q_norm=None, k_norm=None,
          eps: float = 1e-6, out=None):
    """q/k RMSNorm (where weights are given), rotary positions and the
    quantised write of K and V: qkv [tokens, (heads + 2 kv_heads) head_dim]
    (float32, float16 or bfloat16), int32 positions and slots [tokens] (slot
    -1: not stored; the slots of a call are distinct).  Returns q, float16
    [tokens, heads * head_dim]."""
    index, d = cache._index, cache.head_dim
    if not isinstance(qkv, torch.Tensor) or qkv.dtype not in _TYPES or qkv.dim() != 2:
        _refuse("qkv must be a float32, float16 or bfloat16 matrix")
    tokens, width = qkv.shape
    hq = width // d - 2 * cache.kv_heads
    if width % d or hq <= 0:
        _refuse(f"qkv rows of {width} are not (heads + 2 x {cache.kv_heads}) x {d}")
    if rope.rotary_dim > d:
        _refuse(f"rope turns {rope.rotary_dim} of a head of {d}")
    x = _need(qkv, "qkv", qkv.dtype, index)
    p = _need(positions, "positions", torch.int32, index, (tokens,))
    s = _need(slots, "slots", torch.int32, index, (tokens,))
    qn = _need(q_norm, "q_norm", torch.float32, index, (d,), optional=True)
    kn = _need(k_norm, "k_norm", torch.float32, index, (d,), optional=True)
    if rope._index != index:
        _refuse(f"rope's table is on {rope.turns.device}, the cache on {cache.device}")
    if out is None:
        out = qkv.new_empty((tokens, hq * d), dtype=torch.float16)
        o = out.data_ptr()
    else:
        o = _need(out, "out", torch.float16, index, (tokens, hq * d))
    _call("hllm_b200_kv8_write", index, cache._ref, x, _TYPES[qkv.dtype], tokens, hq, p, s, qn,
          kn, eps, rope._turns, rope.rotary_dim, rope.interleaved, rope.factor, o, cache._status)
    return out


def read(cache: Cache, block_tables, lengths, offsets, tokens: int, first=None,
         dtype=torch.float16, out=None):
    """Cached rows as values of `dtype`: row r's positions [first[r],
    lengths[r]) go to rows [offsets[r], offsets[r + 1]) of k and v [tokens,
    kv_heads, head_dim] (int32 tensors; first None: 0).  Returns (k, v); `out`
    is such a pair to fill, whose rows from offsets[-1] on are left alone."""
    index = cache._index
    if dtype not in _TYPES:
        _refuse("dtype must be float32, float16 or bfloat16")
    if not isinstance(block_tables, torch.Tensor) or block_tables.dim() != 2:
        _refuse("block_tables must be [rows, most pages]")
    rows, width = block_tables.shape
    t = _need(block_tables, "block_tables", torch.int32, index)
    n = _need(lengths, "lengths", torch.int32, index, (rows,))
    f = _need(first, "first", torch.int32, index, (rows,), optional=True)
    c = _need(offsets, "offsets", torch.int32, index, (rows + 1,))
    shape = (tokens, cache.kv_heads, cache.head_dim)
    if out is None:
        values = cache.k.new_empty(shape, dtype=dtype)
        out = (values, torch.empty_like(values))
        k, v = values.data_ptr(), out[1].data_ptr()
    else:
        k, v = (_need(x, name, dtype, index, shape) for x, name in zip(out, ("k", "v")))
    _call("hllm_b200_kv8_read", index, cache._ref, t, rows, width, f, n, c, tokens,
          _TYPES[dtype], k, v, cache._status)
    return out


def attention_workspace(rows: int, tokens: int, max_tokens: int, heads: int, kv_heads: int,
                        head_dim: int, device="cuda"):
    """A workspace for ``attention`` calls of at most these counts, one after
    another (calls that run at the same time need one each)."""
    n = C.c_uint64()
    with torch.cuda.device(device):
        _lib.check(lib().hllm_b200_kv8_attention_workspace(rows, tokens, max_tokens, heads, kv_heads,
                                                           head_dim, C.byref(n)))
        return torch.empty(n.value, dtype=torch.uint8, device=device)


def attention(cache: Cache, q, cu_seqlens, lengths, block_tables, max_tokens: Optional[int] = None,
              scale: Optional[float] = None, out=None, workspace=None):
    """Causal attention of each row's new tokens over its cached keys: q
    float16 [tokens, heads * head_dim] (rows may be strided), row r's tokens
    being rows [cu_seqlens[r], cu_seqlens[r + 1]) at the last positions of its
    lengths[r] keys; int32 block_tables [rows, most pages].  ``max_tokens`` is
    the most new tokens of a row (default: tokens; 1 for a decode batch),
    ``scale`` defaults to 1/sqrt(head_dim).  Returns float16 like q."""
    index, d = cache._index, cache.head_dim
    if not isinstance(q, torch.Tensor) or q.dim() != 2 or q.dtype != torch.float16:
        _refuse("q must be a float16 matrix")
    tokens, width = q.shape
    hq = width // d
    if width % d or hq == 0 or hq % cache.kv_heads:
        _refuse(f"q rows of {width} are not heads x {d}, a multiple of {cache.kv_heads} heads")
    if q.get_device() != index:
        _refuse(f"q is on {q.device}, the cache on {cache.device}")
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
    elif (not isinstance(out, torch.Tensor) or out.dtype != torch.float16
          or out.get_device() != index or out.shape != (tokens, width)):
        _refuse(f"out must be a float16 {(tokens, width)} matrix on {cache.device}")
    ld_q = ld_out = width
    if tokens > 0:
        (step_q, across), (step_out, out_across) = q.stride(), out.stride()
        if tokens > 1:  # (torch leaves the stride of a single row open)
            ld_q, ld_out = step_q, step_out
        if across != 1 or ld_q < width:
            _refuse("q must have contiguous rows")
        if out_across != 1 or ld_out < width:
            _refuse("out must have contiguous rows")
    if not isinstance(block_tables, torch.Tensor) or block_tables.dim() != 2:
        _refuse("block_tables must be [rows, most pages]")
    rows, blocks = block_tables.shape
    t = _need(block_tables, "block_tables", torch.int32, index)
    n = _need(lengths, "lengths", torch.int32, index, (rows,))
    c = _need(cu_seqlens, "cu_seqlens", torch.int32, index, (rows + 1,))
    most = tokens if max_tokens is None else int(max_tokens)
    if most < 0:
        _refuse("max_tokens must not be negative")
    if workspace is None:
        workspace = attention_workspace(rows, tokens, most, hq, cache.kv_heads, d,
                                        cache.device)
    w = _need(workspace, "workspace", torch.uint8, index)
    _call("hllm_b200_kv8_attention", index, cache._ref, q.data_ptr(),
          ld_q, c, n, t, rows, tokens, most, hq, blocks,
          1.0 / math.sqrt(d) if scale is None else scale, out.data_ptr(),
          ld_out, w, workspace.numel(), cache._status)
    return out
