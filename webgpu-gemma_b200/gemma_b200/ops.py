"""Operators on device memory over torch tensors: the serving step around a paged 8-bit KV cache.

A step of a scheduler runs them in this order::

    plan = plan_blocks(old_len, new_len, table, free_list, free_count, block_tokens, max_rows)
    q, k = rope(q, k, plan.positions, freqs)
    cache.append(k, v, plan.slots)
    out = cache.attend(q, plan.cu_rows, plan.lens, table, max_rows=..., max_len=...)

Each is one or two kernels of libgemma_b200.so on the current stream of the tensors' device
(declarations, formulas and limits: include/gemma_b200.h). Nothing is synchronised or copied to the host and every call may
be captured into a CUDA graph. Shapes, types and devices are checked here (ValueError); lengths,
slots and block ids live on the device and are bounds-checked by the kernels. No operator records
gradients: tensors that require one are refused while grad mode is on, and so are dual tensors of
forward-mode differentiation. The gradient of ``rope`` is
``rope(..., inverse=True)`` of the outputs' gradients.
"""
from __future__ import annotations

import ctypes
import struct
from functools import lru_cache
from typing import NamedTuple

import torch
from torch.autograd import forward_ad

from . import native
from .native import GG_OK, GemmaB200Error, GGKv8AttentionCall, GGKv8Cache, GGRows

_TYPES = {torch.float32: native.GG_T_F32, torch.bfloat16: native.GG_T_BF16, torch.float16: native.GG_T_F16}
_CODES = {torch.int8: native.GG_KV8_INT8, torch.float8_e4m3fn: native.GG_KV8_E4M3}
_LAYOUTS = {"half": native.GG_ROPE_HALF, "interleaved": native.GG_ROPE_INTERLEAVED}
_SCALINGS = {"none": native.GG_ROPE_NONE, "linear": native.GG_ROPE_LINEAR, "bands": native.GG_ROPE_BANDS,
             "yarn": native.GG_ROPE_YARN}

# A call of a few microseconds is made of host work as much as of the kernel, so the argument
# structures of include/gemma_b200.h (native.GGRopeCall and its like) are packed here in one step
# each and handed over as bytes: a third of the time that filling ctypes structures takes.
_ROWS = "Pqqii"
_pack_plan = struct.Struct("@PPPq" + "P" * 9 + "iiiiixxxx").pack
_pack_rope = struct.Struct("@" + _ROWS * 4 + "PPdiiiiixxxx").pack
_pack_append = struct.Struct("@" + _ROWS * 2 + "Pixxxx").pack
_pack_attend = struct.Struct("@" + _ROWS * 2 + "PPPPqPNdiiiiixxxx").pack
_NO_ROWS = (0, 0, 0, 0, 0)

_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)
_lib = None


def _library():
    global _lib
    if _lib is None:
        _lib = native.load()
    return _lib


def _check(rc: int):
    if rc != GG_OK:
        raise GemmaB200Error(rc, _library().gg_last_error(None).decode())


def _call(index: int, fn, *args):
    """fn(*args, stream) with device `index` current, on its current stream."""
    if torch.cuda.current_device() != index:
        with torch.cuda.device(index):
            rc = fn(*args, _raw_stream(index))
    else:
        rc = fn(*args, _raw_stream(index))
    if rc != GG_OK:
        _check(rc)


def _gpu_index(name: str, t: torch.Tensor) -> int:
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor, not on {t.device}")
    return t.get_device()


def _elsewhere(name: str, t: torch.Tensor, index: int):
    _gpu_index(name, t)
    raise ValueError(f"{name} is on {t.device}, the other tensors on cuda:{index}")


def _no_gradient(name: str, t: torch.Tensor):
    """Refuses what autograd would follow: in reverse mode, or as a dual tensor in forward mode."""
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} requires a gradient, which this operator does not record")
    if forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None:
        raise ValueError(f"{name} carries a tangent, which this operator does not propagate")


def _int32(name: str, value: int):
    """Sizes travel as 32 bits: neither struct nor ctypes may see one that does not fit."""
    if not -(1 << 31) <= value < 1 << 31:
        raise ValueError(f"{name} {value} does not fit 32 bits")


def _rows(name: str, t: torch.Tensor, index: int) -> tuple:
    """gg_rows of a [rows][heads][head_dim] tensor of any strides with contiguous heads."""
    stride = t.stride()
    if len(stride) != 3:
        raise ValueError(f"{name} must be [rows][heads][head_dim], not {tuple(t.shape)}")
    type_ = _TYPES.get(t.dtype)
    if type_ is None:
        raise ValueError(f"{name} must be float32, bfloat16 or float16, not {t.dtype}")
    if t.get_device() != index:
        _elsewhere(name, t, index)
    if t.requires_grad or forward_ad._current_level >= 0:
        _no_gradient(name, t)
    shape = t.shape
    if stride[2] != 1 and shape[2] > 1:
        raise ValueError(f"the values of a head of {name} must be contiguous (stride {stride[2]})")
    # a data pointer of an empty tensor is null; no row of it is read
    return t.data_ptr() or 16, stride[0], stride[1], shape[1], type_


def _ints(name: str, t: torch.Tensor, index: int, numel: int) -> int:
    if t.dtype != torch.int32:
        raise ValueError(f"{name} must be int32, not {t.dtype}")
    if t.get_device() != index:
        _elsewhere(name, t, index)
    if t.shape != (numel,):
        raise ValueError(f"{name} has shape {tuple(t.shape)}, ({numel},) needed")
    if numel > 1 and t.stride() != (1,):
        raise ValueError(f"{name} must be contiguous")
    return t.data_ptr() or 16


def _table(t: torch.Tensor, index: int, seqs: int) -> tuple:
    """(pointer, row stride, blocks of a row)"""
    shape, stride = t.shape, t.stride()
    if t.dtype != torch.int32 or len(shape) != 2 or (stride[1] != 1 and shape[1] > 1):
        raise ValueError(f"table must be an int32 [requests][blocks] tensor with contiguous rows, not {t.dtype} {tuple(shape)}")
    if t.get_device() != index:
        _elsewhere("table", t, index)
    if shape[0] != seqs:
        raise ValueError(f"table has {shape[0]} rows for {seqs} requests")
    if shape[0] > 1 and stride[0] < shape[1]:
        raise ValueError("the rows of table overlap")
    return t.data_ptr() or 16, max(stride[0], shape[1]), shape[1]


class BlockPlan(NamedTuple):
    """What ``plan_blocks`` computes; all int32 on the GPU. ``status`` is 0 or a sum of native.GG_PLAN_*."""

    cu_rows: torch.Tensor     # [requests + 1]
    lens: torch.Tensor        # [requests]
    row_seq: torch.Tensor     # [rows], -1 behind the last new token
    positions: torch.Tensor   # [rows], -1
    slots: torch.Tensor       # [rows], -1
    free_count: torch.Tensor  # [1]
    status: torch.Tensor      # [1]


def plan_blocks(old_len: torch.Tensor, new_len: torch.Tensor, table: torch.Tensor, free_list: torch.Tensor,
                free_count: torch.Tensor, block_tokens: int, rows: int, out: BlockPlan | None = None) -> BlockPlan:
    """Block table, free stack and the rows of a step in which request i goes from ``old_len[i]`` to
    ``new_len[i]`` tokens (gg_plan_blocks). ``table`` and ``free_list`` are updated in place;
    ``free_count`` only if it is also ``out.free_count``. ``rows`` is the size of the row arrays.
    A plan that does not fit changes nothing and says so in ``status``."""
    dev = _gpu_index("old_len", old_len)
    n = old_len.shape[0] if old_len.dim() else 0
    _int32("rows", rows)
    _int32("block_tokens", block_tokens)
    if out is None:
        if rows < 0:
            raise ValueError(f"rows must not be negative, not {rows}")
        flat = torch.empty(2 * n + 3 + 3 * rows, dtype=torch.int32, device=old_len.device)
        # integers, which autograd never sees: views without its bookkeeping (a microsecond less)
        out = BlockPlan(*flat.unsafe_split_with_sizes((n + 1, n, rows, rows, rows, 1, 1)))
        p = flat.data_ptr()
        q = p + 4 * (2 * n + 1)
        outs = (p, p + 4 * (n + 1), q, q + 4 * rows, q + 8 * rows, q + 12 * rows, q + 12 * rows + 4)
    else:
        outs = tuple(_ints("out." + name, t, dev, k) for name, t, k in zip(out._fields, out, (n + 1, n, rows, rows, rows, 1, 1)))
    tp, stride, blocks = _table(table, dev, n)
    free = free_list.shape[0] if free_list.dim() else 0
    _call(dev, _library().gg_plan_blocks,
          _pack_plan(_ints("old_len", old_len, dev, n), _ints("new_len", new_len, dev, n), tp, stride, _ints("free_list", free_list, dev, free),
                     _ints("free_count", free_count, dev, 1), *outs, n, blocks, block_tokens, free, rows))
    return out


def rope_frequencies(rot_dim: int, theta: float, scaling: str = "none", factor: float = 1.0, trained: float = 8192.0,
                     low: float = 1.0, high: float = 4.0, device="cuda") -> tuple[torch.Tensor, float]:
    """(freqs, mscale) for ``rope``: radians per position of each pair, float64 on `device`, and the
    factor on cos and sin (gg_rope_freqs gives the formulas). scaling: "none", "linear" (Gemma 3's
    global layers from 4B on: factor 8), "bands" (low 1, high 4 usually) or "yarn" (low 1, high 32)."""
    if scaling not in _SCALINGS:
        raise ValueError(f"unknown scaling {scaling!r} (one of {', '.join(_SCALINGS)})")
    f = torch.empty(max(rot_dim // 2, 1), dtype=torch.float64)
    m = ctypes.c_double()
    _check(native.load().gg_rope_freqs(_SCALINGS[scaling], rot_dim, theta, factor, trained, low, high, f.data_ptr(), ctypes.byref(m)))
    return f.to(device), m.value


def rope(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, freqs: torch.Tensor, layout: str = "half",
         mscale: float = 1.0, inverse: bool = False, out: tuple | None = None):
    """Rotary positions on q [rows][heads][head_dim] and k (or None) in one kernel (gg_rope); rotates
    the first 2 * len(freqs) values of each head. Returns (q, k) as new tensors, or ``out``, which may
    be (q, k) itself. A row at a negative position is copied."""
    dev = _gpu_index("q", q)
    code = _LAYOUTS.get(layout)
    if code is None:
        raise ValueError(f"unknown layout {layout!r} (half or interleaved)")
    pairs = freqs.shape[0] if freqs.dim() == 1 else 0
    if freqs.dtype != torch.float64 or not pairs or (pairs > 1 and freqs.stride(0) != 1):
        raise ValueError("freqs must be a contiguous float64 vector (rope_frequencies)")
    if freqs.get_device() != dev:
        _elsewhere("freqs", freqs, dev)
    if freqs.requires_grad or forward_ad._current_level >= 0:
        _no_gradient("freqs", freqs)
    vq = _rows("q", q, dev)
    n, _, dim = q.shape
    vk = wk = _NO_ROWS
    if k is not None:
        vk = _rows("k", k, dev)
        if k.shape[0] != n or k.shape[2] != dim or vk[4] != vq[4]:
            raise ValueError(f"q {tuple(q.shape)} {q.dtype} and k {tuple(k.shape)} {k.dtype} differ in rows, head_dim or type")
    if out is None:
        oq = torch.empty_like(q, memory_format=torch.contiguous_format)
        wq = (oq.data_ptr() or 16, vq[3] * dim, dim, vq[3], vq[4])
        ok = None
        if k is not None:
            ok = torch.empty_like(k, memory_format=torch.contiguous_format)
            wk = (ok.data_ptr() or 16, vk[3] * dim, dim, vk[3], vk[4])
    else:
        oq, ok = out
        if oq.shape != q.shape or (k is None) != (ok is None) or (k is not None and ok.shape != k.shape):
            raise ValueError("out must be (q, k) of the same shapes")
        wq = _rows("out[0]", oq, dev)
        if ok is not None:
            wk = _rows("out[1]", ok, dev)
    _call(dev, _library().gg_rope,
          _pack_rope(*vq, *vk, *wq, *wk, _ints("positions", positions, dev, n), freqs.data_ptr(), mscale, n, dim, 2 * pairs, code,
                     1 if inverse else 0))
    return oq, ok


@lru_cache(maxsize=1024)
def _attend_bytes(num_blocks, block_tokens, kv_heads, head_dim, code, heads, type_, seqs, rows, max_rows, max_len, window) -> int:
    """Workspace of a call of these sizes (a pure function of them)."""
    for name, value in (("requests", seqs), ("rows", rows), ("max_rows", max_rows), ("max_len", max_len), ("window", window)):
        _int32(name, value)
    c = GGKv8Cache(16, 16, 16, 16, num_blocks, block_tokens, kv_heads, head_dim, code)
    call = GGKv8AttentionCall(q=GGRows(heads=heads, type=type_), seqs=seqs, rows=rows, max_rows=max_rows, max_len=max_len, window=window)
    need = ctypes.c_size_t()
    _check(_library().gg_kv8_attention_workspace(ctypes.byref(c), ctypes.byref(call), ctypes.byref(need)))
    return need.value


class KV8Cache:
    """A paged KV cache in 8 bits over tensors the caller owns: codes [blocks][kv_heads][block_tokens]
    [head_dim] (int8 or float8_e4m3fn) and scales [blocks][kv_heads] (float32), for K and for V."""

    def __init__(self, k_codes: torch.Tensor, v_codes: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor):
        dev = _gpu_index("k_codes", k_codes)
        if k_codes.dim() != 4 or k_codes.dtype not in _CODES:
            raise ValueError(f"codes must be int8 or float8_e4m3fn [blocks][kv_heads][block_tokens][head_dim], not {k_codes.dtype} {tuple(k_codes.shape)}")
        if v_codes.shape != k_codes.shape or v_codes.dtype != k_codes.dtype:
            raise ValueError("k_codes and v_codes differ in shape or type")
        for name, t in (("k_scale", k_scale), ("v_scale", v_scale)):
            if t.dtype != torch.float32 or t.shape != k_codes.shape[:2]:
                raise ValueError(f"{name} must be float32 {tuple(k_codes.shape[:2])}, not {t.dtype} {tuple(t.shape)}")
        for name, t in (("k_codes", k_codes), ("v_codes", v_codes), ("k_scale", k_scale), ("v_scale", v_scale)):
            if t.get_device() != dev:
                _elsewhere(name, t, dev)
            if not t.is_contiguous():
                raise ValueError(f"{name} must be contiguous")
        self.k_codes, self.v_codes, self.k_scale, self.v_scale = k_codes, v_codes, k_scale, v_scale
        self.device = k_codes.device
        self._index = dev
        self.num_blocks, self.kv_heads, self.block_tokens, self.head_dim = k_codes.shape
        self._sizes = (self.num_blocks, self.block_tokens, self.kv_heads, self.head_dim, _CODES[k_codes.dtype])
        self._c = bytes(GGKv8Cache(k_codes.data_ptr(), v_codes.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), *self._sizes))

    @classmethod
    def empty(cls, num_blocks: int, block_tokens: int, kv_heads: int, head_dim: int, code: str = "int8", device="cuda") -> "KV8Cache":
        """A cache of zeros; code is "int8" or "e4m3"."""
        if code not in ("int8", "e4m3"):
            raise ValueError(f"unknown code {code!r} (int8 or e4m3)")
        shape = (num_blocks, kv_heads, block_tokens, head_dim)
        raw = [torch.zeros(shape, dtype=torch.int8, device=device) for _ in range(2)]
        if code == "e4m3":
            raw = [t.view(torch.float8_e4m3fn) for t in raw]
        return cls(*raw, *(torch.ones(shape[:2], dtype=torch.float32, device=device) for _ in range(2)))

    def append(self, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
        """Quantises k and v [rows][kv_heads][head_dim] into ``slots`` (-1: no slot), as gg_kv8_append."""
        dev = self._index
        vk, vv = _rows("k", k, dev), _rows("v", v, dev)
        shape = k.shape
        if shape[2] != self.head_dim or v.shape[2] != self.head_dim or v.shape[0] != shape[0]:
            raise ValueError(f"k and v must be [rows][{self.kv_heads}][{self.head_dim}], not {tuple(shape)} and {tuple(v.shape)}")
        n = shape[0]
        _call(dev, _library().gg_kv8_append, self._c, _pack_append(*vk, *vv, _ints("slots", slots, dev, n), n))

    def attend(self, q: torch.Tensor, cu_rows: torch.Tensor, lens: torch.Tensor, table: torch.Tensor, *, max_rows: int, max_len: int,
               scale: float | None = None, window: int = 0, out: torch.Tensor | None = None, return_lse: bool = False,
               workspace: torch.Tensor | None = None):
        """Attention of q [rows][heads][head_dim] over the cached tokens of each row's request
        (gg_kv8_attention): rows cu_rows[i] .. cu_rows[i + 1] - 1 are the last tokens of request i.
        ``scale`` defaults to head_dim^-0.5. Returns out, or (out, lse) with the rows' f32 log-sum-exp.
        Rows behind the last request are not written (a new ``out`` holds anything there). Without a
        ``workspace`` (uint8) the call takes one from torch's allocator."""
        dev = self._index
        vq = _rows("q", q, dev)
        rows, heads, dim = shape = q.shape
        if dim != self.head_dim:
            raise ValueError(f"q has head_dim {dim}, the cache {self.head_dim}")
        if out is None:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
            vo = (out.data_ptr() or 16, heads * dim, dim, heads, vq[4])
        else:
            if out.shape != shape:
                raise ValueError(f"out is {tuple(out.shape)}, q {tuple(shape)}")
            vo = _rows("out", out, dev)
        n = lens.shape[0] if lens.dim() else 0
        tp, stride, blocks = _table(table, dev, n)
        if max_len > blocks * self.block_tokens:
            raise ValueError(f"max_len {max_len} is more than a table row of {blocks} blocks holds")
        need = _attend_bytes(*self._sizes, heads, vq[4], n, rows, max_rows, max_len, window)
        wp = size = 0
        if workspace is not None:
            if workspace.dtype != torch.uint8 or workspace.dim() != 1 or not workspace.is_contiguous():
                raise ValueError("workspace must be a contiguous uint8 vector")
            if workspace.get_device() != dev:
                _elsewhere("workspace", workspace, dev)
            wp, size = workspace.data_ptr(), workspace.numel()
        elif need:
            workspace = torch.empty(need, dtype=torch.uint8, device=self.device)
            wp, size = workspace.data_ptr(), need
        lse = torch.empty(rows, heads, dtype=torch.float32, device=self.device) if return_lse else None
        _call(dev, _library().gg_kv8_attention, self._c,
              _pack_attend(*vq, *vo, lse.data_ptr() if lse is not None else 0, _ints("cu_rows", cu_rows, dev, n + 1), _ints("lens", lens, dev, n),
                           tp, stride, wp, size, dim ** -0.5 if scale is None else scale, n, rows, max_rows, max_len, window))
        return (out, lse) if return_lse else out

    def workspace_bytes(self, q: torch.Tensor, seqs: int, max_rows: int, max_len: int, window: int = 0) -> int:
        """Bytes of ``workspace`` that ``attend`` needs for such a batch."""
        vq = _rows("q", q, self._index)
        return _attend_bytes(*self._sizes, vq[3], vq[4], seqs, q.shape[0], max_rows, max_len, window)
