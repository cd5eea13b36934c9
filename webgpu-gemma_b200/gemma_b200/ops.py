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
gradients: tensors that require one are refused while grad mode is on. The gradient of ``rope`` is
``rope(..., inverse=True)`` of the outputs' gradients.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch

from . import native
from .native import GG_OK, GemmaB200Error, GGBlockPlan, GGKv8Batch, GGKv8Cache, GGRows

_TYPES = {torch.float32: native.GG_T_F32, torch.bfloat16: native.GG_T_BF16, torch.float16: native.GG_T_F16}
_CODES = {torch.int8: native.GG_KV8_INT8, torch.float8_e4m3fn: native.GG_KV8_E4M3}
_LAYOUTS = {"half": native.GG_ROPE_HALF, "interleaved": native.GG_ROPE_INTERLEAVED}
_SCALINGS = {"none": native.GG_ROPE_NONE, "linear": native.GG_ROPE_LINEAR, "bands": native.GG_ROPE_BANDS,
             "yarn": native.GG_ROPE_YARN}


def _check(rc: int):
    if rc != GG_OK:
        raise GemmaB200Error(rc, native.load().gg_last_error(None).decode())


def _call(device: torch.device, fn, *args):
    """fn(*args, stream) with `device` current, on its current stream."""
    if torch.cuda.current_device() != device.index:
        with torch.cuda.device(device):
            _check(fn(*args, torch.cuda.current_stream(device).cuda_stream))
    else:
        _check(fn(*args, torch.cuda.current_stream(device).cuda_stream))


def _on_gpu(name: str, t: torch.Tensor, device: torch.device | None = None) -> torch.device:
    if t.device.type != "cuda":
        raise ValueError(f"{name} must be a CUDA tensor, not on {t.device}")
    if device is not None and t.device != device:
        raise ValueError(f"{name} is on {t.device}, the other tensors on {device}")
    return t.device


def _rows(name: str, t: torch.Tensor, device: torch.device) -> GGRows:
    """View of a [rows][heads][head_dim] tensor of any strides with contiguous heads."""
    if t.dim() != 3:
        raise ValueError(f"{name} must be [rows][heads][head_dim], not {tuple(t.shape)}")
    type_ = _TYPES.get(t.dtype)
    if type_ is None:
        raise ValueError(f"{name} must be float32, bfloat16 or float16, not {t.dtype}")
    if t.device != device:
        _on_gpu(name, t, device)
    if t.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"{name} requires a gradient, which this operator does not record")
    sr, sh, sd = t.stride()
    if sd != 1 and t.shape[2] > 1:
        raise ValueError(f"the values of a head of {name} must be contiguous (stride {sd})")
    # a data pointer of an empty tensor is null; no row of it is read
    return GGRows(t.data_ptr() or 16, sr, sh, t.shape[1], type_)


def _ints(name: str, t: torch.Tensor, device: torch.device, numel: int | None = None, at_least: bool = False) -> int:
    if t.dtype != torch.int32:
        raise ValueError(f"{name} must be int32, not {t.dtype}")
    if t.device != device:
        _on_gpu(name, t, device)
    if t.dim() != 1 or (t.stride(0) != 1 and t.shape[0] > 1):
        raise ValueError(f"{name} must be a contiguous 1-D tensor")
    if numel is not None and (t.shape[0] < numel if at_least else t.shape[0] != numel):
        raise ValueError(f"{name} has {t.shape[0]} entries, {'at least ' if at_least else ''}{numel} needed")
    return t.data_ptr() or 16


def _table(t: torch.Tensor, device: torch.device, seqs: int) -> tuple[int, int]:
    if t.dtype != torch.int32 or t.dim() != 2 or (t.stride(1) != 1 and t.shape[1] > 1):
        raise ValueError(f"table must be an int32 [requests][blocks] tensor with contiguous rows, not {t.dtype} {tuple(t.shape)}")
    _on_gpu("table", t, device)
    if t.shape[0] != seqs:
        raise ValueError(f"table has {t.shape[0]} rows for {seqs} requests")
    if t.shape[0] > 1 and t.stride(0) < t.shape[1]:
        raise ValueError("the rows of table overlap")
    return t.data_ptr() or 16, max(t.stride(0), t.shape[1])


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
    dev = _on_gpu("old_len", old_len)
    n = old_len.shape[0] if old_len.dim() else 0
    if out is None:
        flat = torch.empty(2 * n + 3 + 3 * rows, dtype=torch.int32, device=dev)
        a, b = 2 * n + 1, 2 * n + 3
        out = BlockPlan(flat[:n + 1], flat[n + 1:a], flat[b:b + rows], flat[b + rows:b + 2 * rows], flat[b + 2 * rows:],
                        flat[a:a + 1], flat[a + 1:b])
    tp, stride = _table(table, dev, n)
    p = GGBlockPlan(_ints("old_len", old_len, dev, n), _ints("new_len", new_len, dev, n), tp, stride,
                    _ints("free_list", free_list, dev), _ints("free_count", free_count, dev, 1),
                    _ints("out.cu_rows", out.cu_rows, dev, n + 1), _ints("out.lens", out.lens, dev, n),
                    _ints("out.row_seq", out.row_seq, dev, rows), _ints("out.positions", out.positions, dev, rows),
                    _ints("out.slots", out.slots, dev, rows), _ints("out.free_count", out.free_count, dev, 1),
                    _ints("out.status", out.status, dev, 1), n, table.shape[1], block_tokens, free_list.shape[0], rows)
    _call(dev, native.load().gg_plan_blocks, ctypes.byref(p))
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
    dev = _on_gpu("q", q)
    code = _LAYOUTS.get(layout)
    if code is None:
        raise ValueError(f"unknown layout {layout!r} (half or interleaved)")
    if freqs.dtype != torch.float64 or freqs.dim() != 1 or (freqs.shape[0] > 1 and freqs.stride(0) != 1):
        raise ValueError("freqs must be a contiguous float64 vector (rope_frequencies)")
    _on_gpu("freqs", freqs, dev)
    vq = _rows("q", q, dev)
    vk = _rows("k", k, dev) if k is not None else None
    if k is not None and (k.shape[0] != q.shape[0] or k.shape[2] != q.shape[2] or k.dtype != q.dtype):
        raise ValueError(f"q {tuple(q.shape)} {q.dtype} and k {tuple(k.shape)} {k.dtype} differ in rows, head_dim or type")
    if out is None:
        out = (torch.empty(q.shape, dtype=q.dtype, device=dev), None if k is None else torch.empty(k.shape, dtype=k.dtype, device=dev))
    oq, ok = out
    if oq.shape != q.shape or (k is None) != (ok is None) or (k is not None and ok.shape != k.shape):
        raise ValueError("out must be (q, k) of the same shapes")
    wq = _rows("out[0]", oq, dev)
    wk = _rows("out[1]", ok, dev) if ok is not None else None
    ref = ctypes.byref
    _call(dev, native.load().gg_rope, ref(vq), ref(vk) if vk is not None else None, ref(wq), ref(wk) if wk is not None else None,
          q.shape[0], q.shape[2], 2 * freqs.shape[0], code, _ints("positions", positions, dev, q.shape[0]), freqs.data_ptr() or 16,
          mscale, 1 if inverse else 0)
    return oq, ok


class KV8Cache:
    """A paged KV cache in 8 bits over tensors the caller owns: codes [blocks][kv_heads][block_tokens]
    [head_dim] (int8 or float8_e4m3fn) and scales [blocks][kv_heads] (float32), for K and for V."""

    def __init__(self, k_codes: torch.Tensor, v_codes: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor):
        dev = _on_gpu("k_codes", k_codes)
        if k_codes.dim() != 4 or k_codes.dtype not in _CODES:
            raise ValueError(f"codes must be int8 or float8_e4m3fn [blocks][kv_heads][block_tokens][head_dim], not {k_codes.dtype} {tuple(k_codes.shape)}")
        if v_codes.shape != k_codes.shape or v_codes.dtype != k_codes.dtype:
            raise ValueError("k_codes and v_codes differ in shape or type")
        for name, t in (("k_scale", k_scale), ("v_scale", v_scale)):
            if t.dtype != torch.float32 or t.shape != k_codes.shape[:2]:
                raise ValueError(f"{name} must be float32 {tuple(k_codes.shape[:2])}, not {t.dtype} {tuple(t.shape)}")
        for name, t in (("k_codes", k_codes), ("v_codes", v_codes), ("k_scale", k_scale), ("v_scale", v_scale)):
            _on_gpu(name, t, dev)
            if not t.is_contiguous():
                raise ValueError(f"{name} must be contiguous")
        self.k_codes, self.v_codes, self.k_scale, self.v_scale = k_codes, v_codes, k_scale, v_scale
        self.device = dev
        self.num_blocks, self.kv_heads, self.block_tokens, self.head_dim = k_codes.shape
        self._c = GGKv8Cache(k_codes.data_ptr(), v_codes.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), self.num_blocks,
                             self.block_tokens, self.kv_heads, self.head_dim, _CODES[k_codes.dtype])
        self._ref = ctypes.byref(self._c)

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
        dev = self.device
        for name, t in (("k", k), ("v", v)):
            if t.dim() != 3 or t.shape[2] != self.head_dim or t.shape[0] != k.shape[0]:
                raise ValueError(f"{name} must be [rows][{self.kv_heads}][{self.head_dim}], not {tuple(t.shape)}")
        vk, vv = _rows("k", k, dev), _rows("v", v, dev)
        _call(dev, native.load().gg_kv8_append, self._ref, ctypes.byref(vk), ctypes.byref(vv), _ints("slots", slots, dev, k.shape[0]), k.shape[0])

    def attend(self, q: torch.Tensor, cu_rows: torch.Tensor, lens: torch.Tensor, table: torch.Tensor, *, max_rows: int, max_len: int,
               scale: float | None = None, window: int = 0, out: torch.Tensor | None = None, return_lse: bool = False,
               workspace: torch.Tensor | None = None):
        """Attention of q [rows][heads][head_dim] over the cached tokens of each row's request
        (gg_kv8_attention): rows cu_rows[i] .. cu_rows[i + 1] - 1 are the last tokens of request i.
        ``scale`` defaults to head_dim^-0.5. Returns out, or (out, lse) with the rows' f32 log-sum-exp.
        Rows behind the last request are not written (a new ``out`` holds anything there). Without a
        ``workspace`` (uint8) the call takes one from torch's allocator."""
        dev = self.device
        vq = _rows("q", q, dev)
        if q.shape[2] != self.head_dim:
            raise ValueError(f"q has head_dim {q.shape[2]}, the cache {self.head_dim}")
        n, rows = lens.shape[0] if lens.dim() else 0, q.shape[0]
        if out is None:
            out = torch.empty(q.shape, dtype=q.dtype, device=dev)
        elif out.shape != q.shape:
            raise ValueError(f"out is {tuple(out.shape)}, q {tuple(q.shape)}")
        vo = _rows("out", out, dev)
        tp, stride = _table(table, dev, n)
        if max_len > table.shape[1] * self.block_tokens:
            raise ValueError(f"max_len {max_len} is more than a table row of {table.shape[1]} blocks holds")
        batch = GGKv8Batch(_ints("cu_rows", cu_rows, dev, n + 1), _ints("lens", lens, dev, n), tp, stride, n, rows, max_rows, max_len)
        lib, ref = native.load(), ctypes.byref
        need = ctypes.c_size_t()
        _check(lib.gg_kv8_attention_workspace(self._ref, ref(vq), ref(batch), window, ref(need)))
        if workspace is None:
            workspace = torch.empty(need.value, dtype=torch.uint8, device=dev) if need.value else None
        elif workspace.dtype != torch.uint8 or workspace.dim() != 1 or not workspace.is_contiguous():
            raise ValueError("workspace must be a contiguous uint8 vector")
        elif workspace.device != dev:
            _on_gpu("workspace", workspace, dev)
        lse = torch.empty(rows, q.shape[1], dtype=torch.float32, device=dev) if return_lse else None
        _call(dev, lib.gg_kv8_attention, self._ref, ref(vq), ref(vo), lse.data_ptr() or None if lse is not None else None, ref(batch),
              self.head_dim ** -0.5 if scale is None else scale, window, workspace.data_ptr() if workspace is not None else None,
              workspace.numel() if workspace is not None else 0)
        return (out, lse) if return_lse else out

    def workspace_bytes(self, q: torch.Tensor, seqs: int, max_rows: int, max_len: int, window: int = 0) -> int:
        """Bytes of ``workspace`` that ``attend`` needs for such a batch."""
        vq = _rows("q", q, self.device)
        batch = GGKv8Batch(16, 16, 16, -(-max_len // self.block_tokens), seqs, q.shape[0], max_rows, max_len)
        need = ctypes.c_size_t()
        _check(native.load().gg_kv8_attention_workspace(self._ref, ctypes.byref(vq), ctypes.byref(batch), window, ctypes.byref(need)))
        return need.value
