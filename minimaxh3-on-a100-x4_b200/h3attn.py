"""Torch-facing binding of libh3attn.so (the sm_100a kernels behind include/h3attn.h).

Every function here validates its tensors, passes raw device pointers, element strides
and the current CUDA stream through ctypes, and raises on a negative return code. There
is no CPU path: a missing library or a non-CUDA tensor is an error.

Reference counterparts:
  attention            SDPA FLASH call, harness/sp_runtime.py:119-121 (and the unwired
                       fa3(q, k, v, o) of attn_sm80/attn_sm80.py:26-31)
  qknorm_rope_pack     ck.rms_rope_split_half_ + transposes + send reshape, sp_runtime.py:93-104, :69
  seq_to_head_unpack   receive-side permute copy, sp_runtime.py:71
  head_to_seq_unpack   transpose/reshape ahead of out_proj, sp_runtime.py:125
Without a counterpart in the reference:
  RopePositions, rope_axes   rotary positions over several axes (time, height, width)
  window_attention           sliding window with first tokens that stay visible
  linear_lora                low-rank adapters of many requests beside a shared projection
"""
from __future__ import annotations

import contextlib
import ctypes
import functools
import math
import os

import torch

HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(HERE, "libh3attn.so")
D = 128

_ERRORS = {
    -1: "a required pointer is NULL",
    -2: "a pointer is not 16-byte aligned",
    -3: "a size is out of range",
    -4: "a stride is not a multiple of 8 elements or is too small",
    -5: "the CUDA runtime refused the launch",
    -6: "cuTensorMapEncodeTiled rejected the layout",
    -7: "driver entry point unavailable",
    -8: "unsupported configuration",
    -9: "a CUDA runtime call failed",
    -10: "the call needs more than the no-alloc entry point's static scratch",
    -11: "a kernel gave up waiting (bounded-wait timeout)",
    -12: "the workspace is smaller than the call needs",
}
STATUS_NAMES = {
    0: "ok", 1: "timeout waiting for Q tiles", 2: "timeout in the K/V ring", 3: "timeout waiting for S",
    4: "timeout waiting for P", 5: "timeout waiting for O", 6: "timeout draining copies", 7: "timeout in a tile KAT",
}

_lib = None
_status = {}


class H3Error(RuntimeError):
    pass


def lib() -> ctypes.CDLL:
    """Load libh3attn.so once. Raises ImportError when it has not been built."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise ImportError(f"{LIB_PATH} is missing: build it with `python {os.path.join(HERE, 'build.py')}`")
        L = ctypes.CDLL(LIB_PATH)
        i64, vp, f32, i32p = ctypes.c_int64, ctypes.c_void_p, ctypes.c_float, ctypes.c_void_p
        L.h3_version.restype = ctypes.c_int
        L.h3_attn_fwd.argtypes = [vp, vp, vp, vp] + [i64] * 11 + [f32, i32p, vp]
        L.h3_attn_fwd.restype = ctypes.c_int
        L.h3_attn_fwd_variant.argtypes = [vp, vp, vp, vp] + [i64] * 11 + [f32, i32p, ctypes.c_int32, vp]
        L.h3_attn_fwd_variant.restype = ctypes.c_int
        L.h3_qknorm_rope_pack.argtypes = [vp, vp, vp, i64, vp, i64, vp, vp, f32, vp, vp, vp, i64, i64, i64, i64,
                                          i64, vp]
        L.h3_qknorm_rope_pack.restype = ctypes.c_int
        L.h3_seq_to_head_unpack.argtypes = [vp, vp] + [i64] * 7 + [vp]
        L.h3_seq_to_head_unpack.restype = ctypes.c_int
        L.h3_head_to_seq_unpack.argtypes = [vp, vp, i64, i64, vp]
        L.h3_head_to_seq_unpack.restype = ctypes.c_int
        L.h3_tile_kat_qk.argtypes = [vp, vp, vp, i32p, vp]
        L.h3_tile_kat_qk.restype = ctypes.c_int
        L.h3_tile_kat_pv.argtypes = [vp, vp, vp, i32p, vp]
        L.h3_tile_kat_pv.restype = ctypes.c_int
        L.h3_wait_kat.argtypes = [vp, i64, i32p, vp]
        L.h3_wait_kat.restype = ctypes.c_int
        for name in ("h3_tile_kat_pair_qk", "h3_tile_kat_pair_pv"):
            getattr(L, name).argtypes = [vp, vp, vp, i32p, vp]
            getattr(L, name).restype = ctypes.c_int
        L.h3_gemm_bf16.argtypes = [vp, i64, i64, i64, i64, i64, vp, i64, i64, vp, i64, ctypes.c_int32, i32p, vp]
        L.h3_gemm_bf16.restype = ctypes.c_int
        L.h3_gemm_adapters_workspace.argtypes = [i64, i64, i64, i64, ctypes.c_int32, i64, i64]
        L.h3_gemm_adapters_workspace.restype = i64
        L.h3_gemm_adapters.argtypes = [vp, i64, i64, i64, i64, i64, vp, i64, i64, vp, i64, vp, i64, i64, i64, vp, vp, vp,
                                       i64, ctypes.c_int32, vp, i64, i32p, vp]
        L.h3_gemm_adapters.restype = ctypes.c_int
        L.h3_norm_modulate.argtypes = [vp, i64, vp, i64, vp, vp, i64, vp, vp, i64, vp, vp, i64, i64, i64,
                                       ctypes.c_float, vp]
        L.h3_norm_modulate.restype = ctypes.c_int
        L.h3_gated_residual.argtypes = [vp, i64, vp, i64, vp, i64, vp, vp, i64, i64, i64, vp]
        L.h3_gated_residual.restype = ctypes.c_int
        L.h3_qknorm_rope_pack_peer.argtypes = [vp, vp, vp, i64, vp, i64, vp, vp, ctypes.c_float, vp, i64, i64, i64,
                                               i64, i64, i64, i64, vp]
        L.h3_qknorm_rope_pack_peer.restype = ctypes.c_int
        L.h3_attn_fwd_peer.argtypes = [vp] * 5 + [i64] * 11 + [ctypes.c_float, i32p, vp]
        L.h3_attn_fwd_peer.restype = ctypes.c_int
        L.h3_window_attn_workspace.argtypes = [i64] * 7 + [ctypes.c_int32, i64, i64]
        L.h3_window_attn_workspace.restype = i64
        L.h3_window_attn.argtypes = [vp] * 4 + [i64] * 12 + [f32, i64, i64, i64, ctypes.c_int32, i64, i64, vp, i64, i32p,
                                     vp]
        L.h3_window_attn.restype = ctypes.c_int
        L.h3_window_plan_kat.argtypes = [i64] * 7 + [ctypes.c_int32, i64, i64, ctypes.c_int32, vp, i64]
        L.h3_window_plan_kat.restype = i64
        L.h3_window_mask_kat.argtypes = [i64] * 4 + [ctypes.c_int32] + [i64] * 4 + [ctypes.c_int32, vp]
        L.h3_window_mask_kat.restype = ctypes.c_int
        L.h3_adapters_deal_kat.argtypes = [i64, i64, i64, ctypes.c_int32, vp, i64, vp]
        L.h3_adapters_deal_kat.restype = i64
        L.h3_pack_ranks_kat.argtypes = [i64, i64, vp]
        L.h3_pack_ranks_kat.restype = ctypes.c_int
        L.h3_rope_axes.argtypes = [vp, i64, i64, vp, ctypes.c_int32, i64, vp, vp, ctypes.c_int32, vp, i64, i64, i64,
                                   i64, vp]
        L.h3_rope_axes.restype = ctypes.c_int
        L.h3_qknorm_rope_pack_axes.argtypes = [vp, vp, vp, i64, vp, ctypes.c_int32, i64, vp, vp, vp, vp, f32, vp, vp,
                                               vp, i64, i64, i64, i64, i64, vp]
        L.h3_qknorm_rope_pack_axes.restype = ctypes.c_int
        L.h3_qknorm_rope_pack_axes_peer.argtypes = [vp, vp, vp, i64, vp, ctypes.c_int32, i64, vp, vp, vp, vp, f32, vp,
                                                    i64, i64, i64, i64, i64, i64, i64, vp]
        L.h3_qknorm_rope_pack_axes_peer.restype = ctypes.c_int
        L.h3_copy_2d.argtypes = [vp, i64, vp, i64, i64, i64, vp]
        L.h3_copy_2d.restype = ctypes.c_int
        L.h3_status_read.argtypes = [i32p, vp]
        L.h3_status_read.restype = ctypes.c_int
        _lib = L
    return _lib


def _check(rc: int, what: str) -> None:
    if rc != 0:
        raise H3Error(f"{what}: {_ERRORS.get(rc, 'error')} (code {rc})")


def _stream() -> int:
    """The raw handle of the current stream (torch.cuda.current_stream() builds a Stream object around it, which
    costs 3 us a call)."""
    return torch._C._cuda_getCurrentRawStream(torch.cuda.current_device())


def _cuda(t: torch.Tensor, name: str, dtype=torch.bfloat16) -> None:
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise H3Error(f"{name} must be a CUDA tensor (this library has no CPU path)")
    if t.dtype != dtype:
        raise H3Error(f"{name} must be {dtype}, got {t.dtype}")


def _together(index: int, **tensors) -> None:
    """Every given tensor lives on GPU `index`."""
    for n, t in tensors.items():
        if t is not None and t.get_device() != index:
            raise H3Error(f"{n} is on {t.device}, the call runs on cuda:{index}")


_HERE = contextlib.nullcontext()


def _on(index: int):
    """Context in which GPU `index` is the current device: a launch goes to its tensors' device, on the
    stream that is current there."""
    return _HERE if index == torch.cuda.current_device() else torch.cuda.device(index)


def _status_ptr(index: int) -> int:
    """Address of the status word, made before the first launch that hands it out, and not inside a graph capture,
    whose pool would own it."""
    st = _status.get(index)
    if st is None:
        if torch.cuda.is_current_stream_capturing():
            raise H3Error("call status_word() once before the first graph capture on this device")
        st = status_word(torch.device("cuda", index))
    return st.data_ptr()


def status_word(device=None) -> torch.Tensor:
    """The int32 device status word this process hands to every kernel on `device`."""
    dev = torch.device("cuda", torch.cuda.current_device() if device is None else torch.device(device).index or 0)
    st = _status.get(dev.index)
    if st is None:
        st = torch.zeros(1, dtype=torch.int32, device=dev)
        if not torch.cuda.is_current_stream_capturing():
            torch.cuda.current_stream(dev).synchronize()  # zero before a call on any other stream reads it
        _status[dev.index] = st
    return st


def check_status(device=None) -> None:
    """Synchronise with the stream that is current on `device` and raise if a kernel there reported a bounded-wait
    timeout."""
    st = status_word(device)
    with _on(st.get_device()):
        code = lib().h3_status_read(ctypes.c_void_p(st.data_ptr()), ctypes.c_void_p(_stream()))
    if code < 0:
        _check(code, "h3_status_read")
    if code != 0:
        st.zero_()
        raise H3Error(f"device status {code}: {STATUS_NAMES.get(code, 'unknown')}")


# ----------------------------------------------------------------------------- attention
def _out_layout(layout: str, H: int, sq: int, world: int):
    """(shape, rows per rank, rank / head / row strides) of an attention output layout."""
    if layout == "head":
        return (H, sq, D), sq, 0, sq * D, D
    if layout == "token":
        return (sq, H * D), sq, 0, D, H * D
    if layout == "send":
        if sq % world:
            raise H3Error(f"send layout needs rows {sq} divisible by world {world}")
        sl = sq // world
        return (world, H, sl, D), sl, H * sl * D, sl * D, D
    raise H3Error(f"unknown layout {layout!r}")


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, s_kv: int | None = None,
              scale: float | None = None, out: torch.Tensor | None = None, layout: str = "head",
              world: int = 1, variant: int | None = None) -> torch.Tensor:
    """Exact attention over heads: q [H, Sq, 128], k/v [H, Skv, 128] (bf16, last dim
    contiguous, any head/row strides that are multiples of 8). Keys/values stop at s_kv
    (default Skv). Output layout:
      "head":  [H, Sq, 128]
      "token": [Sq, H*128] (what out_proj consumes)
      "send":  [world, H, Sq/world, 128] -- the head->seq all-to-all send buffer
    """
    for n, t in (("q", q), ("k", k), ("v", v)):
        _cuda(t, n)
        if t.dim() != 3 or t.shape[-1] != D or t.stride(-1) != 1:
            raise H3Error(f"{n} must be [heads, rows, 128] with a contiguous last dim, got {tuple(t.shape)}")
    H, sq, _ = q.shape
    if k.shape[0] != H or v.shape[0] != H or k.shape[1] != v.shape[1]:
        raise H3Error("q, k, v disagree on heads or key count")
    if k.stride() != v.stride():
        raise H3Error("k and v must share strides")
    skv_alloc = k.shape[1]
    s_kv = skv_alloc if s_kv is None else int(s_kv)
    if not 1 <= s_kv <= skv_alloc:
        raise H3Error(f"s_kv={s_kv} outside [1, {skv_alloc}]")
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    shape, rank_rows, rank_stride, head_stride, row_stride = _out_layout(layout, H, sq, world)
    if out is None:
        out = torch.empty(shape, dtype=torch.bfloat16, device=q.device)
    else:
        _cuda(out, "out")
        if tuple(out.shape) != tuple(shape) or not out.is_contiguous():
            raise H3Error(f"out must be contiguous {shape}, got {tuple(out.shape)}")
    args = (q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), H, sq, s_kv, q.stride(0), q.stride(1),
            k.stride(0), k.stride(1), rank_rows, rank_stride, head_stride, row_stride, scale,
            status_word(q.device).data_ptr())
    if variant is None:
        rc = lib().h3_attn_fwd(*args, _stream())
    else:
        rc = lib().h3_attn_fwd_variant(*args, int(variant), _stream())
    _check(rc, "h3_attn_fwd")
    return out


# ----------------------------------------------------------------------------- windowed attention
@functools.lru_cache(maxsize=4096)
def _window_workspace(dev_index: int, *shape) -> int:
    """Workspace bytes of a windowed attention call of these sizes on the current device."""
    n = lib().h3_window_attn_workspace(*shape)
    if n < 0:
        _check(n, "h3_window_attn_workspace")
    return n


def _head_strides(t: torch.Tensor, heads: int, rows: int) -> tuple:
    """(head, row) strides of [heads, rows, 128]; an axis of one element has whatever stride, 128 stands for it."""
    st = t.stride()
    return st[0] if heads > 1 else D, st[1] if rows > 1 else D


def window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, left: int | None, right: int | None,
                     sinks: int = 0, causal: bool = False, q_start: int | None = None, s_kv: int | None = None,
                     scale: float | None = None, out: torch.Tensor | None = None, layout: str = "head",
                     world: int = 1, splits: int | None = None) -> torch.Tensor:
    """Attention with a sliding window and first tokens that stay visible: q [H, Sq, 128], k/v [Hkv, Skv, 128]
    (bf16, last dim contiguous, strides multiples of 8; H a multiple of Hkv, query head h reads key head
    h // (H // Hkv)). Query i sits at key position p = q_start + i and sees key j < s_kv when j < sinks or
    p - left <= j <= p + right; causal=True also asks j <= p. None for left / right: no bound on that side. q_start
    defaults to max(s_kv - Sq, 0): the queries are the last keys. A query that sees no key gets zeros. K and V
    may hold anything at keys that no query sees. out / layout / world as attention().
    splits: how many parts the key axis is worked in (None: chosen by the call's sizes); with 1 a query row's
    bits do not depend on how many key heads share the call, each with the same number of query heads."""
    for n, t in (("q", q), ("k", k), ("v", v)):
        _cuda(t, n)
        if t.dim() != 3 or t.shape[-1] != D or t.stride(-1) != 1:
            raise H3Error(f"{n} must be [heads, rows, 128] with a contiguous last dim, got {tuple(t.shape)}")
    dev = q.get_device()
    _together(dev, k=k, v=v, out=out)
    H, sq, _ = q.shape
    hk, skv_alloc, _ = k.shape
    if v.shape != k.shape or hk < 1 or H % hk:
        raise H3Error("k and v must share a shape, and the query heads be a multiple of the key heads")
    q_st, k_st = _head_strides(q, H, sq), _head_strides(k, hk, skv_alloc)
    if _head_strides(v, hk, skv_alloc) != k_st:
        raise H3Error("k and v must share strides")
    s_kv = skv_alloc if s_kv is None else int(s_kv)
    if not 1 <= s_kv <= skv_alloc:
        raise H3Error(f"s_kv={s_kv} outside [1, {skv_alloc}]")
    for n, side in (("left", left), ("right", right)):
        if side is not None and side < 0:
            raise H3Error(f"{n}={side}: a window side is a count of keys, or None for no bound")
    if sinks < 0 or (splits is not None and splits < 1):
        raise H3Error(f"sinks={sinks}, splits={splits} out of range")
    q_start = max(s_kv - sq, 0) if q_start is None else int(q_start)
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    shape, rank_rows, rank_stride, head_stride, row_stride = _out_layout(layout, H, sq, world)
    if out is None:
        out = q.new_empty(shape)
    else:
        _cuda(out, "out")
        if tuple(out.shape) != tuple(shape) or not out.is_contiguous():
            raise H3Error(f"out must be contiguous {shape}, got {tuple(out.shape)}")
    # sides past every key are no bound: keep them inside the C call's integers
    big = sq + s_kv + abs(q_start)
    lo, hi = (-1 if side is None or side > big else int(side) for side in (left, right))
    sinks = min(int(sinks), s_kv)
    with _on(dev):
        ws_bytes = _window_workspace(dev, H, hk, sq, s_kv, lo, hi, sinks, int(causal), q_start, splits or 0)
        ws = q.new_empty((ws_bytes // 2,)) if ws_bytes else None
        rc = lib().h3_window_attn(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), H, hk, sq, s_kv,
                                  *q_st, *k_st, rank_rows, rank_stride,
                                  head_stride, row_stride, scale, lo, hi, sinks, int(causal), q_start, splits or 0,
                                  ws.data_ptr() if ws_bytes else None, ws_bytes, _status_ptr(dev), _stream())
    _check(rc, "h3_window_attn")
    return out


# ----------------------------------------------------------------------------- rotary positions
def rope_axes_freqs(sections, theta: float = 10000.0, interleaved: bool = False, device=None):
    """(inv_freq, axis) of a rotary plan over len(sections) axes for RopePositions: axis a turns sections[a]
    of the head's 64 pairs with frequencies theta^(-j / sections[a]), j = 0, 1, ... Pairs are handed
    out axis after axis, or pair by pair in turn when interleaved; sections may sum to less than 64, the
    last pairs then keep their values. Made once per model."""
    sections = [int(n) for n in sections]
    if not 1 <= len(sections) <= 64 or min(sections) < 0 or sum(sections) > D // 2 or not theta > 0:
        raise H3Error(f"sections must be 1 to 64 counts >= 0 that sum to at most {D // 2}, theta > 0")
    pairs = [(j, a) for a, n in enumerate(sections) for j in range(n)]
    if interleaved:
        pairs.sort()
    rest = D // 2 - len(pairs)
    inv = [float(theta) ** (-j / sections[a]) for j, a in pairs] + [0.0] * rest
    return (torch.tensor(inv, dtype=torch.float64, device=device),
            torch.tensor([a for _, a in pairs] + [-1] * rest, dtype=torch.int32, device=device))


_PAIRS = torch.Size([D // 2])


class RopePositions:
    """Positions of tokens on several axes and the frequencies that turn them:
      pos: [tokens, axes] int32 or fp32; inv_freq: fp64 [64] radians per unit position of pair (i, i + 64);
      axis: int32 [64], the axis of each pair (outside [0, axes): the pair keeps its values, if finite).
    Accepted by qknorm_rope_pack / _peer in place of a table of rotation matrices, by rope_axes, and as
    sp_runtime's rope_freqs."""

    __slots__ = ("pos", "inv_freq", "axis")

    def __init__(self, pos: torch.Tensor, inv_freq: torch.Tensor, axis: torch.Tensor):
        self.pos, self.inv_freq, self.axis = pos, inv_freq, axis

    def rows(self, lo: int, hi: int, tokens: int | None = None) -> "RopePositions":
        """The positions of tokens [lo, hi) of a sequence of `tokens` (default: all that there are positions for);
        tokens past its last one (padding) sit at position 0."""
        n = self.pos.shape[0] if tokens is None else tokens
        if not 0 <= n <= self.pos.shape[0]:
            raise H3Error(f"positions of {self.pos.shape[0]} tokens, the sequence has {n}")
        pos = self.pos[min(lo, n):min(hi, n)]
        if pos.shape[0] < hi - lo:
            pos = torch.cat([pos, pos.new_zeros((hi - lo - pos.shape[0],) + tuple(pos.shape[1:]))])
        return RopePositions(pos.contiguous(), self.inv_freq, self.axis)

    def _args(self, tokens: int, index: int) -> tuple:
        """(pos, type, axes, inv_freq, axis) for the C calls, checked."""
        pos, f, a = self.pos, self.inv_freq, self.axis
        _cuda(f, "inv_freq", torch.float64)
        _cuda(a, "axis", torch.int32)
        if f.shape != _PAIRS or a.shape != _PAIRS or not (f.is_contiguous() and a.is_contiguous()):
            raise H3Error(f"inv_freq and axis must be contiguous [{D // 2}]")
        real = isinstance(pos, torch.Tensor) and pos.dtype == torch.float32
        _cuda(pos, "pos", torch.float32 if real else torch.int32)
        shape = pos.shape
        if len(shape) != 2 or shape[0] != tokens or not 1 <= shape[1] <= 64 or not pos.is_contiguous():
            raise H3Error(f"pos must be contiguous [{tokens}, axes] with 1 to 64 axes, got {tuple(shape)}")
        _together(index, pos=pos, inv_freq=f, axis=a)
        return pos.data_ptr(), int(real), shape[1], f.data_ptr(), a.data_ptr()


def rope_axes(x: torch.Tensor, positions: RopePositions, inverse: bool = False,
              out: torch.Tensor | None = None) -> torch.Tensor:
    """Rotate x [tokens, heads, 128] (bf16, last dim contiguous, row and head strides multiples of 8) by
    its tokens' positions; inverse=True applies the transposed rotation, which is the rotation's gradient.
    out (default: a new contiguous tensor) may be x itself."""
    _cuda(x, "x")
    if x.dim() != 3 or x.shape[-1] != D or x.stride(-1) != 1:
        raise H3Error(f"x must be [tokens, heads, 128] with a contiguous last dim, got {tuple(x.shape)}")
    if out is None:
        out = x.new_empty(x.shape)
    else:
        _cuda(out, "out")
        if out.shape != x.shape or out.stride(-1) != 1:
            raise H3Error(f"out must be {tuple(x.shape)} with a contiguous last dim")
    tokens, heads, _ = x.shape
    dev, x_st, o_st = x.get_device(), x.stride(), out.stride()
    _together(dev, out=out)
    args = positions._args(tokens, dev)
    with _on(dev):
        rc = lib().h3_rope_axes(x.data_ptr(), x_st[0], x_st[1], *args, int(inverse), out.data_ptr(), o_st[0], o_st[1],
                                tokens, heads, _stream())
    _check(rc, "h3_rope_axes")
    return out


# ----------------------------------------------------------------------------- fused exchanges (peer memory)
def qknorm_rope_pack_peer(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, rope: torch.Tensor | None,
                          q_weight: torch.Tensor | None, k_weight: torch.Tensor | None, eps: float, world: int,
                          rank_base: torch.Tensor, tensor_stride: int, head_stride: int, row_offset: int) -> None:
    """The pack with the seq->head exchange fused in: head g of each token goes straight to rank
    g // (H/world)'s buffer at rank_base[rank] (int64 device tensor [world] of addresses mapped in
    this process) + tensor*tensor_stride + local_head*head_stride + (row_offset + token)*128."""
    axes = rope if isinstance(rope, RopePositions) else None
    q2, k2, v2, sl, H, rope_ptr, rope_stride, wptr = _pack_args(q, k, v, None if axes else rope, q_weight, k_weight)
    if H % world:
        raise H3Error(f"heads {H} not divisible by world {world}")
    _cuda(rank_base, "rank_base", torch.int64)
    if tuple(rank_base.shape) != (world,) or not rank_base.is_contiguous():
        raise H3Error("rank_base must be a contiguous int64 [world] device tensor")
    if axes is not None:
        dev = q.get_device()
        _together(dev, k=k, v=v, q_weight=q_weight, k_weight=k_weight, rank_base=rank_base)
        with _on(dev):
            rc = lib().h3_qknorm_rope_pack_axes_peer(
                q2.data_ptr(), k2.data_ptr(), v2.data_ptr(), q2.stride(0), *axes._args(sl, dev), wptr[0], wptr[1],
                float(eps), rank_base.data_ptr(), world, tensor_stride, head_stride, row_offset, sl, H, H // world,
                _stream())
        _check(rc, "h3_qknorm_rope_pack_axes_peer")
        return
    rc = lib().h3_qknorm_rope_pack_peer(q2.data_ptr(), k2.data_ptr(), v2.data_ptr(), q2.stride(0), rope_ptr,
                                        rope_stride, wptr[0], wptr[1], float(eps), rank_base.data_ptr(), world,
                                        tensor_stride, head_stride, row_offset, sl, H, H // world, _stream())
    _check(rc, "h3_qknorm_rope_pack_peer")


def attention_peer(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, o_local: torch.Tensor, o_peer: torch.Tensor,
                   rank_rows: int, head_stride: int, row_stride: int, s_kv: int | None = None,
                   scale: float | None = None) -> None:
    """Attention with the head->seq exchange fused into the epilogue: query row i of head h goes to
    o_peer[i // rank_rows] + h*head_stride + (i % rank_rows)*row_stride (elements)."""
    for n, t in (("q", q), ("k", k), ("v", v)):
        _cuda(t, n)
        if t.dim() != 3 or t.shape[-1] != D or t.stride(-1) != 1:
            raise H3Error(f"{n} must be [heads, rows, 128] with a contiguous last dim")
    _cuda(o_local, "o_local")
    _cuda(o_peer, "o_peer", torch.int64)
    H, sq, _ = q.shape
    if k.shape[0] != H or v.shape[0] != H or k.shape[1] != v.shape[1] or k.stride() != v.stride():
        raise H3Error("q, k, v disagree on heads, key count or strides")
    if o_peer.dim() != 1 or o_peer.shape[0] * rank_rows < sq or not o_peer.is_contiguous():
        raise H3Error("o_peer must hold one address per destination rank")
    s_kv = k.shape[1] if s_kv is None else int(s_kv)
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    rc = lib().h3_attn_fwd_peer(q.data_ptr(), k.data_ptr(), v.data_ptr(), o_local.data_ptr(), o_peer.data_ptr(),
                                o_peer.shape[0], H, sq, s_kv, q.stride(0), q.stride(1), k.stride(0), k.stride(1), rank_rows, head_stride,
                                row_stride, scale, status_word(q.device).data_ptr(), _stream())
    _check(rc, "h3_attn_fwd_peer")


# ----------------------------------------------------------------------------- pack / unpack
def _pack_args(q, k, v, rope, q_weight, k_weight):
    """Checks shared by the pack entry points; returns (q2, k2, v2, tokens, heads, rope_ptr,
    rope_row_stride, [q_weight_ptr, k_weight_ptr])."""
    rows = []
    for n, t in (("q", q), ("k", k), ("v", v)):
        _cuda(t, n)
        if t.dim() == 3:
            t = t.reshape(t.shape[0], -1)
        if t.dim() != 2 or t.stride(-1) != 1:
            raise H3Error(f"{n} must be [tokens, heads*128] with a contiguous last dim")
        rows.append(t)
    q2, k2, v2 = rows
    sl, hd = q2.shape
    if hd % D or k2.shape != q2.shape or v2.shape != q2.shape:
        raise H3Error("q, k, v must share shape [tokens, heads*128]")
    if not (q2.stride(0) == k2.stride(0) == v2.stride(0)):
        raise H3Error("q, k, v must share a row stride")
    rope_ptr, rope_stride = None, 0
    if rope is not None:
        _cuda(rope, "rope", torch.float32)
        if rope.dim() == 5:
            if rope.shape[0] != 1:
                raise H3Error("rope batch dim must be 1")
            rope = rope[0]
        if tuple(rope.shape[1:]) != (64, 2, 2) or rope.shape[0] != sl or not rope[0].is_contiguous():
            raise H3Error(f"rope must be [tokens, 64, 2, 2] fp32 (rot_dim 128), got {tuple(rope.shape)}")
        rope_ptr, rope_stride = rope.data_ptr(), rope.stride(0)
    wptr = []
    for n, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is None:
            wptr.append(None)
            continue
        _cuda(w, n)
        if tuple(w.shape) != (D,) or not w.is_contiguous():
            raise H3Error(f"{n} must be contiguous [128] bf16")
        wptr.append(w.data_ptr())
    return q2, k2, v2, sl, hd // D, rope_ptr, rope_stride, wptr


def qknorm_rope_pack(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, rope: torch.Tensor | None,
                     q_weight: torch.Tensor | None, k_weight: torch.Tensor | None, eps: float, world: int,
                     out: torch.Tensor | None = None, head_major: bool = False) -> torch.Tensor:
    """q, k, v: [S_l, H*128] (views of the fused QKV output are fine; rows may be strided).
    rope: fp32 [S_l, 64, 2, 2], a RopePositions over S_l tokens, or None. Returns the seq->head send buffer
    [world, 3, H/world, S_l, 128] with q and k RMS-normalised (+ rotated); head_major=True lays
    it out [H/world, world, 3, S_l, 128] instead, so each local head's blocks for all peers are
    one contiguous all-to-all buffer (head-by-head pipelining)."""
    axes = rope if isinstance(rope, RopePositions) else None
    q2, k2, v2, sl, H, rope_ptr, rope_stride, wptr = _pack_args(q, k, v, None if axes else rope, q_weight, k_weight)
    if H % world:
        raise H3Error(f"heads {H} not divisible by world {world}")
    hl = H // world
    shape = (hl, world, 3, sl, D) if head_major else (world, 3, hl, sl, D)
    if out is None:
        out = torch.empty(shape, dtype=torch.bfloat16, device=q.device)
    elif tuple(out.shape) != shape or not out.is_contiguous():
        raise H3Error(f"out must be contiguous {shape}")
    if head_major:  # element (h, rank, tensor, row) at ((h*world + rank)*3 + tensor)*sl + row
        tstride, rank_stride, head_stride = sl * D, 3 * sl * D, world * 3 * sl * D
    else:           # element (rank, tensor, h, row) at ((rank*3 + tensor)*hl + h)*sl + row
        tstride, rank_stride, head_stride = hl * sl * D, 3 * hl * sl * D, sl * D
    base = out.data_ptr()
    if axes is not None:
        _cuda(out, "out")
        dev = q.get_device()
        _together(dev, k=k, v=v, q_weight=q_weight, k_weight=k_weight, out=out)
        with _on(dev):
            rc = lib().h3_qknorm_rope_pack_axes(
                q2.data_ptr(), k2.data_ptr(), v2.data_ptr(), q2.stride(0), *axes._args(sl, dev), wptr[0], wptr[1],
                float(eps), base, base + 2 * tstride, base + 4 * tstride, sl, H, hl, rank_stride, head_stride,
                _stream())
        _check(rc, "h3_qknorm_rope_pack_axes")
        return out
    rc = lib().h3_qknorm_rope_pack(q2.data_ptr(), k2.data_ptr(), v2.data_ptr(), q2.stride(0), rope_ptr, rope_stride,
                                   wptr[0], wptr[1], float(eps), base, base + 2 * tstride, base + 4 * tstride, sl, H,
                                   hl, rank_stride, head_stride, _stream())
    _check(rc, "h3_qknorm_rope_pack")
    return out


def seq_to_head_unpack(recv: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """recv [W, T, Hl, Sl, 128] (one block per source rank) -> [T, Hl, W*Sl, 128]."""
    _cuda(recv, "recv")
    if recv.dim() != 5 or recv.shape[-1] != D or not recv.is_contiguous():
        raise H3Error("recv must be contiguous [world, tensors, heads, tokens, 128]")
    W, T, hl, sl, _ = recv.shape
    if out is None:
        out = torch.empty((T, hl, W * sl, D), dtype=torch.bfloat16, device=recv.device)
    elif tuple(out.shape) != (T, hl, W * sl, D) or not out.is_contiguous():
        raise H3Error("out has the wrong shape")
    rc = lib().h3_seq_to_head_unpack(recv.data_ptr(), out.data_ptr(), W, hl, sl, T, T * hl * sl * D, hl * sl * D,
                                     hl * W * sl * D, _stream())
    _check(rc, "h3_seq_to_head_unpack")
    return out


def copy_2d(dst_ptr: int, dst_pitch: int, src_ptr: int, src_pitch: int, width: int, rows: int,
            stream: torch.cuda.Stream | None = None) -> None:
    """Copy-engine copy of `rows` rows of `width` bytes (pitches in bytes) on `stream` (default: the
    current one); either address may be a peer GPU's mapped memory. Used for the all-to-all
    exchanges of SP_OVERLAP=ce: each rank writes its chunk straight into every destination's
    attention / out_proj input."""
    st = (stream or torch.cuda.current_stream()).cuda_stream
    _check(lib().h3_copy_2d(dst_ptr, dst_pitch, src_ptr, src_pitch, width, rows, st), "h3_copy_2d")


def head_to_seq_unpack(recv: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """[H, Sl, 128] head-major -> [Sl, H*128] token-major."""
    _cuda(recv, "recv")
    if recv.dim() != 3 or recv.shape[-1] != D or not recv.is_contiguous():
        raise H3Error("recv must be contiguous [heads, tokens, 128]")
    H, sl, _ = recv.shape
    if out is None:
        out = torch.empty((sl, H * D), dtype=torch.bfloat16, device=recv.device)
    elif tuple(out.shape) != (sl, H * D) or not out.is_contiguous():
        raise H3Error("out has the wrong shape")
    rc = lib().h3_head_to_seq_unpack(recv.data_ptr(), out.data_ptr(), H, sl, _stream())
    _check(rc, "h3_head_to_seq_unpack")
    return out


# ----------------------------------------------------------------------------- projection GEMM
def _linear_args(a, weight, out, epilogue):
    """Checks shared by the projections; returns (m, chunks, chunk columns, chunk stride, row stride, output columns,
    epilogue code, out)."""
    _cuda(a, "a")
    _cuda(weight, "weight")
    if weight.dim() != 2 or weight.stride(-1) != 1:
        raise H3Error("weight must be [out, in] with a contiguous last dim")
    if a.dim() == 2:
        if a.stride(-1) != 1:
            raise H3Error("a must have a contiguous last dim")
        m, k = a.shape
        chunks, chunk_cols, chunk_stride, row_stride = 1, k, 0, a.stride(0)
    elif a.dim() == 3:
        if a.stride(-1) != 1:
            raise H3Error("a must have a contiguous last dim")
        chunks, m, chunk_cols = a.shape
        chunk_stride, row_stride = a.stride(0), a.stride(1)
        k = chunks * chunk_cols
    else:
        raise H3Error(f"a must be 2-D or 3-D, got {tuple(a.shape)}")
    if weight.shape[1] != k:
        raise H3Error(f"weight has {weight.shape[1]} inputs, a has {k}")
    ep = {"none": 0, "swiglu": 1}.get(epilogue)
    if ep is None:
        raise H3Error(f"unknown epilogue {epilogue!r}")
    n = weight.shape[0] // 2 if ep == 1 else weight.shape[0]
    if ep == 1 and weight.shape[0] % 2:
        raise H3Error("swiglu weight needs an even row count")
    if out is None:
        out = a.new_empty((m, n))
    else:
        _cuda(out, "out")
        if tuple(out.shape) != (m, n) or out.stride(-1) != 1:
            raise H3Error(f"out must be [{m}, {n}] with a contiguous last dim")
    return m, chunks, chunk_cols, chunk_stride, row_stride, n, ep, out


def linear(a: torch.Tensor, weight: torch.Tensor, out: torch.Tensor | None = None,
           epilogue: str = "none") -> torch.Tensor:
    """Row-independent a @ weight.T (bf16, fp32 accumulate): the bits of an output row depend only
    on that row of `a`, never on how many rows the call has.
      a: [m, k] with a contiguous last dim, or head-major [H, m, 128] (read in place as [m, H*128]);
      weight: [n, k] (nn.Linear layout); epilogue "swiglu": weight = [gate; up] (2F rows) and the
      result is silu(a @ gate.T) * (a @ up.T), [m, F]."""
    m, chunks, chunk_cols, chunk_stride, row_stride, n, ep, out = _linear_args(a, weight, out, epilogue)
    rc = lib().h3_gemm_bf16(a.data_ptr(), m, chunks, chunk_cols, chunk_stride, row_stride, weight.data_ptr(), n,
                            weight.stride(0), out.data_ptr(), out.stride(0), ep, status_word(a.device).data_ptr(),
                            _stream())
    _check(rc, "h3_gemm_bf16")
    return out


# ----------------------------------------------------------------------------- adapters beside a projection
_RANKS = (8, 16, 32, 64, 128, 192, 256)
_ROW_INDEPENDENT = 0x100  # H3_GEMM_ROW_INDEPENDENT


def stack_adapters(pairs, scales, device=None):
    """(lora_a, lora_b, scale) as linear_lora takes them, from [(A [r, k], B [n, r]), ...] with ranks up to 256 and one
    factor each: ranks are padded with zeros to the smallest of 8, 16, 32, 64, 128, 192, 256 that holds them all. Laid
    out once per set of adapters."""
    pairs = list(pairs)
    if not pairs or len(scales) != len(pairs):
        raise H3Error("one (A, B) pair and one scale per adapter")
    k, n = pairs[0][0].shape[1], pairs[0][1].shape[0]
    for A, B in pairs:
        if A.dim() != 2 or B.dim() != 2 or A.shape[1] != k or B.shape[0] != n or A.shape[0] != B.shape[1]:
            raise H3Error("adapters must be A [r, k], B [n, r] with one k and one n")
        if not bool(torch.isfinite(B.to(torch.bfloat16)).all()):
            raise H3Error("an adapter's B is not finite: it would reach the rows of other adapters")
    most = max(A.shape[0] for A, _ in pairs)
    rank = next((r for r in _RANKS if r >= most), None)
    if rank is None:
        raise H3Error(f"rank {most} is above {_RANKS[-1]}")
    device = pairs[0][0].device if device is None else device
    lora_a = torch.zeros(len(pairs) * rank, k, dtype=torch.bfloat16, device=device)
    lora_b = torch.zeros(n, len(pairs) * rank, dtype=torch.bfloat16, device=device)
    for i, (A, B) in enumerate(pairs):
        lora_a[i * rank:i * rank + A.shape[0]] = A
        lora_b[:, i * rank:i * rank + A.shape[0]] = B
    return lora_a, lora_b, torch.tensor([float(x) for x in scales], dtype=torch.float32, device=device)


@functools.lru_cache(maxsize=4096)
def _adapters_workspace(dev_index: int, *shape) -> int:
    """Workspace bytes of a call of these sizes on the current device."""
    n = lib().h3_gemm_adapters_workspace(*shape)
    if n < 0:
        _check(n, "h3_gemm_adapters_workspace")
    return n


def linear_lora(a: torch.Tensor, weight: torch.Tensor, lora_a: torch.Tensor, lora_b: torch.Tensor,
                scale: torch.Tensor, rows: torch.Tensor, out: torch.Tensor | None = None,
                epilogue: str = "none", row_independent: bool = False) -> torch.Tensor:
    """linear() with a low-rank adapter per row: a @ weight.T + scale[g] * (a @ A_g.T) @ B_g.T with g = rows[row]
    (outside [0, adapters): the projection alone), rounded once; epilogue "swiglu" as linear().
      a, weight, out: as linear(); lora_a: [adapters * rank, k], lora_b: [weight rows, adapters * rank] bf16, adapter g at
      [g * rank, (g + 1) * rank) of both (stack_adapters lays them out); rank 8, 16, 32 or a multiple of 64 up to 256;
      scale: fp32 [adapters]; rows: int32 [m] (segment_rows makes it from token segments).
    In calls of more than 64 rows a row's bits do not depend on the other rows, and a row without an adapter has
    linear()'s bits; up to 64 rows the order of its sums follows which adapters the call uses, unless row_independent is
    set (slower: for shards of one sequence that must agree bit for bit whatever their lengths). B must be finite where
    it is used: rows meet the adapters that share their group of 64 stacked columns with zero weights."""
    m, chunks, chunk_cols, chunk_stride, row_stride, n, ep, out = _linear_args(a, weight, out, epilogue)
    _cuda(lora_a, "lora_a")
    _cuda(lora_b, "lora_b")
    _cuda(scale, "scale", torch.float32)
    _cuda(rows, "rows", torch.int32)
    dev = a.get_device()
    _together(dev, weight=weight, lora_a=lora_a, lora_b=lora_b, scale=scale, rows=rows, out=out)
    if scale.dim() != 1 or scale.shape[0] < 1 or not scale.is_contiguous():
        raise H3Error("scale must be a contiguous fp32 [adapters]")
    n_adapters = scale.shape[0]
    if lora_a.dim() != 2 or lora_a.shape[1] != weight.shape[1] or lora_a.shape[0] % n_adapters or lora_a.stride(1) != 1:
        raise H3Error(f"lora_a must be [{n_adapters} * rank, {weight.shape[1]}] with a contiguous last dim")
    if lora_b.shape != (weight.shape[0], lora_a.shape[0]) or lora_b.stride(1) != 1:
        raise H3Error(f"lora_b must be [{weight.shape[0]}, {lora_a.shape[0]}] with a contiguous last dim")
    if rows.shape != (m,) or not rows.is_contiguous():
        raise H3Error(f"rows must be a contiguous int32 [{m}]")
    rank = lora_a.shape[0] // n_adapters
    if row_independent:
        ep |= _ROW_INDEPENDENT
    with _on(dev):
        ws_bytes = _adapters_workspace(dev, m, chunks, chunk_cols, n, ep, rank, n_adapters)
        ws = a.new_empty(((ws_bytes + 1) // 2,))
        rc = lib().h3_gemm_adapters(a.data_ptr(), m, chunks, chunk_cols, chunk_stride, row_stride, weight.data_ptr(), n,
                                    weight.stride(0), lora_a.data_ptr(), lora_a.stride(0), lora_b.data_ptr(),
                                    lora_b.stride(0), rank, n_adapters, scale.data_ptr(), rows.data_ptr(),
                                    out.data_ptr(), out.stride(0), ep, ws.data_ptr(), ws_bytes,
                                    _status_ptr(dev), _stream())
    _check(rc, "h3_gemm_adapters")
    return out


# ----------------------------------------------------------------------------- AdaLN modulation
def segment_rows(mod_segments, rows: int, device) -> torch.Tensor:
    """int32 [rows]: the modulation row of each token ((a, b, row) segments, later ones win as in
    the host model's per-segment assignments), -1 outside every segment."""
    seg = torch.full((rows,), -1, dtype=torch.int32, device=device)
    for a, b, row in mod_segments:
        a, b = max(int(a), 0), min(int(b), rows)
        if a < b:
            seg[a:b] = int(row)
    return seg


def _rows2d(t: torch.Tensor, name: str, hidden: int) -> None:
    _cuda(t, name)
    if t.dim() != 2 or t.shape[1] != hidden or t.stride(1) != 1:
        raise H3Error(f"{name} must be [rows, {hidden}] with a contiguous last dim, got {tuple(t.shape)}")


def norm_modulate(x: torch.Tensor, shift: torch.Tensor, scale: torch.Tensor, seg_row: torch.Tensor, eps: float,
                  y: torch.Tensor | None = None, gate: torch.Tensor | None = None,
                  x_out: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """h = LN(xr) * (1 + scale[seg]) + shift[seg] with xr = x + gate[seg] * y when y is given
    (xr also written to x_out). x, y: [rows, hidden]; shift/scale/gate: [mod_rows, hidden] views
    sharing one row stride; seg_row: int32 [rows]."""
    rows, hidden = x.shape
    _rows2d(x, "x", hidden)
    for n, t in (("shift", shift), ("scale", scale)) + ((("gate", gate),) if y is not None else ()):
        _rows2d(t, n, hidden)
    if scale.stride(0) != shift.stride(0) or (y is not None and gate.stride(0) != shift.stride(0)):
        raise H3Error("shift, scale and gate must share a row stride")
    if y is not None:
        _rows2d(y, "y", hidden)
        if y.shape[0] != rows:
            raise H3Error("y and x disagree on rows")
    _cuda(seg_row, "seg_row", torch.int32)
    if seg_row.shape != (rows,) or not seg_row.is_contiguous():
        raise H3Error("seg_row must be a contiguous int32 [rows]")
    if x_out is not None:
        _rows2d(x_out, "x_out", hidden)
    if out is None:
        out = torch.empty((rows, hidden), dtype=torch.bfloat16, device=x.device)
    else:
        _rows2d(out, "out", hidden)
    rc = lib().h3_norm_modulate(x.data_ptr(), x.stride(0), y.data_ptr() if y is not None else None,
                                y.stride(0) if y is not None else 0, gate.data_ptr() if y is not None else None,
                                x_out.data_ptr() if x_out is not None else None,
                                x_out.stride(0) if x_out is not None else 0, shift.data_ptr(), scale.data_ptr(),
                                shift.stride(0), seg_row.data_ptr(), out.data_ptr(), out.stride(0), rows, hidden,
                                float(eps), _stream())
    _check(rc, "h3_norm_modulate")
    return out


def gated_residual(x: torch.Tensor, y: torch.Tensor, gate: torch.Tensor, seg_row: torch.Tensor,
                   out: torch.Tensor | None = None) -> torch.Tensor:
    """out = x + gate[seg] * y on segment tokens, x elsewhere."""
    rows, hidden = x.shape
    for n, t in (("x", x), ("y", y), ("gate", gate)):
        _rows2d(t, n, hidden)
    _cuda(seg_row, "seg_row", torch.int32)
    if y.shape[0] != rows or seg_row.shape != (rows,) or not seg_row.is_contiguous():
        raise H3Error("x, y and seg_row disagree on rows")
    if out is None:
        out = torch.empty((rows, hidden), dtype=torch.bfloat16, device=x.device)
    else:
        _rows2d(out, "out", hidden)
    rc = lib().h3_gated_residual(x.data_ptr(), x.stride(0), y.data_ptr(), y.stride(0), gate.data_ptr(), gate.stride(0),
                                 seg_row.data_ptr(), out.data_ptr(), out.stride(0), rows, hidden, _stream())
    _check(rc, "h3_gated_residual")
    return out


# ----------------------------------------------------------------------------- tile KATs
def tile_kat_qk(q: torch.Tensor, k: torch.Tensor) -> torch.Tensor:
    _cuda(q, "q")
    _cuda(k, "k")
    assert q.shape == (128, 128) and k.shape == (128, 128) and q.is_contiguous() and k.is_contiguous()
    s = torch.empty((128, 128), dtype=torch.float32, device=q.device)
    _check(lib().h3_tile_kat_qk(q.data_ptr(), k.data_ptr(), s.data_ptr(), status_word(q.device).data_ptr(),
                                _stream()), "h3_tile_kat_qk")
    return s


def tile_kat_pv(p: torch.Tensor, v: torch.Tensor) -> torch.Tensor:
    _cuda(p, "p")
    _cuda(v, "v")
    assert p.shape == (128, 128) and v.shape == (128, 128) and p.is_contiguous() and v.is_contiguous()
    o = torch.empty((128, 128), dtype=torch.float32, device=p.device)
    _check(lib().h3_tile_kat_pv(p.data_ptr(), v.data_ptr(), o.data_ptr(), status_word(p.device).data_ptr(),
                                _stream()), "h3_tile_kat_pv")
    return o


def tile_kat_pair_qk(q: torch.Tensor, k: torch.Tensor) -> torch.Tensor:
    """S[256][128] = q[256][128] . k[128][128]^T through an SM pair (cta_group::2)."""
    _cuda(q, "q")
    _cuda(k, "k")
    assert q.shape == (256, 128) and k.shape == (128, 128) and q.is_contiguous() and k.is_contiguous()
    s = torch.empty((256, 128), dtype=torch.float32, device=q.device)
    _check(lib().h3_tile_kat_pair_qk(q.data_ptr(), k.data_ptr(), s.data_ptr(), status_word(q.device).data_ptr(),
                                     _stream()), "h3_tile_kat_pair_qk")
    return s


def tile_kat_pair_pv(p: torch.Tensor, v: torch.Tensor) -> torch.Tensor:
    """O[256][128] = p[256][128] . v[128][128] through an SM pair (cta_group::2)."""
    _cuda(p, "p")
    _cuda(v, "v")
    assert p.shape == (256, 128) and v.shape == (128, 128) and p.is_contiguous() and v.is_contiguous()
    o = torch.empty((256, 128), dtype=torch.float32, device=p.device)
    _check(lib().h3_tile_kat_pair_pv(p.data_ptr(), v.data_ptr(), o.data_ptr(), status_word(p.device).data_ptr(),
                                     _stream()), "h3_tile_kat_pair_pv")
    return o


def wait_kat(tile: torch.Tensor, limit_ns: int) -> None:
    """Launch the bounded-wait KAT: one CTA loads `tile` [128, 128] bf16 by TMA, then waits up to
    limit_ns on a barrier nothing completes, reports H3_STATUS_TIMEOUT_KAT in the status word and
    returns. Read the outcome with check_status() (which raises on it)."""
    _cuda(tile, "tile")
    if tuple(tile.shape) != (128, 128) or not tile.is_contiguous():
        raise H3Error("tile must be a contiguous [128, 128] bf16 tensor")
    _check(lib().h3_wait_kat(tile.data_ptr(), int(limit_ns), status_word(tile.device).data_ptr(), _stream()),
           "h3_wait_kat")
