"""Launchers of the paged 8-bit key/value cache (``csrc/cuda/paged*.cu``; layout and contract in ``gb_paged.h``).

A pool of pages of 64 tokens holds keys and values as codes of 8 bits with one scale a page and key head.  A page belongs to whoever's table names it; the
pages of one text may be anywhere in the pool, and one table serves all layers of a model (a pool each).  Every call takes ``B`` sequences:
``start[b]`` tokens are in the pages ``table[b]`` already, and the call's own ``count[b]`` ones are the rows ``first[b]`` ... of its tensors (without
``first`` and ``count``: row ``b``, one token each: the token step).  ``max_new`` is the most of ``count`` (it may be more); all these numbers stay on the device.

    pages = paged.new_pages(n, kv_heads, head_dim, device)
    q = paged.append(pages, qkv, table, start, max_new, cos_sin, H)        # rotate; keys and values into the pages
    o = paged.attn(pages, q, table, start, max_new, H, scale)              # the same table and start: attention up to each token's own place

Keys and values that are not finite are held as zero.  That, and numbers that do not fit (a page outside the pool, tokens past the table),
set the device's status word, which ``_lib.check_status`` reads.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional

import torch

from ..utils import canary as CA
from . import _lib

c_int, c_ll, c_vp, c_float = ctypes.c_int, ctypes.c_longlong, ctypes.c_void_p, ctypes.c_float

PAGE = 64
HEAD_DIMS = (32, 64, 128)


class Pages(NamedTuple):
    """One layer's pool: codes ``k`` int8 [pages, kv_heads, 64, head_dim] and ``v`` int8 [pages, kv_heads, head_dim, 64], scales ``ks`` and ``vs`` fp32 [pages, kv_heads]."""
    k: torch.Tensor
    ks: torch.Tensor
    v: torch.Tensor
    vs: torch.Tensor


class PagedArgs(ctypes.Structure):
    _fields_ = [
        ("k", c_vp), ("ks", c_vp), ("v", c_vp), ("vs", c_vp),
        ("pages", c_int), ("KV", c_int), ("hd", c_int),
        ("table", c_vp), ("W", c_int),
        ("B", c_int), ("start", c_vp), ("first", c_vp), ("count", c_vp),
        ("max_new", c_int), ("rows", c_ll), ("is_bf16", c_int), ("status", c_vp),
    ]


_proto = None


def _protos():
    global _proto
    if _proto is None:
        L = _lib.lib()
        P = ctypes.POINTER(PagedArgs)
        L.gb_paged_append.argtypes = [P, c_vp, c_ll, c_int, c_vp, c_ll, c_vp, c_vp, c_float, c_vp, c_int, c_int, c_vp]
        L.gb_paged_read.argtypes = [P, c_vp, c_ll, c_vp, c_ll, c_vp]
        L.gb_paged_attn.argtypes = [P, c_vp, c_ll, c_int, c_float, c_int, c_vp, c_ll, c_vp, c_ll, c_vp]
        L.gb_paged_attn_ws.argtypes = [P, c_int, c_int]
        L.gb_paged_attn_ws.restype = c_ll
        _proto = L
    return _proto


def new_pages(pages: int, kv_heads: int, head_dim: int, device) -> Pages:
    """An empty pool for ``pages * 64`` tokens."""
    if head_dim not in HEAD_DIMS:
        raise ValueError("paged caches support head_dim 32, 64 and 128")
    if pages < 1 or kv_heads < 1:
        raise ValueError("a pool needs at least one page and one key head")
    i8, f32 = dict(dtype=torch.int8, device=device), dict(dtype=torch.float32, device=device)
    return Pages(CA.zeros(pages, kv_heads, PAGE, head_dim, **i8), CA.zeros(pages, kv_heads, **f32),
                 CA.zeros(pages, kv_heads, head_dim, PAGE, **i8), CA.zeros(pages, kv_heads, **f32))


def _args(p: Pages, table, start, max_new, first, count, rows, dtype, what) -> PagedArgs:
    k, ks, v, vs = p
    dev = k.device
    pages, KV, page, hd = k.shape
    if hd not in HEAD_DIMS or page != PAGE or v.shape != (pages, KV, hd, PAGE) or ks.shape != (pages, KV) or vs.shape != (pages, KV):
        raise ValueError(f"{what}: the pool's tensors do not belong together: {tuple(k.shape)}, {tuple(v.shape)}, {tuple(ks.shape)}, {tuple(vs.shape)}")
    if k.dtype != torch.int8 or v.dtype != torch.int8 or ks.dtype != torch.float32 or vs.dtype != torch.float32:
        raise ValueError(f"{what}: a pool holds int8 codes and float32 scales")
    if dtype != torch.float16 and dtype != torch.bfloat16:
        raise ValueError(f"{what}: rows are float16 or bfloat16, not {dtype}")
    if table.dim() != 2 or start.dim() != 1 or start.shape[0] != table.shape[0]:
        raise ValueError(f"{what}: table is [B, width] and start [B], got {tuple(table.shape)} and {tuple(start.shape)}")
    B, W = table.shape
    if (first is None) != (count is None):
        raise ValueError(f"{what}: first and count come together")
    for t in (table, start) if count is None else (table, start, first, count):
        if t.dtype != torch.int32 or t.device != dev or not t.is_contiguous() or (t is not table and t.shape != (B,)):
            raise ValueError(f"{what}: table, start, first and count are contiguous int32 tensors on the pool's device, one number a sequence")
    if not (k.is_contiguous() and v.is_contiguous() and ks.is_contiguous() and vs.is_contiguous() and v.device == dev and ks.device == dev and vs.device == dev):
        raise ValueError(f"{what}: the pool's tensors are contiguous and on one device")
    if max_new < 0 or max_new > W * PAGE or (count is None and max_new != 1):
        raise ValueError(f"{what}: max_new is {max_new}; a table of {W} pages holds {W * PAGE} tokens" +
                         (", and without count every sequence has one" if count is None else ""))
    if dev.type != "cuda" or dev.index != torch.cuda.current_device():
        raise ValueError(f"{what}: the pool is on {dev}, which is not the current device")
    return PagedArgs(k.data_ptr(), ks.data_ptr(), v.data_ptr(), vs.data_ptr(), pages, KV, hd, table.data_ptr(), W, B, start.data_ptr(),
                     None if first is None else first.data_ptr(), None if count is None else count.data_ptr(), max_new, rows, dtype == torch.bfloat16,
                     _lib.status_word(dev).data_ptr())


def _stream(dev):
    return torch.cuda.current_stream(dev.index).cuda_stream


def _rows(t, width, dtype, dev, what):
    """Checks a [rows, width] tensor of 16-bit rows."""
    if t.dim() != 2 or t.shape[1] != width or t.dtype != dtype or t.device != dev or t.stride(1) != 1 or t.stride(0) % 8 or t.data_ptr() % 16:
        raise ValueError(f"{what}: expected rows of {width} {dtype} numbers on {dev}, each 16-byte aligned, got {tuple(t.shape)} {t.dtype} "
                         f"on {t.device} with strides {t.stride()}")
    return t


def _out(t, rows, width, dtype, dev, what):
    if t is None:
        return torch.empty(rows, width, dtype=dtype, device=dev)
    if t.shape[0] < rows:
        raise ValueError(f"{what}: {t.shape[0]} rows for the results of {rows}")
    return _rows(t, width, dtype, dev, what)


def append(pages: Pages, qkv, table, start, max_new: int, cos_sin, H: int, *, first=None, count=None, q_out=None, qw=None, kw=None, eps: float = 1e-6,
           rope_type: int = 0):
    """Rotated queries [rows, H * hd] of the rows ``qkv`` [rows, (H + 2 * kv_heads) * hd]; their keys, rotated, and values go into the pages.
    ``cos_sin``: :func:`kernels.rope_table`; ``rope_type`` 0 turns neighbouring dimensions, 1 the halves of a head; ``qw``, ``kw``: weights of an RMS norm of
    each head ahead of the rotation, or None.  Rows of no sequence are not written (without ``q_out`` they hold anything)."""
    KV, hd, dev = pages.k.shape[1], pages.k.shape[3], pages.k.device
    if H < 1 or H % KV:
        raise ValueError(f"paged append: {H} query heads for {KV} key heads")
    _rows(qkv, (H + 2 * KV) * hd, qkv.dtype, dev, "paged append")
    q_out = _out(q_out, qkv.shape[0], H * hd, qkv.dtype, dev, "paged append")
    if cos_sin.dim() != 2 or cos_sin.shape[1] != hd or cos_sin.dtype != torch.float32 or cos_sin.device != dev or not cos_sin.is_contiguous():
        raise ValueError("paged append: cos_sin is a contiguous float32 table [positions, head_dim] on the pool's device")
    for w in (qw, kw):
        if w is not None and (w.shape != (hd,) or w.dtype != torch.float32 or w.device != dev or not w.is_contiguous()):
            raise ValueError("paged append: norm weights are contiguous float32 [head_dim] on the pool's device")
    if rope_type not in (0, 1):
        raise ValueError(f"paged append: rope_type is 0 or 1, not {rope_type}")
    a = _args(pages, table, start, max_new, first, count, qkv.shape[0], qkv.dtype, "paged append")
    rc = _protos().gb_paged_append(ctypes.byref(a), qkv.data_ptr(), qkv.stride(0), H, q_out.data_ptr(), q_out.stride(0),
                                   None if qw is None else qw.data_ptr(), None if kw is None else kw.data_ptr(), eps, cos_sin.data_ptr(), cos_sin.shape[0],
                                   rope_type, _stream(dev))
    _lib.check_rc(rc, "gb_paged_append")
    return q_out


def attn(pages: Pages, q, table, start, max_new: int, H: int, scale: float, *, window: int = 0, first=None, count=None, out=None, scratch=None):
    """Attention of the new tokens' queries ``q`` [rows, H * hd] over the pages, which hold the new tokens' keys already (:func:`append` with the same
    ``start``): each sees the tokens up to its own place, the last ``window`` of them where that is not 0.  Rows of no sequence are not
    written (without ``out`` they hold anything).  ``scratch``: float32, :func:`attn_scratch` numbers, one call's at a time; without it the call allocates its own."""
    KV, hd, dev = pages.k.shape[1], pages.k.shape[3], pages.k.device
    if H < 1 or H % KV:
        raise ValueError(f"paged attention: {H} query heads for {KV} key heads")
    if not scale > 0 or window < 0:
        raise ValueError(f"paged attention: scale is positive and window not negative, got {scale} and {window}")
    _rows(q, H * hd, q.dtype, dev, "paged attention")
    out = _out(out, q.shape[0], H * hd, q.dtype, dev, "paged attention")
    a = _args(pages, table, start, max_new, first, count, q.shape[0], q.dtype, "paged attention")
    L = _protos()
    need = L.gb_paged_attn_ws(ctypes.byref(a), H, window)
    if need > 0 and scratch is None:
        scratch = torch.empty(need, dtype=torch.float32, device=dev)
    if need > 0 and (scratch.dtype != torch.float32 or scratch.device != dev or not scratch.is_contiguous() or scratch.numel() < need):
        raise ValueError(f"paged attention: scratch is {need} contiguous float32 numbers on the pool's device")
    rc = L.gb_paged_attn(ctypes.byref(a), q.data_ptr(), q.stride(0), H, scale, window, out.data_ptr(), out.stride(0),
                         scratch.data_ptr() if need > 0 else None, need, _stream(dev))
    _lib.check_rc(rc, "gb_paged_attn")
    return out


def attn_scratch(B: int, width: int, kv_heads: int, head_dim: int, max_new: int, H: int, window: int = 0) -> int:
    """float32 numbers that :func:`attn` needs for ``B`` sequences with tables of ``width`` pages."""
    a = PagedArgs()
    for f in ("k", "ks", "v", "vs", "table", "start", "status"):
        setattr(a, f, 4096)                                   # sizes alone count
    a.pages, a.KV, a.hd, a.W, a.B, a.max_new, a.rows = 1, kv_heads, head_dim, width, B, max_new, B * max_new
    need = _protos().gb_paged_attn_ws(ctypes.byref(a), H, window)
    if need < 0:
        _lib.check_rc(int(need), "gb_paged_attn_ws")
    return int(need)


def read(pages: Pages, table, start, max_new: int, dtype, rows: int, *, first=None, count=None, k_out=None, v_out=None):
    """The tokens ``start[b]`` ... ``start[b] + count[b] - 1`` of the sequences as 16-bit rows: (k, v), each [rows, kv_heads, hd].  ``k_out``, ``v_out``:
    [rows, kv_heads * hd] tensors to write to."""
    KV, hd, dev = pages.k.shape[1], pages.k.shape[3], pages.k.device
    k = _out(k_out, rows, KV * hd, dtype, dev, "paged read")
    v = _out(v_out, rows, KV * hd, dtype, dev, "paged read")
    a = _args(pages, table, start, max_new, first, count, rows, dtype, "paged read")
    rc = _protos().gb_paged_read(ctypes.byref(a), k.data_ptr(), k.stride(0), v.data_ptr(), v.stride(0), _stream(dev))
    _lib.check_rc(rc, "gb_paged_read")
    return k.unflatten(1, (KV, hd)), v.unflatten(1, (KV, hd))
