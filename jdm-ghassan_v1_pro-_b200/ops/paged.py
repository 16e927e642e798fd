"""Launchers of the paged 8-bit key/value cache (``csrc/cuda/paged*.cu``; layout and contract in ``gb_paged.h``).

A pool of pages of 64 tokens holds keys and values as codes of 8 bits with one scale a page and key head.  A page belongs to whoever's table names it; the
pages of one text may be anywhere in the pool, and one table serves all layers of a model (a pool each).  Every call takes ``B`` sequences:
``start[b]`` tokens are in the pages ``table[b]`` already, and the call's own ``count[b]`` ones are the rows ``first[b]`` ... of its tensors (without
``first`` and ``count``: row ``b``, one token each: the token step).  ``max_new`` is the most of ``count`` (it may be more); all these numbers stay on the device.

    pages = paged.new_pages(n, kv_heads, head_dim, device)
    q = paged.append(pages, qkv, table, start, max_new, cos_sin, H)        # rotate; keys and values into the pages
    o = paged.attn(pages, q, table, start, max_new, H, scale)              # the same table and start: attention up to each token's own place

A page that one sequence appends to is in no other's table, nor twice in its own, and results do not lie over a call's inputs.
Keys and values that are not finite are held as zero.  That, and numbers that do not fit (a page outside the pool, tokens past the table),
set the device's status word, which ``_lib.check_status`` reads.
"""
from __future__ import annotations

import ctypes
import struct
from typing import NamedTuple

import torch

from ..utils import canary as CA
from . import _lib

c_int, c_ll, c_vp, c_float = ctypes.c_int, ctypes.c_longlong, ctypes.c_void_p, ctypes.c_float

PAGE = 64
HEAD_DIMS = (32, 64, 128)


class Pages(NamedTuple):
    """One layer's pool: codes ``k`` int8 [pages, kv_heads, 64, head_dim] and ``v`` int8 [pages, kv_heads, head_dim, 64], scales ``ks`` and ``vs`` fp32 [pages, kv_heads],
    powers of two."""
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


# The same block as bytes: filling a ctypes structure took 2 us of a call's 20, and a token step is a few of them a layer.
_pack = struct.Struct("@4P3iP2i3PiqiP").pack
assert struct.calcsize("@4P3iP2i3PiqiP") == ctypes.sizeof(PagedArgs)
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)      # what current_stream() asks, in 0.1 us instead of 3
_status_ptr: dict = {}
_scratch: dict = {}              # scratch numbers by sizes
_proto = None


def _protos():
    global _proto
    if _proto is None:
        L = _lib.lib()
        L.gb_paged_append.argtypes = [c_vp, c_vp, c_ll, c_int, c_vp, c_ll, c_vp, c_vp, c_float, c_vp, c_int, c_int, c_vp]
        L.gb_paged_read.argtypes = [c_vp, c_vp, c_ll, c_vp, c_ll, c_vp]
        L.gb_paged_attn.argtypes = [c_vp, c_vp, c_ll, c_int, c_float, c_int, c_vp, c_ll, c_vp, c_ll, c_vp]
        L.gb_paged_attn_ws.argtypes = [c_vp, c_int, c_int]
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


def _pool(p: Pages, what):
    """(pages, kv_heads, head_dim, device index, the four addresses) of a pool whose tensors belong together: every call looks, since a tensor can be resized or
    replaced in place, and the kernels write to wherever its sizes say."""
    k, ks, v, vs = p
    if k.dim() == 4:
        pages, KV, page, hd = k.shape
        dev = k.get_device()
        if (page == PAGE and hd in HEAD_DIMS and v.shape == (pages, KV, hd, PAGE) and ks.shape == (pages, KV) and vs.shape == (pages, KV)
                and k.dtype is torch.int8 and v.dtype is torch.int8 and ks.dtype is torch.float32 and vs.dtype is torch.float32
                and k.is_contiguous() and v.is_contiguous() and ks.is_contiguous() and vs.is_contiguous()
                and v.get_device() == dev and ks.get_device() == dev and vs.get_device() == dev):
            return pages, KV, hd, dev, (k.data_ptr(), ks.data_ptr(), v.data_ptr(), vs.data_ptr())
    raise ValueError(f"{what}: the pool's tensors do not belong together: contiguous int8 codes [pages, kv_heads, 64, head_dim] and [pages, kv_heads, head_dim, 64], float32 "
                     f"scales [pages, kv_heads], on one device; got " + ", ".join(f"{tuple(t.shape)} {t.dtype} on {t.device}" for t in p))


def _args(p: Pages, pool, table, start, max_new, first, count, rows, dtype, what) -> bytes:
    pages, KV, hd, dev, at = pool
    if dtype is not torch.float16 and dtype is not torch.bfloat16:
        raise ValueError(f"{what}: rows are float16 or bfloat16, not {dtype}")
    if table.dim() != 2 or start.dim() != 1 or start.shape[0] != table.shape[0]:
        raise ValueError(f"{what}: table is [B, width] and start [B], got {tuple(table.shape)} and {tuple(start.shape)}")
    B, W = table.shape
    if (first is None) != (count is None):
        raise ValueError(f"{what}: first and count come together")
    for t in (table, start) if count is None else (table, start, first, count):
        if t.dtype is not torch.int32 or t.get_device() != dev or not t.is_contiguous() or (t is not table and t.numel() != B):
            raise ValueError(f"{what}: table, start, first and count are contiguous int32 tensors on the pool's device, one number a sequence")
    if max_new < 0 or max_new > W * PAGE or (count is None and max_new != 1):
        raise ValueError(f"{what}: max_new is {max_new}; a table of {W} pages holds {W * PAGE} tokens" +
                         (", and without count every sequence has one" if count is None else ""))
    if dev < 0 or dev != torch._C._cuda_getDevice():
        raise ValueError(f"{what}: the pool is on {p.k.device}, which is not the current device")
    status = _status_ptr.get(dev)
    if status is None:
        status = _status_ptr[dev] = _lib.status_word(p.k.device).data_ptr()
    return _pack(*at, pages, KV, hd, table.data_ptr(), W, B, start.data_ptr(),
                 0 if first is None else first.data_ptr(), 0 if count is None else count.data_ptr(), max_new, rows, dtype is torch.bfloat16, status)


def _rows(t, width, dtype, dev, what):
    """Checks a [rows, width] tensor of 16-bit rows; its row pitch."""
    if t.dim() == 2:
        ld, one = t.stride()
        if t.shape[0] <= 1:                                   # whose pitch means nothing
            ld = width
        if t.shape[1] == width and one == 1 and ld >= width and ld % 8 == 0 and t.dtype is dtype and t.get_device() == dev and t.data_ptr() % 16 == 0:
            return ld
    raise ValueError(f"{what}: expected rows of {width} {dtype} numbers on the pool's device, each 16-byte aligned, got {tuple(t.shape)} {t.dtype} "
                     f"on {t.device} with strides {t.stride()}")


def _out(t, rows, width, like, dtype, dev, what):
    """The tensor for ``rows`` rows of results (of ``like``'s type) and its row pitch."""
    if t is None:
        return like.new_empty((rows, width)), width
    if t.shape[0] < rows:
        raise ValueError(f"{what}: {t.shape[0]} rows for the results of {rows}")
    return t, _rows(t, width, dtype, dev, what)


def append(pages: Pages, qkv, table, start, max_new: int, cos_sin, H: int, *, first=None, count=None, q_out=None, qw=None, kw=None, eps: float = 1e-6,
           rope_type: int = 0):
    """Rotated queries [rows, H * hd] of the rows ``qkv`` [rows, (H + 2 * kv_heads) * hd]; their keys, rotated, and values go into the pages.
    ``cos_sin``: :func:`kernels.rope_table`; ``rope_type`` 0 turns neighbouring dimensions, 1 the halves of a head; ``qw``, ``kw``: weights of an RMS norm of
    each head ahead of the rotation, or None.  Rows of no sequence are not written (without ``q_out`` they hold anything)."""
    pool = _pool(pages, "paged append")
    _, KV, hd, dev, _ = pool
    if H < 1 or H % KV:
        raise ValueError(f"paged append: {H} query heads for {KV} key heads")
    rows, dtype = qkv.shape[0], qkv.dtype
    ld = _rows(qkv, (H + 2 * KV) * hd, dtype, dev, "paged append")
    q_out, ld_q = _out(q_out, rows, H * hd, qkv, dtype, dev, "paged append")
    if cos_sin.dim() != 2 or cos_sin.shape[1] != hd or cos_sin.dtype is not torch.float32 or cos_sin.get_device() != dev or not cos_sin.is_contiguous():
        raise ValueError("paged append: cos_sin is a contiguous float32 table [positions, head_dim] on the pool's device")
    for w in (qw, kw):
        if w is not None and (w.shape != (hd,) or w.dtype is not torch.float32 or w.get_device() != dev or not w.is_contiguous()):
            raise ValueError("paged append: norm weights are contiguous float32 [head_dim] on the pool's device")
    if rope_type not in (0, 1):
        raise ValueError(f"paged append: rope_type is 0 or 1, not {rope_type}")
    a = _args(pages, pool, table, start, max_new, first, count, rows, dtype, "paged append")
    if not (rows and max_new):
        return q_out
    rc = _protos().gb_paged_append(a, qkv.data_ptr(), ld, H, q_out.data_ptr(), ld_q, None if qw is None else qw.data_ptr(),
                                   None if kw is None else kw.data_ptr(), eps, cos_sin.data_ptr(), cos_sin.shape[0], rope_type, _raw_stream(dev))
    if rc:
        _lib.check_rc(rc, "gb_paged_append")
    return q_out


def attn(pages: Pages, q, table, start, max_new: int, H: int, scale: float, *, window: int = 0, first=None, count=None, out=None, scratch=None):
    """Attention of the new tokens' queries ``q`` [rows, H * hd] over the pages, which hold the new tokens' keys already (:func:`append` with the same
    ``start``): each sees the tokens up to its own place, the last ``window`` of them where that is not 0.  Rows of no sequence are not
    written (without ``out`` they hold anything).  ``scratch``: float32, :func:`attn_scratch` numbers, one call's at a time; without it the call allocates its own."""
    pool = _pool(pages, "paged attention")
    _, KV, hd, dev, _ = pool
    if H < 1 or H % KV:
        raise ValueError(f"paged attention: {H} query heads for {KV} key heads")
    if not scale > 0 or window < 0:
        raise ValueError(f"paged attention: scale is positive and window not negative, got {scale} and {window}")
    rows, dtype = q.shape[0], q.dtype
    ld = _rows(q, H * hd, dtype, dev, "paged attention")
    out, ld_o = _out(out, rows, H * hd, q, dtype, dev, "paged attention")
    a = _args(pages, pool, table, start, max_new, first, count, rows, dtype, "paged attention")
    B, W = table.shape
    if not (B and rows and max_new):
        return out
    window = min(window, W * PAGE)                            # as many as there can be, and few enough for the interface's 32 bits
    L = _protos()
    need = attn_scratch(B, W, KV, hd, max_new, H, window)
    if need:
        if scratch is None:
            scratch = q.new_empty(need, dtype=torch.float32)
        elif scratch.dtype is not torch.float32 or scratch.get_device() != dev or not scratch.is_contiguous() or scratch.numel() < need or scratch.data_ptr() % 16:
            raise ValueError(f"paged attention: scratch is {need} contiguous float32 numbers on the pool's device, 16-byte aligned")
    rc = L.gb_paged_attn(a, q.data_ptr(), ld, H, scale, window, out.data_ptr(), ld_o, scratch.data_ptr() if need else None, need, _raw_stream(dev))
    if rc:
        _lib.check_rc(rc, "gb_paged_attn")
    return out


def attn_scratch(B: int, width: int, kv_heads: int, head_dim: int, max_new: int, H: int, window: int = 0) -> int:
    """float32 numbers that :func:`attn` needs on the current device for ``B`` sequences with tables of ``width`` pages."""
    window = min(window, width * PAGE)
    key = (B, width, kv_heads, head_dim, max_new, H, window, torch._C._cuda_getDevice())
    need = _scratch.get(key)
    if need is None:
        # sizes alone count, and rows do not: with fewer of them a launch takes more sequences, which need no less
        a = _pack(4096, 4096, 4096, 4096, 1, kv_heads, head_dim, 4096, width, B, 4096, 0, 0, max_new, 1, 0, 4096)
        need = _protos().gb_paged_attn_ws(a, H, window)
        if need < 0:
            _lib.check_rc(int(need), "gb_paged_attn_ws")
        if len(_scratch) > 4096:
            _scratch.clear()
        _scratch[key] = need
    return need


def read(pages: Pages, table, start, max_new: int, dtype, rows: int, *, first=None, count=None, k_out=None, v_out=None):
    """The tokens ``start[b]`` ... ``start[b] + count[b] - 1`` of the sequences as 16-bit rows: (k, v), each [rows, kv_heads, hd].  ``k_out``, ``v_out``:
    [rows, kv_heads * hd] tensors to write to."""
    pool = _pool(pages, "paged read")
    _, KV, hd, dev, _ = pool
    if rows < 0:
        raise ValueError(f"paged read: {rows} rows")
    if dtype is not torch.float16 and dtype is not torch.bfloat16:
        raise ValueError(f"paged read: rows are float16 or bfloat16, not {dtype}")
    if k_out is None or v_out is None:
        k, v = pages.k.new_empty((2, rows, KV, hd), dtype=dtype).unbind(0)
        at_k, at_v, ld_k, ld_v = k.data_ptr(), v.data_ptr(), KV * hd, KV * hd
    if k_out is not None:
        k_out, ld_k = _out(k_out, rows, KV * hd, None, dtype, dev, "paged read")
        at_k, k = k_out.data_ptr(), k_out.unflatten(1, (KV, hd))
    if v_out is not None:
        v_out, ld_v = _out(v_out, rows, KV * hd, None, dtype, dev, "paged read")
        at_v, v = v_out.data_ptr(), v_out.unflatten(1, (KV, hd))
    a = _args(pages, pool, table, start, max_new, first, count, rows, dtype, "paged read")
    if not (rows and max_new):
        return k, v
    rc = _protos().gb_paged_read(a, at_k, ld_k, at_v, ld_v, _raw_stream(dev))
    if rc:
        _lib.check_rc(rc, "gb_paged_read")
    return k, v
