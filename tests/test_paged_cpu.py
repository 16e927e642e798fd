"""Refusals of the paged 8-bit cache's launchers, and the arithmetic its pages rest on.  Every refusal comes before anything is launched."""
import copy
import ctypes
import os
import pickle

import numpy as np
import pytest
import torch

from paged_oracle import PAGE, Seq, scale_of

from ghassan_b200.ops import _lib
from ghassan_b200.ops import paged as P


def pool(pages=4, KV=2, hd=64):
    return P.new_pages(pages, KV, hd, "cpu")


def i32(*x):
    return torch.tensor(x, dtype=torch.int32)


TABLE, START = torch.zeros(2, 3, dtype=torch.int32), i32(0, 0)
H, HD, KV = 4, 64, 2


def call(name, p=None, **kw):
    p = p or pool()
    a = dict(table=TABLE, start=START, max_new=1, first=None, count=None, rows=2, dtype=torch.float16)
    a.update(kw)
    common = dict(first=a["first"], count=a["count"])
    if name == "append":
        x = a.get("x", torch.zeros(a["rows"], (H + 2 * KV) * HD, dtype=a["dtype"]))
        return P.append(p, x, a["table"], a["start"], a["max_new"], a.get("cos_sin", torch.zeros(200, HD)), a.get("H", H), q_out=a.get("out"),
                        qw=a.get("qw"), rope_type=a.get("rope_type", 0), **common)
    if name == "attn":
        x = a.get("x", torch.zeros(a["rows"], H * HD, dtype=a["dtype"]))
        return P.attn(p, x, a["table"], a["start"], a["max_new"], a.get("H", H), a.get("scale", 0.1), window=a.get("window", 0), out=a.get("out"), **common)
    return P.read(p, a["table"], a["start"], a["max_new"], a["dtype"], a["rows"], k_out=a.get("out"), **common)


@pytest.mark.parametrize("name", ["append", "attn", "read"])
def test_refusals_of_every_call(name):
    good = pool()
    for why, kw in [
        ("int32", dict(table=TABLE.long())), ("int32", dict(start=START.long())), (r"\[B, width\]", dict(start=i32(0))), (r"\[B, width\]", dict(table=TABLE[0])),
        ("int32", dict(table=torch.zeros(3, 2, dtype=torch.int32).t())), ("together", dict(first=i32(0, 1))), ("together", dict(count=i32(1, 1))),
        ("int32", dict(first=i32(0, 1), count=i32(1))), ("max_new", dict(max_new=2)), ("max_new", dict(max_new=-1, first=i32(0, 1), count=i32(1, 1))),
        ("max_new", dict(max_new=3 * PAGE + 1, first=i32(0, 1), count=i32(1, 1))), ("float16 or bfloat16|16-byte", dict(dtype=torch.float32)),
        ("belong together", dict(p=good._replace(v=good.v[:3]))), ("belong together", dict(p=good._replace(ks=good.ks[:2]))),
        ("int8", dict(p=good._replace(k=good.k.to(torch.uint8)))), ("float32", dict(p=good._replace(vs=good.vs.double()))),
        ("contiguous", dict(p=good._replace(ks=torch.zeros(2, 4).t()))), ("current device", dict()),
    ]:
        with pytest.raises(ValueError, match=why):
            call(name, **kw)


def test_refusals_of_rows_and_options():
    wide = torch.zeros(2, (H + 2 * KV) * HD + 4, dtype=torch.float16)
    for name, why, kw in [
        ("append", "query heads", dict(H=3)), ("attn", "query heads", dict(H=5)), ("attn", "query heads", dict(H=0)),
        ("append", "16-byte", dict(x=wide[:, :-4])), ("append", "16-byte", dict(x=wide[:, 4:])), ("append", "16-byte", dict(x=wide)),
        ("append", "cos_sin", dict(cos_sin=torch.zeros(200, 32))), ("append", "cos_sin", dict(cos_sin=torch.zeros(200, HD, dtype=torch.float64))),
        ("append", "norm weights", dict(qw=torch.ones(32))), ("append", "rope_type", dict(rope_type=2)),
        ("attn", "scale", dict(scale=0.0)), ("attn", "scale", dict(scale=float("nan"))), ("attn", "scale", dict(window=-1)),
        ("attn", "16-byte", dict(x=torch.zeros(2, 3 * HD, dtype=torch.float16))), ("attn", "16-byte", dict(out=torch.zeros(2, H * HD, dtype=torch.bfloat16))),
        ("attn", "rows for", dict(out=torch.zeros(1, H * HD, dtype=torch.float16))), ("read", "rows for", dict(out=torch.zeros(1, KV * HD, dtype=torch.float16))),
    ]:
        with pytest.raises(ValueError, match=why):
            call(name, **kw)
    for bad in (48, 256, 0):
        with pytest.raises(ValueError, match="head_dim"):
            P.new_pages(4, 2, bad, "cpu")
    with pytest.raises(ValueError, match="at least one page"):
        P.new_pages(0, 2, 64, "cpu")


def test_a_pool_that_was_good_is_checked_again_when_it_is_another():
    p = pool()
    with pytest.raises(ValueError, match="current device"):        # all is well but for the device
        call("attn", p)
    p.k.data = p.k.data[:, :1].contiguous()
    with pytest.raises(ValueError, match="belong together"):
        call("attn", p)
    p = pool()
    P._pool(p, "")
    for q in (copy.copy(p), copy.deepcopy(p), pickle.loads(pickle.dumps(p))):
        assert isinstance(q, P.Pages) and not hasattr(q, "_known")


def test_a_pool_that_changed_in_place_is_another():
    """Tensors that are where they were, with another number of pages, type or order: nothing of an earlier call's check is kept."""
    def halved(t):
        t.resize_(2, *t.shape[1:])

    def turned(t):
        t.transpose_(0, 1)

    def retyped(t):
        t.data = t.data.view(torch.uint8 if t.dtype == torch.int8 else torch.int32)

    for change in (halved, turned, retyped):
        for i in range(4):
            p = pool()
            with pytest.raises(ValueError, match="current device"):    # all is well but for the device
                call("attn", p)
            at = p[i].data_ptr()
            change(p[i])
            assert p[i].data_ptr() == at
            for name in ("append", "attn", "read"):
                with pytest.raises(ValueError, match="belong together"):
                    call(name, p)


@pytest.mark.parametrize("window,least", [(2 ** 32 + 5, 3 * PAGE), (2 ** 31, 3 * PAGE), (3 * PAGE - 1, 3 * PAGE - 1), (0, 0)])
def test_a_window_past_32_bits_is_not_a_short_one(window, least, monkeypatch):
    seen = []

    class Lib:
        def __getattr__(self, name):
            return lambda *a: seen.append((name, a)) or 0

    monkeypatch.setattr(P, "_protos", Lib)
    monkeypatch.setattr(P, "_scratch", {})
    monkeypatch.setattr(P, "_args", lambda *a: b"")
    monkeypatch.setattr(P, "_raw_stream", lambda dev: 0)
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    call("attn", window=window)
    assert [(n, a[2] if n == "gb_paged_attn_ws" else a[5]) for n, a in seen] == [("gb_paged_attn_ws", least), ("gb_paged_attn", least)]


@pytest.mark.skipif(not _lib.available(), reason="the kernel library is not built")
def test_the_c_launchers_refuse_before_they_touch_the_device():
    """Argument blocks that only look like pointers: every call returns a code."""
    L = ctypes.CDLL(os.path.join(os.path.dirname(_lib.__file__), "..", "_gb200_cuda.so"))
    for n, t in (("gb_paged_append", [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_longlong, ctypes.c_int, ctypes.c_void_p, ctypes.c_longlong, ctypes.c_void_p,
                                      ctypes.c_void_p, ctypes.c_float, ctypes.c_void_p, ctypes.c_int, ctypes.c_int, ctypes.c_void_p]),
                 ("gb_paged_attn", [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_longlong, ctypes.c_int, ctypes.c_float, ctypes.c_int,
                                   ctypes.c_void_p, ctypes.c_longlong, ctypes.c_void_p, ctypes.c_longlong, ctypes.c_void_p]),
                 ("gb_paged_read", [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_longlong, ctypes.c_void_p, ctypes.c_longlong, ctypes.c_void_p])):
        getattr(L, n).argtypes = t

    def block(**kw):
        a = P.PagedArgs()
        for f in ("k", "ks", "v", "vs", "table", "start", "status"):
            setattr(a, f, 4096)
        a.pages, a.KV, a.hd, a.W, a.B, a.max_new, a.rows = 4, 2, 64, 3, 2, 1, 2
        for k, v in kw.items():
            setattr(a, k, v)
        return ctypes.addressof(a), a

    def three(ptr, x=4096, ldx=512, h=4, out=4096, ldo=256, scale=0.1, window=0, cs=4096, positions=9, rope=0):
        return (L.gb_paged_append(ptr, x, ldx, h, out, ldo, None, None, 1e-6, cs, positions, rope, None),
                L.gb_paged_attn(ptr, x, ldx, h, scale, window, out, ldo, None, 0, None), L.gb_paged_read(ptr, out, ldo, out, ldo, None))

    assert three(None) == (-1, -1, -1)
    for kw, rc in [(dict(k=None), -1), (dict(status=None), -1), (dict(start=None), -1), (dict(hd=96), -2), (dict(KV=0), -3), (dict(pages=0), -3), (dict(W=0), -3),
                   (dict(B=-1), -3), (dict(max_new=-1), -3), (dict(max_new=193), -3), (dict(rows=2 ** 31), -3), (dict(W=2 ** 26), -3), (dict(k=4097), -4),
                   (dict(v=4104), -4)]:
        ptr, keep = block(**kw)
        assert three(ptr) == (rc, rc, rc), kw
    ptr, keep = block(first=4096)
    assert three(ptr) == (-1, -1, -1)                         # first without count
    ptr, keep = block(W=4000, B=200)
    assert three(ptr)[1] == -5                                # no workspace
    ptr, keep = block()
    assert three(ptr, h=3)[:2] == (-1, -1) and three(ptr, x=4098)[:2] == (-4, -4) and three(ptr, out=4098) == (-4, -4, -4) and three(ptr, ldx=504)[0] == -4
    assert three(ptr, ldo=260) == (-4, -4, -4) and three(ptr, scale=0.0)[1] == -1 and three(ptr, window=-1)[1] == -1
    assert three(ptr, cs=None)[0] == -1 and three(ptr, positions=0)[0] == -1 and three(ptr, rope=2)[0] == -1
    ptr, keep = block(B=0)
    assert three(ptr) == (0, 0, 0)                            # nothing to do is no error
    ptr, keep = block(max_new=0)
    assert three(ptr) == (0, 0, 0)


@pytest.mark.skipif(not _lib.available(), reason="the kernel library is not built")
def test_limits_go_by_the_rows_that_there_are(monkeypatch):
    """max_new may be the most that tables hold: a call's own rows say how much there is to do."""
    L = ctypes.CDLL(os.path.join(os.path.dirname(_lib.__file__), "..", "_gb200_cuda.so"))
    L.gb_paged_attn_ws.argtypes, L.gb_paged_attn_ws.restype = [ctypes.c_void_p, ctypes.c_int, ctypes.c_int], ctypes.c_longlong

    def need(B, W, max_new, rows, KV=2, heads=4):
        return L.gb_paged_attn_ws(P._pack(4096, 4096, 4096, 4096, 1, KV, 64, 4096, W, B, 4096, 4096, 4096, max_new, rows, 0, 4096), heads, 0)

    monkeypatch.setattr(P, "_protos", lambda: L)
    monkeypatch.setattr(P, "_scratch", {})
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    for B, W, max_new, rows in [(65535, 700, 44000, 100000), (3, 70000, 70000 * PAGE, 50), (1, 2 ** 24, 2 ** 30, 8), (1024, 32, 2048, 9000), (200, 32, 1, 200),
                                (3, 8, 1, 3), (3, 8, 8, 11), (300, 2 ** 20, 5, 700)]:
        assert P.attn_scratch(B, W, 2, 64, max_new, 4) >= need(B, W, max_new, rows) >= 0, (B, W, max_new, rows)
    assert need(1, 2 ** 24, 2 ** 30, 2 ** 30) == -3           # this many rows are too many indeed


def test_scales_are_the_smallest_powers_of_two():
    for x in [1e-30, 0.3, 1.0, 126.9, 127.0, np.nextafter(np.float32(127), np.float32(200)), 254.0, 6e4, 3e38]:
        s = float(scale_of(np.float32(x)))
        assert np.log2(s) == round(np.log2(s)) and 127 * s >= np.float32(x) and (127 * s / 2 < np.float32(x) or s == 2.0 ** -120)
        assert abs(np.rint(np.float32(x) / np.float32(s))) <= 127


def test_held_values_are_near_what_was_appended():
    """In one call within half a step of the page's scale; token by token within one step, since rescalings add at most 1/2 + 1/4 + ... halves."""
    r = np.random.default_rng(0)
    k, v = ((r.standard_normal((150, 2, 32)) * np.exp(r.standard_normal((150, 1, 1)))).astype(np.float32) for _ in range(2))
    whole, single = Seq(2, 32), Seq(2, 32)
    whole.append(k, v)
    for i in range(150):
        single.append(k[i:i + 1], v[i:i + 1])
    assert np.array_equal(whole.scales, single.scales)
    step = whole.scales[:, np.arange(150) // PAGE][..., None]
    for s, most in ((whole, 0.5), (single, 1.0)):
        for got, want, st in zip(s.held(), (k, v), step):
            assert (np.abs(got - want) <= most * st).all()
