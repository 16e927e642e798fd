"""Paged attention of few rows over tables of more than 16 pages, whatever the texts' lengths: pages are dealt evenly to all warps there, and pieces joined in and across blocks.
Engines are in it by default.  Windows, missing pages, queries that are not numbers, captured steps; the engine with windows and batches, every token of every sequence compared."""
import math

import numpy as np
import pytest
import torch

import test_paged_engine_gpu as E
from paged_oracle import PAGE, Pool, Seq, rotate
from test_paged_gpu import DT, check_attn, cos_sin, i32, ops, seqs_of

pytestmark = pytest.mark.gpu
WIDE = 40


def filled(P, lens, KV, hd, seed, spare=4):
    seqs = seqs_of(lens, KV, hd, seed)
    pool = Pool(P, sum((n + PAGE - 1) // PAGE for n in lens) + spare, KV, hd, seed=seed)
    table = pool.table(lens, WIDE)
    for b, s in enumerate(seqs):
        pool.fill(table, b, s)
    return seqs, pool, table


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("hd,H,KV", [(32, 4, 2), (64, 12, 4), (128, 8, 2), (128, 5, 5), (64, 7, 1), (64, 16, 1)])
@pytest.mark.parametrize("n", [1, 2])
@pytest.mark.parametrize("window", [0, 1000, 1090])
def test_lengths_and_long_windows(hd, H, KV, dt, n, window):
    P, L = ops()
    start = [0, 1, 62, 63, 999, 1000, 1063, 1300, 2400, 1920]
    if n * H // KV > 16:
        start = start[:3]
    seqs, pool, table = filled(P, [s + n for s in start], KV, hd, 1)
    B = len(start)
    rows = B * (n + 1)
    first = [b * (n + 1) for b in range(B)]
    q = torch.randn(rows, H * hd, device="cuda", generator=torch.Generator("cuda").manual_seed(n)).to(DT[dt])
    out = torch.full_like(q, 3.0)
    P.attn(pool.p, q, table, i32(start), n, H, hd ** -0.5, window=window, first=i32(first), count=i32([n] * B), out=out)
    L.check_status()
    check_attn(out, q, seqs, start, [n] * B, first, hd ** -0.5, window, dt, H, hd)
    left = torch.ones(rows, dtype=torch.bool)
    for f in first:
        left[f:f + n] = False
    assert (out[left.cuda()] == 3).all()


@pytest.mark.parametrize("B", [1, 7, 300])
@pytest.mark.parametrize("window", [0, 1001])
def test_ragged_batches(B, window):
    """Counts of none to five tokens; 300 sequences are more pages than warps, so that pieces lie inside, at and across a warp's and a block's run."""
    P, L = ops()
    KV, hd, H = 2, 64, 6
    r = np.random.default_rng(B)
    count = [int(x) for x in r.integers(0, 6, B)]
    count[-1] = 5
    start = [int(x) for x in np.where(r.random(B) < 0.2, r.integers(1000, 2500, B), r.integers(0, 300, B))]
    seqs, pool, table = filled(P, [s + n for s, n in zip(start, count)], KV, hd, B)
    first = [int(x) for x in np.cumsum([0] + count)[:-1]]
    q = torch.randn(sum(count), H * hd, device="cuda", generator=torch.Generator("cuda").manual_seed(B)).half()
    out = P.attn(pool.p, q, table, i32(start), 5, H, 0.125, window=window, first=i32(first), count=i32(count))
    L.check_status()
    check_attn(out, q, seqs, start, count, first, 0.125, window, "f16", H, hd)


@pytest.mark.parametrize("n", [1, 4])
def test_pages_behind_a_long_window_may_be_gone(n):
    P, L = ops()
    KV, hd, H, window, start = 2, 64, 6, 1100, 2200
    seqs, pool, table = filled(P, [start + n, 30 + n], KV, hd, 3)
    table[0, :(start - window + 1) // PAGE] = -1
    q = torch.randn(2 * n, H * hd, device="cuda").half()
    out = P.attn(pool.p, q, table, i32([start, 30]), n, H, 0.125, window=window, first=i32([0, n]), count=i32([n, n]))
    L.check_status()
    check_attn(out, q, seqs, [start, 30], [n, n], [0, n], 0.125, window, "f16", H, hd)


@pytest.mark.parametrize("n", [1, 3])
@pytest.mark.parametrize("missing", [0, 5, 13])
def test_a_missing_page_leaves_its_tokens_out(n, missing):
    """As if the other pages were all there is: the first, one in the middle, or the one with the queries' own keys."""
    P, L = ops()
    KV, hd, H, length = 2, 64, 4, 14 * PAGE
    seqs, pool, table = filled(P, [length, 200], KV, hd, 5)
    table[0, missing] = 2 ** 30
    q = torch.randn(2 * n, H * hd, device="cuda").half()
    out = P.attn(pool.p, q, table, i32([length - n, 200 - n]), n, H, 0.125, first=i32([0, n]), count=i32([n, n]))
    assert int(L.status_word()[0]) == 301
    L.status_word().zero_()
    check_attn(out, q, seqs, [0, 200 - n], [0, n], [0, n], 0.125, 0, "f16", H, hd)        # the other sequence
    k, v = seqs[0].held()
    x = q[:n].double().cpu().numpy().reshape(n, H, hd)
    for i in range(n):
        sees = (np.arange(length) <= length - n + i) & (np.arange(length) // PAGE != missing)
        for h in range(H):
            z = (k[sees, h // 2] @ x[i, h]) * 0.125
            p = np.exp(z - z.max())
            p /= p.sum()
            want, mag = p @ v[sees, h // 2], p @ np.abs(v[sees, h // 2])
            allow = (2.0 ** -11 + 2.0 ** -15) * mag
            allow = allow + 2.0 ** -11 * (np.abs(want) + allow) + 2.0 ** -25
            assert (np.abs(out[i, h * hd:(h + 1) * hd].double().cpu().numpy() - want) <= allow).all(), (i, h)


@pytest.mark.parametrize("n", [1, 3])
def test_all_pages_missing_is_nothing(n):
    """Rows that see no key at all are zero."""
    P, L = ops()
    KV, hd, H = 2, 64, 4
    seqs, pool, table = filled(P, [900, 200], KV, hd, 5)
    table[0] = -1
    q = torch.randn(2 * n, H * hd, device="cuda").half()
    out = P.attn(pool.p, q, table, i32([900 - n, 200 - n]), n, H, 0.125, first=i32([0, n]), count=i32([n, n]))
    assert int(L.status_word()[0]) == 301
    L.status_word().zero_()
    assert (out[:n] == 0).all()
    check_attn(out, q, seqs, [0, 200 - n], [0, n], [0, n], 0.125, 0, "f16", H, hd)


@pytest.mark.parametrize("n", [1, 3])
@pytest.mark.parametrize("length", [200, 2500])
def test_a_query_that_is_not_a_number_spoils_its_own_rows_only(n, length):
    P, L = ops()
    KV, hd, H, B = 2, 64, 4, 3
    seqs, pool, table = filled(P, [length] * B, KV, hd, 1)
    q = torch.randn(B * n, H * hd, device="cuda").half()
    args = (table, i32([length - n] * B), n, H, 0.125)
    kw = dict(first=i32(range(0, B * n, n)), count=i32([n] * B))
    good = P.attn(pool.p, q, *args, **kw)
    check_attn(good, q, seqs, [length - n] * B, [n] * B, list(range(0, B * n, n)), 0.125, 0, "f16", H, hd)
    q[1, hd + 3] = float("nan")
    q[2, 3 * hd] = float("inf")
    bad = P.attn(pool.p, q, *args, **kw)
    L.check_status()
    assert torch.isnan(bad[1, hd:2 * hd]).all() and torch.isnan(bad[2, 3 * hd:]).all()
    bad[1, hd:2 * hd] = good[1, hd:2 * hd]
    bad[2, 3 * hd:] = good[2, 3 * hd:]
    assert torch.equal(bad, good)


@pytest.mark.parametrize("B,n,window", [(1, 1, 0), (3, 1, 0), (60, 1, 0), (3, 4, 0), (3, 4, 1100), (2, 30, 0)])
def test_a_captured_step_follows_the_lengths(B, n, window):
    """One capture; between replays the sequences grow by very different amounts, past 16 pages: which warp and block has which page is found anew every time."""
    P, L = ops()
    KV, hd, H = 2, 64, 6
    r = np.random.default_rng(B)
    seqs = [Seq(KV, hd) for _ in range(B)]
    pool = Pool(P, WIDE * B, KV, hd)
    table = pool.table([WIDE * PAGE] * B)
    qkv = torch.empty(B * n, (H + 2 * KV) * hd, dtype=torch.float16, device="cuda")
    q, o = (torch.empty(B * n, H * hd, dtype=torch.float16, device="cuda") for _ in range(2))
    scratch = torch.empty(max(4, P.attn_scratch(B, WIDE, KV, hd, n, H, window)), device="cuda")
    cs = cos_sin(WIDE * PAGE, hd)
    start, first, count = i32([0] * B), i32(range(0, B * n, n)), i32([n] * B)

    def step():
        P.append(pool.p, qkv, table, start, n, cs, H, first=first, count=count, q_out=q, rope_type=1)
        P.attn(pool.p, q, table, start, n, H, 0.125, window=window, first=first, count=count, out=o, scratch=scratch)

    qkv.zero_()
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for grow in (0, 70, 900, 1100):
        for b, s in enumerate(seqs):
            m = int(r.integers(0, grow + 1)) if B > 1 else grow
            if m:
                s.append(*(r.standard_normal((m, KV, hd)).astype(np.float32) for _ in range(2)))
                pool.fill(table, b, s)
        at = [s.n for s in seqs]
        start.copy_(i32(at))
        qkv.copy_(torch.randn(B * n, (H + 2 * KV) * hd, device="cuda"))
        graph.replay()
        L.check_status()
        x = qkv.float().cpu().numpy().reshape(B, n, -1, hd)
        for b, s in enumerate(seqs):
            s.append(rotate(x[b, :, H:H + KV], at[b] + np.arange(n), cs.cpu().numpy(), 1), x[b, :, H + KV:])
        check_attn(o, q, seqs, at, [n] * B, list(range(0, B * n, n)), 0.125, window, "f16", H, hd)


# ---------------------------------------------------------------------------------------------- the engine
DENSE = dict(use_moe=False)


@pytest.mark.parametrize("over,kw", [(dict(sliding_window=9), {}), (dict(sliding_window=9), dict(max_len=2100)), (dict(sliding_window=9, use_qk_norm=False), dict(fused_step=False)),
                                     (dict(rope_type=1), dict(gemm_min_batch=2)), (dict(sliding_window=5), dict(gemm_min_batch=2, max_len=2100))])
def test_every_token_of_both_sequences_follows_the_fp32_model(over, kw, monkeypatch):
    """Without a router no choice is near another, so that all 24 tokens of both are compared; a window of 9 hides most of them."""
    E.test_logits_follow_the_fp32_model({**DENSE, **over}, kw, monkeypatch)


@pytest.mark.parametrize("over,kw", [(dict(sliding_window=100), {}), (dict(sliding_window=100), dict(max_len=2100)), ({}, dict(max_len=2100)),
                                     (dict(sliding_window=40, use_moe=False), dict(gemm_min_batch=2, max_len=2100))])
def test_portions_equal_single_steps(over, kw):
    """300 tokens of two sequences in portions of 128 against 300 steps (the tolerance of the same comparison without a window)."""
    cfg = E.cfg_of(**over)
    prompt = E.ids_of(2, 300, 4)
    a, _ = E.engine(cfg, batch=2, **kw)
    a.reset(1)
    a.prefill(prompt)
    b, _ = E.engine(cfg, batch=2, **kw)
    b.reset(1)
    for j in range(300):
        b.cur_tok.copy_(prompt[:, j])
        b._forward_token()
    a.check()
    assert torch.allclose(a.logits, b.logits, rtol=5e-2, atol=5e-2), float((a.logits - b.logits).abs().max())


def test_a_prompt_behind_one_that_was_not_a_number():
    """Rows past a portion's tokens keep an earlier prompt's attention; whatever that was, no other row has part in it."""
    for over in ({}, DENSE):
        cfg = E.cfg_of(**over)
        eng, _ = E.engine(cfg, batch=2)
        want, _ = E.engine(cfg, batch=2)
        prompt = E.ids_of(2, 90, 6)
        for e in (eng, want):
            e.reset(1)
            e.prefill(E.ids_of(2, 200, 5))
        eng._prefill_model.layers[0].att.fill_(math.nan)
        for e in (eng, want):
            e.reset(1)
            e.prefill(prompt)
        assert torch.isfinite(eng.logits).all() and torch.equal(eng.logits, want.logits)
        eng.check()
