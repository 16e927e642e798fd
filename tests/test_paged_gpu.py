"""Paged 8-bit key/value cache on the device: appending, attention and reading back against plain arithmetic."""
import math

import numpy as np
import pytest
import torch

from paged_oracle import PAGE, Pool, Seq, attention, rotate, scale_of

pytestmark = pytest.mark.gpu

DT = {"f16": torch.float16, "bf16": torch.bfloat16}
HALF = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}         # half a step, relative
TINY = {"f16": 2.0 ** -25, "bf16": 2.0 ** -134}       # half a step of the smallest numbers


def ops():
    from ghassan_b200.ops import _lib, paged
    return paged, _lib


def i32(x):
    return torch.tensor(list(x), dtype=torch.int32, device="cuda")


def cos_sin(positions, hd):
    from ghassan_b200.ops import kernels as K
    return K.rope_table(1e4 ** (-torch.arange(0, hd, 2, dtype=torch.float64) / hd), positions, "cuda")


def seqs_of(lens, KV, hd, seed, size=1.0):
    r = np.random.default_rng(seed)
    out = []
    for n in lens:
        s = Seq(KV, hd)
        if n:
            s.append((r.standard_normal((n, KV, hd)) * size * np.exp(0.5 * r.standard_normal((1, KV, hd)))).astype(np.float32),
                     (r.standard_normal((n, KV, hd)) * size).astype(np.float32))
        out.append(s)
    return out


def check_attn(got, q, seqs, start, count, first, scale, window, dt, H, hd):
    """Numerators are sums of 16-bit weights (half a step of float16 each, 2^-11) times exact codes; the rest is fp32, for which 2^-15 is ample; then one
    rounding to the output's type."""
    got = got.double().cpu().numpy()
    for b, s in enumerate(seqs):
        if not count[b]:
            continue
        rows = slice(first[b], first[b] + count[b])
        k, v = s.held()
        want, mag = attention(q[rows].double().cpu().numpy().reshape(count[b], H, hd), k, v, start[b], scale, window)
        allow = (2.0 ** -11 + 2.0 ** -15) * mag
        allow = allow + HALF[dt] * (np.abs(want) + allow) + TINY[dt]
        mine = got[rows].reshape(want.shape)
        assert np.array_equal(np.isnan(mine), np.isnan(want)), f"sequence {b}"          # of a query that is not finite
        err = np.where(np.isnan(want), 0, np.abs(mine - want))
        assert (err <= np.where(np.isnan(want), 1, allow)).all(), f"sequence {b}: {float((err / allow).max()):.2f} of the allowance"


# ---------------------------------------------------------------------------------------------- appending
@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("hd,H,KV", [(32, 4, 2), (64, 12, 4), (128, 6, 1), (64, 3, 3)])
@pytest.mark.parametrize("rope_type", [0, 1])
def test_append_gives_the_codes_of_the_definition(hd, H, KV, dt, rope_type):
    P, L = ops()
    start, count = [0, 5, 63, 64, 130, 7, 0], [1, 1, 2, 200, 61, 0, 64]
    first = [3, 0, 1, 10, 220, 9, 300]                      # rows in another order, gaps between
    rows = 370
    seqs = seqs_of(start, KV, hd, 1)
    pool = Pool(P, 24, KV, hd, seed=2)
    table = pool.table([s + n for s, n in zip(start, count)])
    for b, s in enumerate(seqs):
        pool.fill(table, b, s)
    before = [x.clone() for x in pool.p]
    wide = torch.randn(rows, (H + 2 * KV) * hd + 24, device="cuda", generator=torch.Generator("cuda").manual_seed(5)).to(DT[dt])
    qkv = wide[:, 8:8 + (H + 2 * KV) * hd]
    cs = cos_sin(400, hd)
    q_out = torch.full((rows, H * hd + 8), 7.0, dtype=DT[dt], device="cuda")
    P.append(pool.p, qkv, table, i32(start), 200, cs, H, first=i32(first), count=i32(count), q_out=q_out[:, :H * hd], rope_type=rope_type)
    L.check_status()
    x = qkv.float().cpu().numpy().reshape(rows, H + 2 * KV, hd)
    c = cs.cpu().numpy()
    seen = np.zeros(rows, bool)
    mine = set()
    for b, s in enumerate(seqs):
        r = slice(first[b], first[b] + count[b])
        seen[r] = True
        y = rotate(x[r, :H + KV], start[b] + np.arange(count[b]), c, rope_type)
        if count[b]:
            want = torch.from_numpy(y[:, :H].reshape(count[b], -1)).to(DT[dt])
            assert torch.equal(q_out[r, :H * hd].cpu(), want), f"queries of sequence {b}"
            s.append(y[:, H:], x[r, H + KV:])
        n = start[b] + count[b]
        kc, vc, ks, vs = pool.codes(table, b, n)
        pages = (n + PAGE - 1) // PAGE
        assert np.array_equal(ks, s.scales[0, :pages]) and np.array_equal(vs, s.scales[1, :pages]), f"scales of sequence {b}"
        want = s.codes.transpose(0, 1, 3, 2, 4).reshape(2, -1, KV, hd)[:, :n]
        assert np.array_equal(kc, want[0]) and np.array_equal(vc, want[1]), f"codes of sequence {b}"
        mine |= {int(i) for i in table[b, :pages]}
        if n % PAGE:                                        # places past the end are as they were
            i, m = int(table[b, pages - 1]), n % PAGE
            assert torch.equal(pool.p.k[i, :, m:], before[0][i, :, m:]) and torch.equal(pool.p.v[i, :, :, m:], before[2][i, :, :, m:])
    others = [i for i in range(24) if i not in mine]
    assert all(torch.equal(a[others].nan_to_num(9.0), b[others].nan_to_num(9.0)) for a, b in zip(pool.p, before))
    left = torch.from_numpy(~seen).cuda()
    assert (q_out[left] == 7.0).all() and (q_out[:, H * hd:] == 7.0).all()


def test_a_growing_page_is_rescaled_token_by_token():
    P, L = ops()
    KV, hd, H = 2, 64, 4
    r = np.random.default_rng(3)
    pool = Pool(P, 4, KV, hd)
    table = pool.table([70])
    s = Seq(KV, hd)
    cs = torch.cat([torch.ones(70, 32), torch.zeros(70, 32)], 1).cuda()       # no turn: magnitudes stay what they are
    for i in range(70):
        x = (r.standard_normal((1, (H + 2 * KV) * hd)) * 1.35 ** (i % 40)).astype(np.float16)
        if i == 20:
            x[:] = 0
        P.append(pool.p, torch.from_numpy(x).cuda(), table, i32([i]), 1, cs, H)
        y = x.astype(np.float32).reshape(1, -1, hd)
        s.append(rotate(y[:, H:H + KV], np.array([i]), cs.cpu().numpy(), 0), y[:, H + KV:])
    with pytest.raises(RuntimeError, match="303"):            # 1.35^39 times a large draw is past float16: infinite, held as zero
        L.check_status()
    kc, vc, ks, vs = pool.codes(table, 0, 70)
    assert np.array_equal(ks, s.scales[0]) and np.array_equal(vs, s.scales[1])
    want = s.codes.transpose(0, 1, 3, 2, 4).reshape(2, -1, KV, hd)[:, :70]
    assert np.array_equal(kc, want[0]) and np.array_equal(vc, want[1])


@pytest.mark.parametrize("value", [0.0, 6e-8, 127.0, 127.5, 65504.0, 63.5, 2.0 ** -14])
def test_scales_at_the_edges(value):
    P, L = ops()
    pool = Pool(P, 2, 1, 32)
    table = pool.table([1])
    x = torch.full((1, 96), value, dtype=torch.float16, device="cuda")
    cs = torch.cat([torch.ones(1, 16), torch.zeros(1, 16)], 1).cuda()
    P.append(pool.p, x, table, i32([0]), 1, cs, 1)
    L.check_status()
    want = scale_of(np.float32(np.float16(value)))
    kc, vc, ks, vs = pool.codes(table, 0, 1)
    assert ks[0, 0] == want and vs[0, 0] == want
    assert (kc == np.rint(np.float32(np.float16(value)) / want)).all() and (vc == kc).all()
    k, v = P.read(pool.p, table, i32([0]), 1, torch.float16, 1)
    assert torch.isfinite(k).all() and torch.equal(k, v)
    assert abs(float(k[0, 0, 0]) - float(np.float16(value))) <= float(want) / 2


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("rope_type", [0, 1])
def test_head_norms(dt, rope_type):
    """The norm's sum may be taken in any order: values are within one step of the page's scale and, for queries, of the type's rounding."""
    P, L = ops()
    KV, hd, H, n = 2, 64, 6, 90
    r = np.random.default_rng(8)
    pool = Pool(P, 4, KV, hd)
    table = pool.table([n])
    x = torch.from_numpy(r.standard_normal((n, (H + 2 * KV) * hd)).astype(np.float32)).to(DT[dt]).cuda()
    qw, kw = (torch.from_numpy((1 + 0.3 * r.standard_normal(hd)).astype(np.float32)).cuda() for _ in range(2))
    cs = cos_sin(n, hd)
    q = P.append(pool.p, x, table, i32([0]), n, cs, H, first=i32([0]), count=i32([n]), qw=qw, kw=kw, eps=1e-5, rope_type=rope_type)
    L.check_status()
    y = x.double().cpu().numpy().reshape(n, -1, hd)
    y = y / np.sqrt((y ** 2).mean(-1, keepdims=True) + 1e-5)
    y[:, :H] *= qw.double().cpu().numpy()
    y[:, H:H + KV] *= kw.double().cpu().numpy()
    c = cs.double().cpu().numpy()
    half, pos = hd // 2, np.arange(n)
    co, si = c[pos][:, None, :half], c[pos][:, None, half:]
    a, b = (y[..., :half], y[..., half:]) if rope_type else (y[..., 0::2], y[..., 1::2])
    t = np.empty_like(y)
    if rope_type:
        t[..., :half], t[..., half:] = a * co - b * si, a * si + b * co
    else:
        t[..., 0::2], t[..., 1::2] = a * co - b * si, a * si + b * co
    err = np.abs(q.double().cpu().numpy().reshape(n, H, hd) - t[:, :H])
    assert (err <= HALF[dt] * np.abs(t[:, :H]) + 2.0 ** -19 * np.abs(t).max()).all()
    k, _ = P.read(pool.p, table, i32([0]), n, torch.bfloat16, n, first=i32([0]), count=i32([n]))
    step = pool.codes(table, 0, n)[2][np.arange(n) // PAGE][:, :, None]
    assert (np.abs(k.double().cpu().numpy() - t[:, H:H + KV]) <= 0.51 * step).all()


def test_numbers_that_are_not_finite_are_held_as_zero_and_told():
    P, L = ops()
    KV, hd, H = 1, 64, 2
    pool = Pool(P, 2, KV, hd)
    table = pool.table([3])
    x = torch.ones(3, 4 * hd, dtype=torch.float16, device="cuda")
    x[1, 2 * hd + 5] = float("nan")            # a key
    x[2, 3 * hd + 7] = float("inf")            # a value
    cs = torch.cat([torch.ones(3, 32), torch.zeros(3, 32)], 1).cuda()
    P.append(pool.p, x, table, i32([0]), 3, cs, H, first=i32([0]), count=i32([3]))
    with pytest.raises(RuntimeError, match="303"):
        L.check_status()
    k, v = P.read(pool.p, table, i32([0]), 3, torch.float16, 3, first=i32([0]), count=i32([3]))
    k, v = k[:, 0].cpu(), v[:, 0].cpu()
    assert v[2, 7] == 0 and v.sum() == 3 * hd - 1
    assert k[1, 5] == 0 and torch.isfinite(k).all() and k.sum() >= 3 * hd - 2     # rope_type 0 mixes dimensions 4 and 5: 0 * nan


# ---------------------------------------------------------------------------------------------- reading
@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("hd,KV", [(32, 3), (64, 4), (128, 2)])
def test_read_gives_what_codes_stand_for(hd, KV, dt):
    P, L = ops()
    lens = [200, 1, 64, 129]
    start, count, first = [3, 0, 63, 70], [197, 1, 1, 0], [2, 0, 250, 1]
    seqs = seqs_of(lens, KV, hd, 4)
    pool = Pool(P, 12, KV, hd)
    table = pool.table(lens)
    for b, s in enumerate(seqs):
        pool.fill(table, b, s)
    k = torch.full((256, KV * hd + 8), 5.0, dtype=DT[dt], device="cuda")
    v = torch.full((256, KV * hd + 16), 5.0, dtype=DT[dt], device="cuda")
    P.read(pool.p, table, i32(start), 197, DT[dt], 256, first=i32(first), count=i32(count), k_out=k[:, :KV * hd], v_out=v[:, :KV * hd])
    L.check_status()
    left = torch.ones(256, dtype=torch.bool)
    for b, s in enumerate(seqs):
        for got, want in zip((k, v), s.held()):
            want = torch.from_numpy(want[start[b]:start[b] + count[b]].reshape(count[b], KV * hd))
            assert torch.equal(got[first[b]:first[b] + count[b], :KV * hd].cpu(), want.to(DT[dt]))
        left[first[b]:first[b] + count[b]] = False
    assert (k[left.cuda()] == 5).all() and (v[left.cuda()] == 5).all() and (k[:, KV * hd:] == 5).all()


# ---------------------------------------------------------------------------------------------- attention
def run_attn(P, L, hd, H, KV, dt, start, count, window, seed=1, scale=None, size=1.0, q_size=1.0, gaps=True):
    lens = [s + n for s, n in zip(start, count)]
    seqs = seqs_of(lens, KV, hd, seed, size)
    pool = Pool(P, sum((n + PAGE - 1) // PAGE for n in lens) + 5, KV, hd, seed=seed)
    table = pool.table(lens)
    for b, s in enumerate(seqs):
        pool.fill(table, b, s)
    first = list(np.cumsum([0] + [n + (2 if gaps else 0) for n in count])[:-1])
    first = [int(f) for f in first]
    rows = first[-1] + count[-1] + 3
    wide = (torch.randn(rows, H * hd + 16, device="cuda", generator=torch.Generator("cuda").manual_seed(seed)) * q_size).to(DT[dt])
    q = wide[:, 8:8 + H * hd]
    out = torch.full((rows, H * hd + 8), 3.0, dtype=DT[dt], device="cuda")
    scale = scale or 1.0 / math.sqrt(hd)
    P.attn(pool.p, q, table, i32(start), max(count), H, scale, window=window, first=i32(first), count=i32(count), out=out[:, :H * hd])
    L.check_status()
    check_attn(out[:, :H * hd], q, seqs, start, count, first, scale, window, dt, H, hd)
    left = torch.ones(rows, dtype=torch.bool)
    for f, n in zip(first, count):
        left[f:f + n] = False
    assert (out[left.cuda()] == 3).all() and (out[:, H * hd:] == 3).all()


HEADS = [(32, 4, 2), (64, 12, 4), (64, 8, 1), (128, 8, 2), (128, 5, 5), (64, 7, 1), (32, 16, 1), (128, 48, 2)]


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("hd,H,KV", HEADS)
def test_single_tokens(hd, H, KV, dt):
    P, L = ops()
    run_attn(P, L, hd, H, KV, dt, [0, 1, 62, 63, 64, 65, 127, 500, 1300], [1] * 9, 0)


@pytest.mark.parametrize("window", [1, 5, 64, 65, 200])
@pytest.mark.parametrize("hd,H,KV", HEADS[:4])
def test_single_tokens_with_a_window(hd, H, KV, window):
    P, L = ops()
    run_attn(P, L, hd, H, KV, "bf16", [0, 3, 63, 64, 128, 300, 1100], [1] * 7, window)


@pytest.mark.parametrize("n", [1, 2, 5, 6, 11, 16, 17, 40])
@pytest.mark.parametrize("window", [0, 3, 70])
def test_a_few_tokens_a_sequence(n, window):
    P, L = ops()
    run_attn(P, L, 64, 6, 2, "f16", [0, 60, 63, 64, 600, 7], [n, n, max(1, n - 1), 0, n, 1], window)


@pytest.mark.parametrize("dt", ["f16", "bf16"])
@pytest.mark.parametrize("hd,H,KV", HEADS)
@pytest.mark.parametrize("window", [0, 100])
def test_prompts(hd, H, KV, dt, window):
    P, L = ops()
    run_attn(P, L, hd, H, KV, dt, [0, 100, 1, 191, 640], [129, 64, 0, 257, 1], window)


@pytest.mark.parametrize("hd", [32, 64, 128])
def test_items_of_half_and_whole_tiles_take_turns(hd):
    """Rows of a key head that end in the first or the second 128 of 256, over many key tiles: what one half of a block leaves out the other half's warps must not run ahead of."""
    P, L = ops()
    run_attn(P, L, hd, 6, 2, "f16", [3000, 2000, 700], [90, 171, 43], 0)
    run_attn(P, L, hd, 6, 2, "bf16", [1900, 5, 4000], [30, 300, 86], 1500)
    run_attn(P, L, hd, 8, 8, "f16", [1000, 1200], [257, 385], 0)


def test_long_sequences_are_split_and_joined():
    P, L = ops()
    run_attn(P, L, 64, 4, 2, "f16", [20001, 3, 9000], [1, 1, 1], 0)
    run_attn(P, L, 128, 4, 1, "bf16", [9001], [3], 0)
    run_attn(P, L, 64, 4, 1, "bf16", [9001, 0], [40, 9], 8000)


@pytest.mark.parametrize("B", [1, 33, 300])
def test_batches(B):
    P, L = ops()
    r = np.random.default_rng(B)
    run_attn(P, L, 64, 4, 2, "f16", [int(x) for x in r.integers(0, 260, B)], [1] * B, 0, gaps=False)


@pytest.mark.parametrize("hd,n", [(32, 1), (128, 2), (32, 20)])
def test_more_sequences_than_one_launch_takes(hd, n):
    P, L = ops()
    r = np.random.default_rng(n)
    run_attn(P, L, hd, 8, 1, "f16", [int(x) for x in r.integers(0, 130, 1100)], [int(x) for x in r.integers(1, n + 1, 1100)], 0, gaps=False)


def test_rows_without_first_and_count_are_one_a_sequence():
    P, L = ops()
    B, KV, hd, H = 1100, 1, 32, 2
    seqs = seqs_of([1 + b % 70 for b in range(B)], KV, hd, 1)
    pool = Pool(P, 2 * B, KV, hd)
    table = pool.table([s.n for s in seqs])
    for b, s in enumerate(seqs):
        pool.fill(table, b, s)
    start = [s.n - 1 for s in seqs]
    q = torch.randn(B, H * hd, device="cuda").half()
    out = P.attn(pool.p, q, table, i32(start), 1, H, 0.2)
    k, v = P.read(pool.p, table, i32(start), 1, torch.float16, B)
    L.check_status()
    check_attn(out, q, seqs, start, [1] * B, list(range(B)), 0.2, 0, "f16", H, hd)
    assert np.array_equal(v.double().cpu().numpy(), np.stack([s.held()[1][-1] for s in seqs]).astype(np.float16).astype(np.float64))


@pytest.mark.parametrize("n,window", [(1, 100), (2, 64), (30, 70), (300, 129), (300, 1)])
def test_pages_behind_the_window_may_be_gone(n, window):
    """A text's pages that no query sees any more need not be in its table."""
    P, L = ops()
    KV, hd, H, start = 2, 64, 6, 900
    seqs = seqs_of([start + n], KV, hd, 1)
    pool = Pool(P, 30, KV, hd)
    table = pool.table([start + n])
    pool.fill(table, 0, seqs[0])
    table[0, :(start - window + 1) // PAGE] = -1
    q = torch.randn(n, H * hd, device="cuda").half()
    out = P.attn(pool.p, q, table, i32([start]), n, H, 0.125, window=window, first=i32([0]), count=i32([n]))
    L.check_status()
    check_attn(out, q, seqs, [start], [n], [0], 0.125, window, "f16", H, hd)


@pytest.mark.parametrize("n", [1, 30])
def test_weights_far_apart_and_tiny_or_large_values(n):
    """One key that takes nearly all weight, and none; values of very small and large pages; queries at the ends of the type's range."""
    P, L = ops()
    run_attn(P, L, 64, 4, 2, "f16", [300], [n], 0, scale=4.0)
    run_attn(P, L, 64, 4, 2, "bf16", [300], [n], 0, scale=1e-6)
    run_attn(P, L, 64, 4, 2, "bf16", [300], [n], 0, size=1e-20, q_size=1e20)
    run_attn(P, L, 64, 4, 2, "bf16", [300], [n], 0, size=1e15, q_size=1e-15)
    run_attn(P, L, 64, 4, 2, "f16", [300], [n], 0, size=1e-5, q_size=2e4)
    run_attn(P, L, 64, 4, 2, "f16", [300], [n], 0, size=3e3, q_size=1e-6)


@pytest.mark.parametrize("n", [1, 30])
def test_pages_of_very_different_scales(n):
    P, L = ops()
    KV, hd, H, dt = 1, 64, 4, "bf16"
    r = np.random.default_rng(1)
    s = Seq(KV, hd)
    for e in (0, -18, 3, -5, 9, -30, 2):
        s.append((r.standard_normal((64, KV, hd))).astype(np.float32), (r.standard_normal((64, KV, hd)) * 2.0 ** e).astype(np.float32))
    pool = Pool(P, 9, KV, hd)
    table = pool.table([s.n])
    pool.fill(table, 0, s)
    q = torch.randn(n, H * hd, device="cuda").to(DT[dt])
    out = P.attn(pool.p, q, table, i32([s.n - n]), n, H, 0.2, first=i32([0]), count=i32([n]))
    L.check_status()
    check_attn(out, q, [s], [s.n - n], [n], [0], 0.2, 0, dt, H, hd)


@pytest.mark.parametrize("n", [3, 40])
def test_a_query_that_is_not_a_number_spoils_its_own_rows_only(n):
    P, L = ops()
    KV, hd, H = 2, 64, 4
    seqs = seqs_of([200], KV, hd, 1)
    pool = Pool(P, 6, KV, hd)
    table = pool.table([200])
    pool.fill(table, 0, seqs[0])
    q = torch.randn(n, H * hd, device="cuda").half()
    args = (table, i32([200 - n]), n, H, 0.125)
    good = P.attn(pool.p, q, *args, first=i32([0]), count=i32([n]))
    q[1, hd + 3] = float("nan")                              # head 1 of token 1
    q[2, 3 * hd] = float("inf")
    bad = P.attn(pool.p, q, *args, first=i32([0]), count=i32([n]))
    L.check_status()
    assert torch.isnan(bad[1, hd:2 * hd]).all() and torch.isnan(bad[2, 3 * hd:]).all()
    bad[1, hd:2 * hd] = good[1, hd:2 * hd]
    bad[2, 3 * hd:] = good[2, 3 * hd:]
    assert torch.equal(bad, good)


@pytest.mark.parametrize("n", [1, 20])
def test_far_places_of_a_large_pool(n):
    """Codes past the first 4 GiB of a pool, rows past 2^31 bytes of a tensor."""
    P, L = ops()
    KV, hd, H = 8, 128, 8
    pages = (2 ** 32) // (KV * PAGE * hd) + 7
    big = P.Pages(torch.empty(pages, KV, PAGE, hd, dtype=torch.int8, device="cuda"), torch.full((pages, KV), math.nan, device="cuda"),
                  torch.empty(pages, KV, hd, PAGE, dtype=torch.int8, device="cuda"), torch.full((pages, KV), math.nan, device="cuda"))
    ids = [pages - 1, 2, pages - 3]
    table = i32(ids).view(1, 3)
    seq = Seq(KV, hd)
    cs = cos_sin(200, hd)
    rows = 2 ** 31 // (3 * H * hd * 2) + 200
    qkv = torch.empty(rows, 3 * H * hd, dtype=torch.float16, device="cuda")
    at = rows - 181
    qkv[at:at + 180] = torch.randn(180, 3 * H * hd, device="cuda").half()
    q = P.append(big, qkv, table, i32([0]), 180, cs, H, first=i32([at]), count=i32([180]), rope_type=1)
    L.check_status()
    x = qkv[at:at + 180].float().cpu().numpy().reshape(180, 3 * H, hd)
    seq.append(rotate(x[:, H:2 * H], np.arange(180), cs.cpu().numpy(), 1), x[:, 2 * H:])
    assert np.array_equal(big.k[ids[2], :, :52].cpu().numpy(), seq.codes[0, 2, :, :52])
    first, start = at + 180 - n, 180 - n
    out = P.attn(big, q, table, i32([start]), n, H, 0.1, first=i32([first]), count=i32([n]))
    k, v = P.read(big, table, i32([start]), n, torch.float16, n, first=i32([0]), count=i32([n]))
    L.check_status()
    check_attn(out[first:first + n], q[first:first + n], [seq], [start], [n], [0], 0.1, 0, "f16", H, hd)
    assert np.array_equal(v.double().cpu().numpy(), seq.held()[1][start:])


# ---------------------------------------------------------------------------------------------- together, graphs, streams
def follow(P, L, steps, H, KV, hd, dt, window=0, graph=False, seed=0):
    """Three sequences through ``steps`` of (tokens each): append, attend; every step against the oracle."""
    B = 3
    total = [sum(c[b] for c in steps) for b in range(B)]
    pool = Pool(P, sum((n + PAGE - 1) // PAGE for n in total) + 1, KV, hd, seed=seed)
    table = pool.table(total)
    seqs = [Seq(KV, hd) for _ in range(B)]
    cs = cos_sin(max(total) + 1, hd)
    c = cs.cpu().numpy()
    g = torch.Generator("cuda").manual_seed(seed)
    for count in steps:
        start = [s.n for s in seqs]
        first = [int(f) for f in np.cumsum([0] + list(count))[:-1]]
        qkv = torch.randn(sum(count), (H + 2 * KV) * hd, device="cuda", generator=g).to(DT[dt])
        kw = dict(first=i32(first), count=i32(count))
        q = P.append(pool.p, qkv, table, i32(start), max(count), cs, H, rope_type=1, **kw)
        o = P.attn(pool.p, q, table, i32(start), max(count), H, hd ** -0.5, window=window, **kw)
        L.check_status()
        x = qkv.float().cpu().numpy().reshape(sum(count), -1, hd)
        for b, s in enumerate(seqs):
            r = slice(first[b], first[b] + count[b])
            if count[b]:
                y = rotate(x[r, H:H + KV], start[b] + np.arange(count[b]), c, 1)
                s.append(y, x[r, H + KV:])
        check_attn(o, q, seqs, start, count, first, hd ** -0.5, window, dt, H, hd)


@pytest.mark.parametrize("dt", ["f16", "bf16"])
def test_prompts_in_portions_then_tokens(dt):
    P, L = ops()
    follow(P, L, [(100, 30, 0), (70, 1, 129), (3, 5, 2)] + [(1, 1, 1)] * 6, 6, 2, 64, dt)
    follow(P, L, [(64, 128, 1), (200, 0, 63)] + [(1, 1, 1)] * 3, 4, 4, 128, dt, window=90)


@pytest.mark.parametrize("B,n", [(2, 1), (40, 1), (2, 50)])
def test_a_captured_step_replays_at_other_lengths(B, n):
    """One capture of append and attention; the sequences grow between replays, as an engine's do."""
    P, L = ops()
    KV, hd, H = 2, 64, 6
    pool = Pool(P, 10 * B, KV, hd)
    table = pool.table([600] * B)
    seqs = seqs_of([0] * B, KV, hd, 0)
    cs = cos_sin(640, hd)
    qkv = torch.randn(B * n, (H + 2 * KV) * hd, device="cuda").half()
    q, o = torch.empty(B * n, H * hd, dtype=torch.float16, device="cuda"), torch.empty(B * n, H * hd, dtype=torch.float16, device="cuda")
    start, first, count = i32([0] * B), i32(range(0, B * n, n)), i32([n] * B)

    def step():
        P.append(pool.p, qkv, table, start, n, cs, H, first=first, count=count, q_out=q, rope_type=1)
        P.attn(pool.p, q, table, start, n, H, 0.125, first=first, count=count, out=o)

    step()                                                    # set-up outside the capture; the replay writes the same again
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    at = 0
    for more in (0, 0, 0):
        qkv.copy_(torch.randn(B * n, (H + 2 * KV) * hd, device="cuda"))
        start.fill_(at)
        graph.replay()
        L.check_status()
        x = qkv.float().cpu().numpy().reshape(B, n, -1, hd)
        for b, s in enumerate(seqs):
            s.append(rotate(x[b, :, H:H + KV], at + np.arange(n), cs.cpu().numpy(), 1), x[b, :, H + KV:])
        check_attn(o, q, seqs, [at] * B, [n] * B, list(range(0, B * n, n)), 0.125, 0, "f16", H, hd)
        at += n


@pytest.mark.parametrize("n", [1, 50])
def test_two_streams_at_once(n):
    """Calls on two streams with tensors of their own do not meet (each call has its own workspace)."""
    P, L = ops()
    KV, hd, H = 4, 64, 8
    streams, out = [torch.cuda.Stream() for _ in range(2)], [None, None]
    made = []
    for i in range(2):
        lens = [3000, 900]
        seqs = seqs_of(lens, KV, hd, i)
        pool = Pool(P, 70, KV, hd, seed=i)
        table = pool.table(lens)
        for b, s in enumerate(seqs):
            pool.fill(table, b, s)
        q = torch.randn(2 * n, H * hd, device="cuda", generator=torch.Generator("cuda").manual_seed(i)).half()
        start = [m - n for m in lens]
        made.append((seqs, pool, table, q, start, i32(start), i32([0, n]), i32([n, n])))
    torch.cuda.synchronize()
    for _ in range(10):
        for i, st in enumerate(streams):
            seqs, pool, table, q, start, s_dev, f_dev, c_dev = made[i]
            with torch.cuda.stream(st):
                out[i] = P.attn(pool.p, q, table, s_dev, n, H, 0.125, first=f_dev, count=c_dev)
    torch.cuda.synchronize()
    L.check_status()
    for i in range(2):
        seqs, pool, table, q, start = made[i][:5]
        check_attn(out[i], q, seqs, start, [n, n], [0, n], 0.125, 0, "f16", H, hd)


def test_results_are_the_same_every_time():
    P, L = ops()
    KV, hd, H = 4, 64, 12
    seqs = seqs_of([5000, 70, 900], KV, hd, 2)
    pool = Pool(P, 120, KV, hd)
    table = pool.table([5000, 70, 900])
    for b, s in enumerate(seqs):
        pool.fill(table, b, s)
    for n in (1, 60):
        q = torch.randn(3 * n, H * hd, device="cuda").half()
        kw = dict(first=i32([0, n, 2 * n]), count=i32([n] * 3))
        start = i32([5000 - n, 70 - n, 900 - n])
        a = P.attn(pool.p, q, table, start, n, H, 0.125, **kw)
        for _ in range(5):
            assert torch.equal(a, P.attn(pool.p, q, table, start, n, H, 0.125, **kw))


# ---------------------------------------------------------------------------------------------- numbers that do not fit
@pytest.mark.parametrize("n", [1, 40])
def test_what_does_not_fit_is_left_out_and_told(n):
    """Sequence 1 of three has a start, a count, rows or a page that do not fit; the others' results are as without it."""
    P, L = ops()
    KV, hd, H = 2, 64, 4
    lens = [150, 100, 90]
    seqs = seqs_of(lens, KV, hd, 3)

    def tables():
        pool = Pool(P, 12, KV, hd, seed=7)
        table = pool.table(lens)
        for b, s in enumerate(seqs):
            pool.fill(table, b, s)
        return pool, table

    start, first, count = [m - n for m in lens], [0, n, 2 * n], [n] * 3
    q = torch.randn(3 * n, H * hd, device="cuda").half()
    qkv = torch.randn(3 * n, (H + 2 * KV) * hd, device="cuda").half()
    cs = cos_sin(192, hd)
    others = torch.tensor([i < n or i >= 2 * n for i in range(3 * n)], device="cuda")

    def run(start, first, count, spoil=None, max_new=n):
        pool, table = tables()
        if spoil is not None:
            table[1, (lens[1] - 1) // PAGE] = spoil
        kw = dict(first=i32(first), count=i32(count))
        o = P.attn(pool.p, q, table, i32(start), max_new, H, 0.125, out=torch.zeros_like(q), **kw)
        status = [int(L.status_word()[0])]
        L.status_word().zero_()
        k, v = P.read(pool.p, table, i32(start), max_new, torch.float16, 3 * n, **kw)
        status.append(int(L.status_word()[0]))
        L.status_word().zero_()
        was = [x.clone() for x in pool.p]
        q2 = P.append(pool.p, qkv, table, i32(start), max_new, cs, H, q_out=torch.zeros_like(q), **kw)
        status.append(int(L.status_word()[0]))
        L.status_word().zero_()
        keep = [i for b in (0, 2) for i in table[b].tolist() if i >= 0]
        loose = [i for i in range(12) if i not in keep and i not in table[1].tolist()]
        assert all(torch.equal(a[loose].nan_to_num(1.0), b[loose].nan_to_num(1.0)) for a, b in zip(pool.p, was))
        return status, [o[others], k[others], v[others], q2[others]] + [x[keep] for x in pool.p]

    ok, want = run(start, first, count)
    assert ok == [0, 0, 0]
    for bad in (dict(start=[start[0], 3 * PAGE - n + 1, start[2]]), dict(start=[start[0], -1, start[2]]), dict(first=[0, 2 * n + 1, 2 * n]),
                dict(first=[0, -1, 2 * n]), dict(count=[n, n + 1, n]), dict(count=[n, -1, n]), dict(spoil=-1), dict(spoil=12), dict(spoil=2 ** 31 - 1),
                dict(spoil=-2 ** 31)):
        if bad.get("first") == [0, 2 * n + 1, 2 * n] and n == 1:
            bad = dict(first=[0, 3 * n, 2 * n])
        status, got = run(**{**dict(start=start, first=first, count=count), **bad})
        assert status == [301] * 3, (bad, status)
        assert all(torch.equal(a, b) for a, b in zip(got, want)), bad


def test_nothing_to_do():
    P, L = ops()
    pool = Pool(P, 2, 2, 64)
    table = pool.table([0, 0], width=1)
    q = torch.randn(4, 256, device="cuda").half()
    out = torch.full_like(q, 2.0)
    zero = i32([0, 0])
    P.attn(pool.p, q, table, zero, 0, 4, 0.1, first=zero, count=zero, out=out)
    P.attn(pool.p, q, table, zero, 64, 4, 0.1, first=zero, count=zero, out=out)
    k, v = P.read(pool.p, table, zero, 0, torch.float16, 0, first=zero, count=zero)
    empty = torch.empty(0, 1, dtype=torch.int32, device="cuda")
    P.attn(pool.p, q, empty, i32([]), 1, 4, 0.1, out=out)
    L.check_status()
    assert (out == 2).all() and k.shape == (0, 2, 64)


@pytest.mark.parametrize("B,W", [(0, 0), (2, 0), (0, 3)])
def test_nothing_to_do_in_tables_of_no_pages(B, W):
    """The same answer from all three calls."""
    P, L = ops()
    pool = Pool(P, 2, 2, 64).p
    table = torch.empty(B, W, dtype=torch.int32, device="cuda")
    kw = dict(first=i32([0] * B), count=i32([0] * B))
    qkv, cs = torch.zeros(5, 8 * 64, dtype=torch.float16, device="cuda"), cos_sin(9, 64)
    out = [torch.full((5, n), 2.0, dtype=torch.float16, device="cuda") for n in (256, 256, 128, 128)]
    assert P.append(pool, qkv, table, i32([0] * B), 0, cs, 4, q_out=out[0], **kw) is out[0]
    assert P.attn(pool, out[0], table, i32([0] * B), 0, 4, 0.1, out=out[1], **kw) is out[1]
    k, v = P.read(pool, table, i32([0] * B), 0, torch.float16, 5, k_out=out[2], v_out=out[3], **kw)
    L.check_status()
    assert k.shape == v.shape == (5, 2, 64) and all((x == 2).all() for x in out)


# ---------------------------------------------------------------------------------------------- more than a grid has blocks along an axis
@pytest.mark.parametrize("ragged", [False, True])
def test_more_sequences_than_a_grid_has_rows(ragged):
    """65535 blocks go along a grid's second and third axis; all three calls take what is more in several launches."""
    P, L = ops()
    B, hd = 65535 + 70, 32
    g = torch.Generator("cuda").manual_seed(1)
    pool = P.new_pages(B, 1, hd, "cuda")
    table = torch.randperm(B, generator=g, device="cuda").to(torch.int32).view(B, 1)
    count = torch.ones(B, dtype=torch.int32, device="cuda")
    first = torch.arange(B, dtype=torch.int32, device="cuda")
    if ragged:
        count[5::3] = 0                                       # whose rows are nobody's
        first = first.flip(0).contiguous()
    kw = dict(first=first, count=count) if ragged else {}
    start = torch.zeros(B, dtype=torch.int32, device="cuda")
    qkv = torch.randn(B, 3 * hd, device="cuda", generator=g).half()
    cs = torch.cat([torch.ones(1, hd // 2), torch.zeros(1, hd // 2)], 1).cuda()
    out = [torch.full((B, hd), 9.0, dtype=torch.float16, device="cuda") for _ in range(4)]
    P.append(pool, qkv, table, start, 1, cs, 1, q_out=out[0], **kw)
    P.attn(pool, out[0], table, start, 1, 1, 0.2, out=out[1], **kw)
    P.read(pool, table, start, 1, torch.float16, B, k_out=out[2], v_out=out[3], **kw)
    L.check_status()
    there = torch.zeros(B, dtype=torch.bool, device="cuda")
    there[first[count > 0].long()] = True
    assert all((x[~there] == 9).all() for x in out)
    q, k, v = qkv.view(B, 3, hd).unbind(1)
    assert torch.equal(out[0][there], q[there])
    for got, want in ((out[2], k), (out[3], v)):              # half a step of a page that one token has, and float16's own
        amax = want.float().abs().amax(1, keepdim=True)
        assert ((got.float() - want.float()).abs() <= (1 / 127 + 2.0 ** -11) * amax)[there].all()
    assert torch.equal(out[1][there], out[3][there])          # the soft-max over one key


@pytest.mark.parametrize("n", [3, 100])
def test_a_bound_of_more_pages_than_a_grid_has_rows(n):
    """max_new may be far more than there is: as much as the table has places for."""
    P, L = ops()
    KV, hd, H, W = 2, 64, 4, 65535 + 40
    pool = Pool(P, 4, KV, hd)
    table = torch.full((1, W), -1, dtype=torch.int32, device="cuda")
    table[0, :2] = i32([2, 0])
    kw = dict(first=i32([0]), count=i32([n]))
    qkv = torch.randn(n, (H + 2 * KV) * hd, device="cuda").half()
    cs = cos_sin(n, hd)
    q = P.append(pool.p, qkv, table, i32([0]), W * PAGE, cs, H, rope_type=1, **kw)
    o = P.attn(pool.p, q, table, i32([0]), W * PAGE, H, 0.125, **kw)
    k, v = P.read(pool.p, table, i32([0]), W * PAGE, torch.float16, n, **kw)
    L.check_status()
    s = Seq(KV, hd)
    x = qkv.float().cpu().numpy().reshape(n, -1, hd)
    s.append(rotate(x[:, H:H + KV], np.arange(n), cs.cpu().numpy(), 1), x[:, H + KV:])
    check_attn(o, q, [s], [0], [n], [0], 0.125, 0, "f16", H, hd)
    assert np.array_equal(v.double().cpu().numpy(), s.held()[1])
