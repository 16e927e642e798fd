"""Attention over the paged cache where numbers are far apart: values of pages a row does not see or gives no weight, scores of any size."""
import numpy as np
import pytest
import torch

from paged_oracle import PAGE, Pool, Seq
from test_paged_gpu import DT, HALF, TINY, i32, ops

pytestmark = pytest.mark.gpu


def pages_of(k, v):
    """A sequence whose pages come one by one, so that each has the scale of its own numbers."""
    s = Seq(k.shape[1], k.shape[2])
    for at in range(0, k.shape[0], PAGE):
        s.append(k[at:at + PAGE].astype(np.float32), v[at:at + PAGE].astype(np.float32))
    return s


def plain(q, s, start, scale, window, gone=(), step=2.0 ** -31):
    """Results and what they may be off by ahead of the last rounding, in 64 bits.  A weight is rounded to float16 after it was multiplied by a power of two a row, under which
    the largest weight times value scale that the row sees is at least 2^6 in the prompt kernel (2^14 in the token kernel): half a step of 2^-11 of itself, or, below float16's
    normal numbers, 2^-25, which is 2^-31 (2^-39) of that largest product.  It goes with a code of at most 127.  Sums are fp32, for which 2^-15 is ample."""
    k, v = s.held()
    n, H, hd = q.shape
    G = H // k.shape[1]
    pos, key = start + np.arange(n)[:, None], np.arange(k.shape[0])[None]
    sees = (key <= pos) & ((key > pos - window) if window > 0 else True)
    for p in gone:
        sees[:, p * PAGE:(p + 1) * PAGE] = False
    out, allow = np.zeros_like(q), np.zeros_like(q)
    for h in range(H):
        z = np.where(sees, (q[:, h] @ k[:, h // G].T) * scale, -np.inf)
        p = np.exp(z - z.max(1, keepdims=True))
        p /= p.sum(1, keepdims=True)
        unit = (p * s.scales[1][:, h // G].astype(np.float64)[np.arange(k.shape[0]) // PAGE][None]).max(1, keepdims=True)
        out[:, h] = p @ v[:, h // G]
        allow[:, h] = (2.0 ** -11 + 2.0 ** -15) * (p @ np.abs(v[:, h // G])) + step * 127 * sees.sum(1, keepdims=True) * unit
    return out, allow


def check(s, q, start, scale, window, dt, missing=(), status=0, width=None):
    """q [n, H, hd] fp32 on the host: the last n tokens of the sequence.  Once alone, where the kernels give every page to another warp or block, and as 600 sequences with the same
    pages, where a warp or block goes through all pages of some and is cut off in others."""
    P, L = ops()
    n, H, hd = q.shape
    pool = Pool(P, s.codes.shape[1] + 3, s.KV, hd, seed=4)
    table = pool.table([s.n], width)
    pool.fill(table, 0, s)
    for p in missing:
        table[0, p] = -1
    step = 2.0 ** -39 if n * (H // s.KV) <= 16 else 2.0 ** -31
    qd = torch.from_numpy(q.reshape(n, H * hd).astype(np.float32)).to(DT[dt]).cuda()
    want, allow = plain(qd.double().cpu().numpy().reshape(n, H, hd), s, start, scale, window, missing, step)
    allow = allow + HALF[dt] * (np.abs(want) + allow) + TINY[dt]
    for B in (1, 600):
        out = P.attn(pool.p, qd.repeat(B, 1), table.repeat(B, 1), i32([start] * B), n, H, scale, window=window, first=i32(range(0, B * n, n)), count=i32([n] * B))
        got = int(L.status_word()[0])
        L.status_word().zero_()
        assert got == status
        err = np.abs(out.double().cpu().numpy().reshape(B, n, H, hd) - want)
        worst = np.unravel_index(np.nan_to_num(err / allow, nan=np.inf).argmax(), err.shape)
        assert (err <= allow).all(), f"{err[worst] / allow[worst[1:]]:.2f} of the allowance, {B} sequences, at {[int(x) for x in worst]}"


WIDTHS = [None, 40]            # of the table: 40 pages and no window take the token kernel that deals its pages evenly


@pytest.mark.parametrize("hd,H,KV", [(32, 4, 2), (64, 4, 2), (128, 2, 1)])
@pytest.mark.parametrize("n", [6, 60])
@pytest.mark.parametrize("width", WIDTHS)
def test_a_page_behind_a_rows_window_does_not_count(n, hd, H, KV, width):
    """The first token of a call sees the last key of a page whose values are 2^45 times the others', the later ones do not.  (Where the table is wide the window is long.)"""
    r = np.random.default_rng(n)
    window = 64 if width is None else 1200
    start = window + 62
    k, v = (r.standard_normal((start + n, KV, hd)) for _ in range(2))
    v[:PAGE] *= 2.0 ** 45
    check(pages_of(k, v), r.standard_normal((n, H, hd)), start, hd ** -0.5, window, "bf16", width=width)


@pytest.mark.parametrize("hd,H,KV", [(32, 4, 2), (64, 12, 4), (128, 2, 1)])
@pytest.mark.parametrize("n", [1, 5, 70])
@pytest.mark.parametrize("gap", [20, 33, 45, 70])
@pytest.mark.parametrize("width", WIDTHS)
def test_weight_on_a_page_of_small_values(n, gap, hd, H, KV, width):
    """One page in the middle takes all weight but e^-100 of it; the others' values are 2^gap times as large."""
    r = np.random.default_rng(n)
    u = r.standard_normal((1, KV, hd))
    k, v = 0.02 * r.standard_normal((350, KV, hd)), r.standard_normal((350, KV, hd)) * 2.0 ** gap
    k[128:192] += u
    v[128:192] *= 2.0 ** -gap
    q = np.repeat(u, H // KV, 1) + 0.02 * r.standard_normal((n, H, hd))
    check(pages_of(k, v), q, 350 - n, 130.0 / hd, 0, "bf16", width=width)


@pytest.mark.parametrize("n", [1, 5, 70])
@pytest.mark.parametrize("seed", [0, 1, 2])
@pytest.mark.parametrize("width", WIDTHS)
def test_scores_and_scales_that_rise_and_fall(n, seed, width):
    """Every page has a level of scores and a size of values of its own, in random order: what a page adds to the result may be any share of it."""
    r = np.random.default_rng(seed)
    KV, hd, H = 2, 64, 6
    pages = 14
    u = r.standard_normal((1, KV, hd))
    u /= np.sqrt((u ** 2).mean(-1, keepdims=True))
    k, v = 0.02 * r.standard_normal((pages * PAGE, KV, hd)), r.standard_normal((pages * PAGE, KV, hd))
    for p in range(pages):
        k[p * PAGE:(p + 1) * PAGE] += u * r.uniform(-0.5, 0.5)
        v[p * PAGE:(p + 1) * PAGE] *= 2.0 ** r.integers(-50, 50)
    q = np.repeat(u, H // KV, 1) + 0.02 * r.standard_normal((n, H, hd))
    check(pages_of(k, v), q, pages * PAGE - n, 1.0, 0, "bf16", width=width)


@pytest.mark.parametrize("n", [1, 5, 70])
@pytest.mark.parametrize("width", WIDTHS)
def test_a_missing_page_does_not_count(n, width):
    """Its scale is nobody's, whatever the others' are."""
    r = np.random.default_rng(n)
    k, v = (r.standard_normal((400, 2, 64)) for _ in range(2))
    check(pages_of(k, v * 2.0 ** -50), r.standard_normal((n, 4, 64)), 400 - n, 0.125, 0, "bf16", missing=(2,), status=301, width=width)


@pytest.mark.parametrize("n", [1, 5, 70])
@pytest.mark.parametrize("size", [20.0, 300.0, 2000.0, -20.0, -300.0, -2000.0])
@pytest.mark.parametrize("width", WIDTHS)
def test_scores_that_leave_fp32_few_bits(n, size, width):
    """Equal keys and scores of 4.6e3, 1e6 and 4.6e7 in powers of two: weights are equal, whatever their page's value scale.  The last key of every second page scores 1 % less."""
    r = np.random.default_rng(n)
    k, v = np.full((400, 2, 64), abs(size)), r.standard_normal((400, 2, 64))
    for p in range(7):
        v[p * PAGE:(p + 1) * PAGE] *= 2.0 ** (-p % 5)
    k[63::128] *= 1 - 0.01 * np.sign(size)
    check(pages_of(k, v), np.full((n, 4, 64), size), 400 - n, 0.125, 0, "f16", width=width)


@pytest.mark.parametrize("n", [1, 5, 70])
@pytest.mark.parametrize("start", [0, 300])
@pytest.mark.parametrize("width", WIDTHS)
def test_scores_far_below_nothing(n, start, width):
    """All scores are about -1e34: a finite soft-max all the same, the first token's over one key among them."""
    r = np.random.default_rng(n)
    k, v = np.full((start + n, 2, 64), -2.0 ** 43), r.standard_normal((start + n, 2, 64))
    k[::3] *= 2
    check(pages_of(k, v), np.full((n, 4, 64), 2.0 ** 66), start, 0.125, 0, "bf16", width=width)
