"""The paged 8-bit cache in plain arithmetic: a dense image of every sequence, quantised page by page.

Rotations and codes follow the definition in fp32 with each product and sum rounded by itself (numpy), so codes and scales are expected bit for bit; attention is in 64 bits over the
values that the codes stand for."""
import numpy as np
import torch

PAGE, LEAST = 64, -120


def scale_of(amax):
    """Smallest power of two s with 127 * s >= amax, at least 2^-120."""
    if amax == 0:
        return np.float32(2.0 ** LEAST)
    e = int(np.ceil(np.log2(np.float64(amax) / 127.0)))
    while 127.0 * 2.0 ** e < float(amax):
        e += 1
    while 127.0 * 2.0 ** (e - 1) >= float(amax):
        e -= 1
    return np.float32(2.0 ** max(e, LEAST))


def rotate(x, pos, cos_sin, rope_type):
    """x fp32 [n, heads, hd], pos [n] -> rotated fp32, products and sums rounded one by one."""
    half = x.shape[-1] // 2
    co, si = cos_sin[pos][:, None, :half], cos_sin[pos][:, None, half:]
    a, b = (x[..., :half], x[..., half:]) if rope_type else (x[..., 0::2], x[..., 1::2])
    u, v = (a * co).astype(np.float32) - (b * si).astype(np.float32), (a * si).astype(np.float32) + (b * co).astype(np.float32)
    out = np.empty_like(x)
    if rope_type:
        out[..., :half], out[..., half:] = u, v
    else:
        out[..., 0::2], out[..., 1::2] = u, v
    return out


class Seq:
    """One sequence's pages: codes int8 [2, pages, KV, 64, hd] (keys, values), scales fp32 [2, pages, KV]."""

    def __init__(self, KV, hd):
        self.KV, self.hd, self.n = KV, hd, 0
        self.codes = np.zeros((2, 0, KV, PAGE, hd), np.int8)
        self.scales = np.zeros((2, 0, KV), np.float32)

    def append(self, k, v):
        """k, v fp32 [n, KV, hd]: keys after their rotation."""
        n = k.shape[0]
        need = (self.n + n + PAGE - 1) // PAGE - self.codes.shape[1]
        if need > 0:
            self.codes = np.concatenate([self.codes, np.zeros((2, need) + self.codes.shape[2:], np.int8)], 1)
            self.scales = np.concatenate([self.scales, np.zeros((2, need, self.KV), np.float32)], 1)
        for which, x in enumerate((k, v)):
            x = np.where(np.isfinite(x), x, np.float32(0))
            for p in range(self.n // PAGE, (self.n + n + PAGE - 1) // PAGE):
                lo, hi = max(self.n, p * PAGE), min(self.n + n, (p + 1) * PAGE)
                off = lo - p * PAGE
                for g in range(self.KV):
                    y = x[lo - self.n:hi - self.n, g]
                    s = scale_of(np.abs(y).max())
                    if off:
                        was = self.scales[which, p, g]
                        s = max(s, was)
                        old = self.codes[which, p, g, :off].astype(np.float32) * (was / s)
                        self.codes[which, p, g, :off] = np.rint(old).astype(np.int8)
                    self.scales[which, p, g] = s
                    self.codes[which, p, g, off:off + hi - lo] = np.rint(y / s).astype(np.int8)
        self.n += n

    def held(self):
        """Keys and values fp64 [n, KV, hd]."""
        x = self.codes.astype(np.float64) * self.scales.astype(np.float64)[..., None, None]
        x = x.transpose(0, 1, 3, 2, 4).reshape(2, -1, self.KV, self.hd)
        return x[0, :self.n], x[1, :self.n]


def attention(q, k, v, start, scale, window):
    """q fp64 [n, H, hd] of the tokens start ..., k and v fp64 [tokens, KV, hd] -> (out, softmax @ |v|) fp64 [n, H, hd]."""
    n, H, hd = q.shape
    G = H // k.shape[1]
    pos, key = start + np.arange(n)[:, None], np.arange(k.shape[0])[None]
    sees = (key <= pos) & ((key > pos - window) if window > 0 else True)
    out, mag = np.zeros_like(q), np.zeros_like(q)
    for h in range(H):
        z = np.where(sees, (q[:, h] @ k[:, h // G].T) * scale, -np.inf)
        p = np.exp(z - z.max(1, keepdims=True))
        p /= p.sum(1, keepdims=True)
        out[:, h], mag[:, h] = p @ v[:, h // G], p @ np.abs(v[:, h // G])
    return out, mag


class Pool:
    """Device pool with the pages of sequences at random places; unused pages hold what must not be seen."""

    def __init__(self, paged, pages, KV, hd, device="cuda", seed=0):
        self.p = paged.new_pages(pages, KV, hd, device)
        g = torch.Generator().manual_seed(seed)
        for c in (self.p.k, self.p.v):
            c.copy_(torch.randint(-127, 128, c.shape, generator=g, dtype=torch.int8))
        for s in (self.p.ks, self.p.vs):
            s.fill_(float("nan"))
        self.order = torch.randperm(pages, generator=g).tolist()

    def table(self, tokens, width=None):
        """Table of sequences of so many tokens, -1 where no page is needed."""
        used = [(n + PAGE - 1) // PAGE for n in tokens]
        t = np.full((len(tokens), max(max(used), width or 1)), -1, np.int32)
        for b, u in enumerate(used):
            for j in range(u):
                t[b, j] = self.order.pop()
        return torch.from_numpy(t).cuda()

    def fill(self, table, b, seq):
        """Puts an oracle sequence into its pages (tokens past its end keep what is there)."""
        for j in range(seq.codes.shape[1]):
            i, m = int(table[b, j]), min(PAGE, seq.n - j * PAGE)
            self.p.k[i, :, :m] = torch.from_numpy(seq.codes[0, j, :, :m]).cuda()
            self.p.v[i, :, :, :m] = torch.from_numpy(seq.codes[1, j, :, :m]).cuda().transpose(1, 2)
            self.p.ks[i] = torch.from_numpy(seq.scales[0, j]).cuda()
            self.p.vs[i] = torch.from_numpy(seq.scales[1, j]).cuda()

    def codes(self, table, b, n):
        """(k codes, v codes, k scales, v scales) of the first n tokens of sequence b on the host: [tokens, KV, hd], [pages, KV]."""
        ids = table[b, :(n + PAGE - 1) // PAGE].long()
        k = self.p.k[ids].permute(0, 2, 1, 3).reshape(-1, self.p.k.shape[1], self.p.k.shape[3])[:n]
        v = self.p.v[ids].permute(0, 3, 1, 2).reshape(-1, self.p.k.shape[1], self.p.k.shape[3])[:n]
        return k.cpu().numpy(), v.cpu().numpy(), self.p.ks[ids].cpu().numpy(), self.p.vs[ids].cpu().numpy()
