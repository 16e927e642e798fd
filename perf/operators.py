"""The operators of the paged 8-bit key/value cache (``ghassan_b200.ops.paged``): calls of real sizes, with plain forms and 64-bit results.

The cache is a pool of pages of 64 tokens.  A page holds, for each key head, 64 x hd codes of keys (``k`` [pages, KV, 64, hd]) and of values,
with the tokens innermost (``v`` [pages, KV, hd, 64]), and one power of two a page and head for each (``ks``, ``vs`` [pages, KV]): a code c stands for c * scale.
Sequence b of a call has ``start[b]`` tokens in its pages ``table[b]`` and ``count[b]`` new ones, which are the rows ``first[b]`` ... of the call's
tensors.  Table entries that no token needs are -1.

``append``  rotates queries and keys by their positions, and stores keys and values; the case reads back the pages that it wrote to.
``attn``    the new tokens' queries against the cache, which holds their own keys already: each sees the tokens up to its own, at most ``window`` of them.
``read``    tokens of the cache as 16-bit rows.
"""
import math

import numpy as np
import torch

own = False
PAGE = 64
DT = {"f16": torch.float16, "bf16": torch.bfloat16}
LEAST = -120                       # exponent of the scale of a page of zeros


# ------------------------------------------------------------------------------------------ cases
def listed():
    c = []

    def add(name, op, B, H, KV, hd, dtype, start, count, window=0):
        c.append(dict(name=name, op=op, B=B, H=H, KV=KV, hd=hd, dtype=dtype, start_lo=start[0], start_hi=start[1], count_lo=count[0], count_hi=count[1],
                      window=window))

    # one chat's next token: nothing but latency
    add("append_token_1", "append", 1, 12, 4, 64, "f16", (1000, 1000), (1, 1))
    # portions of long prompts that begin inside a page
    add("append_prompts", "append", 6, 32, 8, 128, "bf16", (0, 4001), (511, 2047))
    # one chat's next token after a short and after a very long text
    add("token_1_short", "attn", 1, 12, 4, 64, "f16", (500, 500), (1, 1))
    add("token_1_long", "attn", 1, 32, 8, 128, "bf16", (100001, 100001), (1, 1))
    # the token step of batches of texts of all lengths
    add("tokens_32", "attn", 32, 12, 4, 64, "f16", (3, 4095), (1, 1))
    add("tokens_192", "attn", 192, 8, 2, 64, "bf16", (100, 8000), (1, 1))
    # a few proposed tokens a sequence, checked at once, with a window
    add("drafts_16", "attn", 16, 12, 4, 64, "bf16", (900, 6000), (4, 5), 2500)
    # a prompt into an empty cache; a batch of prompts of all lengths behind a shared opening; a portion of a long text
    add("prompt_1024", "attn", 1, 12, 4, 64, "f16", (0, 0), (1024, 1024))
    add("prompts_ragged", "attn", 7, 12, 4, 64, "bf16", (0, 1777), (1, 3333))
    add("portion_long", "attn", 1, 32, 8, 128, "f16", (14000, 14000), (2048, 2048))
    # the last tokens of a batch, and a whole text, leave the cache in 16 bits
    add("read_tails", "read", 9, 8, 2, 64, "bf16", (0, 3900), (1, 100))
    add("read_text", "read", 1, 32, 8, 128, "f16", (0, 0), (60000, 60000))
    return c


def draw(rng):
    def log_int(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    H, KV, hd = rng.choice([(4, 2, 32), (8, 2, 64), (12, 4, 64), (12, 12, 64), (16, 2, 64), (32, 8, 128), (16, 4, 128), (7, 1, 128)])
    c = dict(op=rng.choice(["append", "attn", "attn", "attn", "read"]), H=H, KV=KV, hd=hd, dtype=rng.choice(["f16", "bf16"]), window=0)
    kind = rng.choice(["tokens", "drafts", "prompts"]) if c["op"] != "read" else "prompts"
    c["B"] = log_int(1, 192 if kind != "prompts" else 16)
    most = min(65536, 190000 // c["B"]) * 512 // (KV * hd) if kind != "prompts" else 6000 // c["B"]
    c["start_hi"] = log_int(1, max(2, most))
    c["start_lo"] = rng.choice([0, c["start_hi"] // 3, c["start_hi"]])
    c["count_lo"], c["count_hi"] = (1, 1)
    if kind == "drafts":
        c["count_hi"] = rng.randint(2, 12)
    if kind == "prompts":
        c["count_hi"] = log_int(13, max(14, 3800 // c["B"]))
        c["count_lo"] = rng.choice([0, 1, c["count_hi"]])
    if c["op"] == "attn" and rng.random() < 0.3:
        c["window"] = log_int(1, c["start_hi"] + c["count_hi"])
    return c


def lengths(case):
    """start and count of every sequence: spread evenly over their ranges, each in its own order."""
    B, at = case["B"], np.arange(case["B"])
    a, b = (at * 0.6180339887498949) % 1.0, (at * 0.7548776662466927 + 0.5) % 1.0
    if B > 1:
        a[0], b[B - 1] = 1.0, 1.0
    else:
        a[0] = b[0] = 1.0
    start = case["start_lo"] + np.floor(a * (case["start_hi"] - case["start_lo"])).astype(np.int64)
    count = case["count_lo"] + np.floor(b * (case["count_hi"] - case["count_lo"])).astype(np.int64)
    return start, count


def visible(case):
    """Pairs of a query and a key that it sees, and keys that any query of its sequence sees, over all sequences."""
    start, count = lengths(case)
    pairs = keys = 0
    for s, n in zip(start.tolist(), count.tolist()):
        seen = np.arange(s + 1, s + n + 1)
        if case["window"] > 0:
            seen = np.minimum(seen, case["window"])
        pairs += int(seen.sum())
        keys += min(s + n, n - 1 + case["window"]) if case["window"] > 0 and n > 0 else (s + n if n else 0)
    return pairs, keys


def work(case):
    H, KV, hd = case["H"], case["KV"], case["hd"]
    start, count = lengths(case)
    n, at0 = int(count.sum()), start // PAGE * PAGE
    if case["op"] == "attn":
        pairs, keys = visible(case)
        return {"bytes": 2 * n * H * hd * 2 + keys * KV * hd * 2 + (keys // PAGE + case["B"]) * KV * 8, "flops": 4 * pairs * H * hd}
    if case["op"] == "read":
        return {"bytes": n * KV * hd * 2 * 3, "flops": n * KV * hd * 2}
    back = int(np.where(count > 0, start + count - at0, 0).sum())
    return {"bytes": n * (H + 2 * KV) * hd * 2 + n * H * hd * 2 + n * hd * 4 + n * KV * hd * 2 + back * KV * hd * 2 * 3,
            "flops": n * (H + KV) * hd * 3 + n * KV * hd * 4}


# ------------------------------------------------------------------------------------------ inputs
def exponent(amax):
    """Smallest e with 127 * 2^e >= amax, at least LEAST."""
    m, x = torch.frexp(amax)
    e = torch.where(m > 127 / 128, x - 6, x - 7)
    return torch.where(amax > 0, e, torch.full_like(e, LEAST)).clamp_min(LEAST)


def prepare(case, seed):
    dev, dt = torch.device("cuda"), DT[case["dtype"]]
    B, H, KV, hd = case["B"], case["H"], case["KV"], case["hd"]
    start, count = lengths(case)
    g = torch.Generator(device=dev).manual_seed(1000003 * int(seed) + 17)
    used = (start + count + PAGE - 1) // PAGE
    W, pages = int(max(1, used.max())), int(used.sum()) + 1
    order = torch.randperm(pages, generator=g, device=dev).cpu().numpy()
    table = np.full((B, W), -1, dtype=np.int32)
    at = 0
    for b in range(B):
        table[b, :used[b]] = order[at:at + used[b]]
        at += used[b]
    s = {"case": case, "table": torch.from_numpy(table).to(dev)}
    for name in ("k", "v"):
        # some dimensions of keys are several times larger than others, heads differ
        size = torch.exp(0.6 * torch.randn(1, KV, 1, hd, generator=g, device=dev))
        codes, scales = [], []
        for lo in range(0, pages, 4096):
            x = torch.randn(min(4096, pages - lo), KV, PAGE, hd, generator=g, device=dev) * size
            e = exponent(x.abs().amax((2, 3)))
            sc = torch.ldexp(torch.ones_like(x[:, :, 0, 0]), e)
            q = torch.round(x / sc[:, :, None, None]).to(torch.int8)
            codes.append(q if name == "k" else q.transpose(2, 3).contiguous())
            scales.append(sc)
        s[name], s[name + "s"] = torch.cat(codes), torch.cat(scales)
    first = np.concatenate([[0], np.cumsum(count)])
    n = int(first[-1])
    s["n"], s["max_new"] = n, int(count.max())
    for name, a in (("start", start), ("count", count), ("first", first[:-1])):
        s[name] = torch.from_numpy(a.astype(np.int32)).to(dev)
    if case["op"] == "append":
        s["qkv"] = torch.randn(max(n, 1), (H + 2 * KV) * hd, generator=g, device=dev).to(dt)
        far = int((start + count).max()) + 1
        ang = torch.arange(far, dtype=torch.float64)[:, None] * (1e4 ** (-torch.arange(0, hd, 2, dtype=torch.float64) / hd))[None]
        s["cos_sin"] = torch.cat([torch.cos(ang), torch.sin(ang)], 1).float().to(dev)
        at0 = start // PAGE * PAGE                          # the pages that are written to, from their first token
        back = np.where(count > 0, start + count - at0, 0)
        s["back_n"], s["back_max"] = int(back.sum()), int(back.max())
        for name, a in (("back_start", at0), ("back_count", back), ("back_first", np.cumsum(back) - back)):
            s[name] = torch.from_numpy(a.astype(np.int32)).to(dev)
    elif case["op"] == "attn":
        s["q"] = (torch.randn(max(n, 1), H * hd, generator=g, device=dev) * 1.3).to(dt)
    return s


# ------------------------------------------------------------------------------------------ passes
def run(s):
    return run_own(s) if own else {"append": plain_append, "attn": plain_attn, "read": plain_read}[s["case"]["op"]](s)


def run_own(s):
    from ghassan_b200.ops import paged as P
    c = s["case"]
    pages = P.Pages(s["k"], s["ks"], s["v"], s["vs"])
    if c["op"] == "append":
        q = P.append(pages, s["qkv"], s["table"], s["start"], s["max_new"], s["cos_sin"], c["H"], first=s["first"], count=s["count"], rope_type=1)
        return q, *P.read(pages, s["table"], s["back_start"], s["back_max"], s["qkv"].dtype, s["back_n"], first=s["back_first"], count=s["back_count"])
    if c["op"] == "attn":
        return P.attn(pages, s["q"], s["table"], s["start"], s["max_new"], c["H"], 1.0 / math.sqrt(c["hd"]), window=c["window"], first=s["first"],
                      count=s["count"])
    return P.read(pages, s["table"], s["start"], s["max_new"], DT[c["dtype"]], s["n"], first=s["first"], count=s["count"])


def rows_of(start, count, first, longest):
    """[B, longest] positions of the tokens of a call, the rows that hold them, and which of them there are."""
    i = torch.arange(max(longest, 1), device=start.device)
    there = i[None] < count[:, None]
    return start[:, None].long() + i[None], torch.where(there, first[:, None].long() + i[None], 0), there


def to16(x, dt):
    top = torch.finfo(dt).max
    return x.clamp(-top, top).to(dt)


def plain_read(s, start="start", count="count", first="first", n="n", longest="max_new"):
    dt = DT[s["case"]["dtype"]]
    pos, row, there = rows_of(s[start], s[count], s[first], s[longest])
    page = torch.gather(s["table"].long(), 1, (pos // PAGE).clamp_max(s["table"].shape[1] - 1))[there]
    at = (pos % PAGE)[there]
    out = []
    for x, sc in ((s["k"][page, :, at], s["ks"]), (s["v"][page, :, :, at], s["vs"])):
        y = torch.empty(s[n], x.shape[1], x.shape[2], dtype=dt, device=x.device)
        y[row[there]] = to16(x.float() * sc[page][:, :, None], dt)
        out.append(y)
    return tuple(out)


def plain_append(s):
    c = s["case"]
    B, H, KV, hd, dt = c["B"], c["H"], c["KV"], c["hd"], DT[c["dtype"]]
    pos, row, there = rows_of(s["start"], s["count"], s["first"], s["max_new"])
    x = s["qkv"].float().view(-1, H + 2 * KV, hd)
    where = torch.empty(s["n"], dtype=torch.long, device=x.device)
    where[row[there]] = pos[there]
    cs = s["cos_sin"][where][:, None]
    co, si = cs[..., :hd // 2], cs[..., hd // 2:]
    x = x[:s["n"]]
    a, b = x[:, :H + KV, :hd // 2], x[:, :H + KV, hd // 2:]
    rot = torch.cat([a * co - b * si, a * si + b * co], -1)
    q = rot[:, :H].reshape(-1, H * hd).to(dt)
    # the pages written to, as [B, pages of a sequence, 64 tokens]
    P = (s["max_new"] + 2 * PAGE - 2) // PAGE
    off = (s["start"] % PAGE).long()
    slot = torch.arange(P * PAGE, device=x.device)[None] - off[:, None]                     # which new token
    new = (slot >= 0) & (slot < s["count"][:, None])
    src = torch.where(new, s["first"][:, None] + slot, 0)
    touched = new.view(B, P, PAGE).any(2)
    old = (slot < 0).view(B, P, PAGE)
    number = (s["start"][:, None] // PAGE + torch.arange(P, device=x.device)[None]).clamp_max(s["table"].shape[1] - 1).long()
    page = torch.gather(s["table"].long(), 1, number).clamp_min(0)
    for codes, scales, y in ((s["k"], s["ks"], rot[:, H:]), (s["v"].transpose(2, 3), s["vs"], x[:, H + KV:])):
        y = torch.nan_to_num(y, 0.0, 0.0, 0.0)[src].view(B, P, PAGE, KV, hd).permute(0, 1, 3, 2, 4)
        y = torch.where(new.view(B, P, 1, PAGE, 1), y, 0.0)
        was = torch.where(old.any(2)[..., None], scales[page], 0.0)                         # [B, P, KV]
        scale = torch.maximum(torch.ldexp(torch.ones_like(was), exponent(y.abs().amax((3, 4)))), was)
        held = codes[page]
        code = torch.where(new.view(B, P, 1, PAGE, 1), torch.round(y / scale[..., None, None]),
                           torch.where(old[:, :, None, :, None], torch.round(held.float() * (was / scale)[..., None, None]), held.float())).to(torch.int8)
        codes[page[touched]] = code[touched]
        scales[page[touched]] = scale[touched]
    return q, *plain_read(s, "back_start", "back_count", "back_first", "back_n", "back_max")


def plain_attn(s):
    c = s["case"]
    B, H, KV, hd, dt = c["B"], c["H"], c["KV"], c["hd"], DT[c["dtype"]]
    pos, row, there = rows_of(s["start"], s["count"], s["first"], s["max_new"])
    W = s["table"].shape[1]
    page = s["table"].long().clamp_min(0)
    k = (s["k"][page].float() * s["ks"][page][..., None, None]).transpose(1, 2).reshape(B, KV, W * PAGE, hd)
    v = (s["v"][page].float() * s["vs"][page][..., None, None]).permute(0, 2, 1, 4, 3).reshape(B, KV, W * PAGE, hd)
    G, N = H // KV, pos.shape[1]
    q = s["q"].float().view(-1, H, hd)[row].view(B, N, KV, G, hd).permute(0, 2, 1, 3, 4).reshape(B, KV, N * G, hd)
    sc = torch.matmul(q, k.transpose(2, 3)).view(B, KV, N, G, W * PAGE).mul_(1.0 / math.sqrt(hd))
    key = torch.arange(W * PAGE, device=q.device)
    sees = (key[None, None] <= pos[..., None]) & there[..., None]
    if c["window"] > 0:
        sees &= key[None, None] > pos[..., None] - c["window"]
    sc.masked_fill_(~sees[:, None, :, None], -math.inf)
    sc -= sc.amax(-1, keepdim=True).clamp_min(-1e30)
    p = sc.exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(B, KV, N * G, W * PAGE), v).view(B, KV, N, G, hd) / torch.where(total > 0, total, 1.0)
    out = torch.empty(s["n"], H * hd, dtype=dt, device=q.device)
    out[row[there]] = o.permute(0, 2, 1, 3, 4).reshape(B, N, H * hd)[there].to(dt)
    return out


# ------------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    """Sequence by sequence and head by head, in 64 bits."""
    s = prepare(case, seed)
    H, KV, hd, G = case["H"], case["KV"], case["hd"], case["H"] // case["KV"]
    start, count = lengths(case)
    first = np.cumsum(count) - count
    if case["B"] * KV > 2000:
        return None
    f64 = dict(dtype=torch.float64, device="cuda")
    tab = s["table"].cpu().numpy()

    def held(b, lo, hi):
        """Keys and values of the tokens lo ... hi - 1 of sequence b: [KV, tokens, hd] each."""
        p0, p1 = lo // PAGE, (hi + PAGE - 1) // PAGE
        pg = torch.from_numpy(tab[b, p0:p1].astype(np.int64)).cuda()
        kk = (s["k"][pg].double() * s["ks"][pg].double()[:, :, None, None]).permute(1, 0, 2, 3).reshape(KV, -1, hd)
        vv = (s["v"][pg].double() * s["vs"][pg].double()[:, :, None, None]).permute(1, 0, 3, 2).reshape(KV, -1, hd)
        return kk[:, lo - p0 * PAGE:hi - p0 * PAGE], vv[:, lo - p0 * PAGE:hi - p0 * PAGE]

    if case["op"] == "attn":
        out = torch.zeros(s["n"], H * hd, **f64)
        for b in range(case["B"]):
            st, n, f = int(start[b]), int(count[b]), int(first[b])
            if n == 0:
                continue
            lo = max(0, st + 1 - case["window"]) if case["window"] > 0 else 0
            kk, vv = held(b, lo, st + n)
            mine = torch.arange(st, st + n, device="cuda")[:, None]
            key = torch.arange(lo, st + n, device="cuda")[None]
            hidden = (key > mine) | ((key <= mine - case["window"]) if case["window"] > 0 else (key < 0))
            for h in range(H):
                z = s["q"][f:f + n, h * hd:(h + 1) * hd].double() @ kk[h // G].T / math.sqrt(hd)
                z[hidden] = -math.inf
                out[f:f + n, h * hd:(h + 1) * hd] = torch.softmax(z, 1) @ vv[h // G]
        return out
    top = float(torch.finfo(DT[case["dtype"]]).max)
    if case["op"] == "read":
        k, v = torch.zeros(s["n"], KV, hd, **f64), torch.zeros(s["n"], KV, hd, **f64)
        for b in range(case["B"]):
            st, n, f = int(start[b]), int(count[b]), int(first[b])
            if n:
                kk, vv = held(b, st, st + n)
                k[f:f + n], v[f:f + n] = kk.transpose(0, 1).clamp(-top, top), vv.transpose(0, 1).clamp(-top, top)
        return k, v
    x = s["qkv"].double().view(-1, H + 2 * KV, hd)
    table = s["cos_sin"].double()
    q = torch.zeros(s["n"], H * hd, **f64)
    back = [torch.zeros(s["back_n"], KV, hd, **f64) for _ in range(2)]
    at = 0
    for b in range(case["B"]):
        st, n, f = int(start[b]), int(count[b]), int(first[b])
        if n == 0:
            continue
        t = x[f:f + n]
        co, si = table[st:st + n, None, :hd // 2], table[st:st + n, None, hd // 2:]
        lo, hi = t[..., :hd // 2], t[..., hd // 2:]
        turned = torch.cat([lo * co - hi * si, hi * co + lo * si], 2)
        q[f:f + n] = turned[:, :H].reshape(n, -1)
        off = st % PAGE
        if off:
            pg = int(tab[b, st // PAGE])
        for which, news in enumerate((turned[:, H:H + KV], t[:, H + KV:])):
            for p in range((off + n + PAGE - 1) // PAGE):
                lo_, hi_ = max(0, p * PAGE - off), min(n, (p + 1) * PAGE - off)
                y = news[lo_:hi_]                                                           # [tokens, KV, hd]
                e = torch.ceil(torch.log2(y.abs().amax((0, 2)) / 127.0))
                if p == 0 and off:
                    was = (s["ks"], s["vs"])[which][pg].double()
                    sc = torch.maximum(torch.exp2(e), was)
                    c = s["k"][pg, :, :off].double().transpose(0, 1) if which == 0 else s["v"][pg, :, :, :off].double().permute(2, 0, 1)
                    back[which][at:at + off] = torch.round(c * (was / sc)[:, None]) * sc[:, None]
                else:
                    sc = torch.exp2(e)
                back[which][at + off + lo_:at + off + hi_] = torch.round(y / sc[:, None]) * sc[:, None]
        at += off + n
    return q, back[0].clamp(-top, top), back[1].clamp(-top, top)
