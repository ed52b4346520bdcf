"""The paged-cache and cross-attention operators as a measured set.

Four operators of a block-causal video transformer's layer that belong
together: K/V rows quantised into a paged cache as they are written
(``write``), read back as bf16 (``read``), attention of new tokens over the
cache's pages (``attention``), and cross attention to an encoder's states of
another length (``cross``).  ``run`` computes each in plain torch operations in
32 bits, or, with ``own`` set, through the package's entry points.

Head dim is 128 everywhere, the only one the package's attention has.  Lengths
of ragged batches follow from the case alone, values and the order of pages
from the seed.
"""

import math
import random

import torch

own = False

DEV = "cuda"
D = 128
QMAX = {"e4m3": 448.0, "int8": 127.0}


def listed():
    return [
        # the smallest call: one new token of one short sequence, the two-head test model
        dict(name="attention_token_tiny", op="attention", cache="bf16", seqs=1, new=1, context=130, heads=2, kv_heads=2,
             page=16, block=1, window=0, sink=0, ragged=False),
        # single tokens of a served batch with shared K/V heads, ragged contexts
        dict(name="attention_tokens_batch", op="attention", cache="e4m3", seqs=32, new=1, context=8192, heads=40,
             kv_heads=8, page=64, block=1, window=0, sink=0, ragged=True),
        # ragged causal prompts over a small-page int8 cache, shared K/V heads
        dict(name="attention_prompts_ragged", op="attention", cache="int8", seqs=6, new=1000, context=4001, heads=16,
             kv_heads=4, page=16, block=1, window=0, sink=0, ragged=True),
        # a 40-head chunk over an anchor chunk and a window of the recent ones, e4m3 pages
        dict(name="attention_chunk_window", op="attention", cache="e4m3", seqs=1, new=4680, context=18720, heads=40,
             kv_heads=40, page=64, block=4680, window=9360, sink=4680, ragged=False),
        # the largest: a 12-head chunk over eight chunks of bf16 frame pages
        dict(name="attention_chunk_frames", op="attention", cache="bf16", seqs=1, new=4680, context=37440, heads=12,
             kv_heads=12, page=1560, block=4680, window=0, sink=0, ragged=False),
        # one chunk's clean K/V written as it is promoted, frame pages
        dict(name="write_chunk", op="write", cache="e4m3", seqs=1, new=4680, context=9360, heads=12, kv_heads=12,
             page=1560, ragged=False),
        # six stages' chunks of the 40-head model at once
        dict(name="write_six_chunks", op="write", cache="e4m3", seqs=6, new=4680, context=4680, heads=40, kv_heads=40,
             page=64, ragged=False),
        # a served step's tokens written and read back, one per sequence
        dict(name="roundtrip_tokens", op="roundtrip", cache="int8", seqs=64, new=1, context=2048, heads=8, kv_heads=8,
             page=64, ragged=True),
        # five chunks of context read back, as an export of the cache does
        dict(name="read_context", op="read", cache="e4m3", seqs=1, new=23400, context=23400, heads=12, kv_heads=12,
             page=1560, ragged=False),
        # ragged sequences of a small-page cache read back
        dict(name="read_ragged", op="read", cache="int8", seqs=7, new=3001, context=4500, heads=8, kv_heads=8, page=16,
             ragged=True),
        # six stages' chunks against six prompts of their own lengths, padded to 512 text tokens
        dict(name="cross_six_stages", op="cross", seqs=6, new=4680, context=512, heads=12, kv_heads=12, masked=False,
             ragged=True),
        # single tokens against masked encoder states of an odd length
        dict(name="cross_tokens_masked", op="cross", seqs=24, new=1, context=257, heads=40, kv_heads=40, masked=True,
             ragged=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    op = rng.choice(["attention", "attention", "attention", "write", "read", "roundtrip", "cross", "cross"])
    kv = rng.choice([1, 2, 3, 4, 5, 8, 12])
    heads = kv * rng.choice([1, 1, 2, 3, 4, 5])
    if op == "cross":
        new = rng.choice([1, rng.randint(2, 60), _log(rng, 61, 4680)])
        return dict(op=op, seqs=rng.randint(1, 24 if new < 500 else 6), new=new, context=_log(rng, 3, 1024), heads=heads,
                    kv_heads=kv, masked=rng.random() < 0.5, ragged=rng.random() < 0.6)
    c = dict(op=op, cache=rng.choice(["bf16", "e4m3", "int8"]), kv_heads=kv, page=rng.choice([16, 24, 64, 100, 128, 390, 1560]),
             ragged=rng.random() < 0.7)
    if op != "attention":
        new = _log(rng, 1, 9000)
        return dict(c, seqs=rng.randint(1, 64 if new < 300 else 4), new=new, context=new + _log(rng, 1, 3000), heads=kv)
    kind = rng.choice(["token", "few", "prompt", "chunk"])
    if kind == "token":
        c.update(seqs=_log(rng, 1, 48), new=1, context=_log(rng, 5, 9000), block=1)
    elif kind == "few":
        c.update(seqs=rng.randint(1, 8), new=rng.randint(2, 48), context=_log(rng, 50, 20000), block=rng.choice([0, 1]))
    elif kind == "prompt":
        new = _log(rng, 49, 1200)
        c.update(seqs=rng.randint(1, 4), new=new, context=new + _log(rng, 1, 3000), block=1)
    else:
        frame, heads = rng.choice([390, 1560]), kv
        c.update(seqs=1, new=3 * frame, context=3 * frame * rng.randint(1, 6), block=3 * frame)
    window = rng.random() < 0.4
    return dict(c, heads=heads, window=_log(rng, 3, 9000) if window else 0,
                sink=_log(rng, 1, 2000) if window and rng.random() < 0.7 else 0)


# ------------------------------------------------------------------ lengths
def _lens(c):
    """(new tokens, total length) of each sequence, from the case alone."""
    r = random.Random(c["seqs"] * 1000003 + c["new"] * 10007 + c["context"])
    new, total = [], []
    for b in range(c["seqs"]):
        n = r.randint(1, c["new"]) if c["ragged"] and b else c["new"]
        t = _log(r, max(n, c["context"] // 8, 1), max(n, c["context"])) if c["ragged"] and b else max(n, c["context"])
        new.append(n)
        total.append(t)
    return new, total


def _cross_lens(c):
    r = random.Random(c["seqs"] * 1000003 + c["new"] * 10007 + c["context"])
    return [r.randint(1, c["context"]) if c["ragged"] else c["context"] for _ in range(c["seqs"])]


def _hi_lo(c, n, t):
    """Visible range [lo, hi) and sink of each new position of one sequence."""
    for p in range(t - n, t):
        hi = min(t, (p // c["block"] + 1) * c["block"]) if c["block"] else t
        lo = max(0, hi - c["window"]) if c["window"] else 0
        yield hi, lo, min(c["sink"], lo) if c["window"] else 0


def work(c):
    H, G = c["heads"], c["kv_heads"]
    if c["op"] == "cross":
        lens, B, n = _cross_lens(c), c["seqs"], c["new"]
        keys = sum(lens) * (0.75 if c["masked"] else 1.0)
        return {"bytes": 2 * D * (2 * B * n * H + 2 * keys * G), "flops": 4 * D * H * n * keys}
    new, total = _lens(c)
    rows = sum(new)
    kv = 2 * D if c["cache"] == "bf16" else D + 4  # bytes of one cached row of one head
    if c["op"] in ("write", "read"):
        return {"bytes": 2 * rows * G * (2 * D + kv), "flops": 0}
    if c["op"] == "roundtrip":
        return {"bytes": 2 * rows * G * 2 * (2 * D + kv), "flops": 0}
    pairs, keys = 0, 0
    for n, t in zip(new, total):
        seen = [(hi, lo, s) for hi, lo, s in _hi_lo(c, n, t)]
        pairs += sum(hi - lo + s for hi, lo, s in seen)
        first = min(lo for _, lo, _ in seen)
        keys += max(hi for hi, _, _ in seen) - first + min(first, max(s for _, _, s in seen))
    return {"bytes": 2 * D * 2 * rows * H + 2 * keys * G * kv, "flops": 4 * D * H * pairs}


# ------------------------------------------------------------------- inputs
def prepare(c, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def randn(*shape):
        return torch.randn(shape, generator=g, device=DEV, dtype=torch.bfloat16)

    if c["op"] == "cross":
        B, Lk, G = c["seqs"], c["context"], c["kv_heads"]
        s = dict(case=c, q=randn(B, c["new"], c["heads"], D), k=randn(B, Lk, G, D), v=randn(B, Lk, G, D), lens=None,
                 mask=None)
        if c["ragged"]:
            s["lens"] = torch.tensor(_cross_lens(c), device=DEV, dtype=torch.int32)
        if c["masked"]:
            s["mask"] = torch.rand((B, Lk), generator=g, device=DEV) < 0.75
        return s
    new, total = _lens(c)
    ps, G, rows = c["page"], c["kv_heads"], sum(new)
    need = [-(-t // ps) for t in total]
    pool = sum(need) + 3
    table = torch.zeros((c["seqs"], max(need)), dtype=torch.int32)
    order = torch.randperm(pool, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    s = dict(case=c, table=table.to(DEV), rows=rows, max_new=max(new), max_len=max(total),
             cu=torch.tensor([0] + new).cumsum(0).to(torch.int32).to(DEV),
             lens=torch.tensor(total, dtype=torch.int32).to(DEV), k_scale=None, v_scale=None)
    if c["op"] in ("write", "roundtrip"):
        # a pool as it is first allocated; rows as they leave the projections, some channels larger than the others
        dt = {"bf16": torch.bfloat16, "e4m3": torch.uint8, "int8": torch.int8}[c["cache"]]
        s["kp"], s["vp"] = (torch.zeros((pool, G, ps, D), device=DEV, dtype=dt) for _ in range(2))
        if c["cache"] != "bf16":
            s["k_scale"], s["v_scale"] = (torch.zeros((pool, G, ps), device=DEV) for _ in range(2))
        gain = torch.rand(D, generator=g, device=DEV) * 3 + 0.2
        s["k"], s["v"] = ((randn(rows, G, D) * gain).to(torch.bfloat16) for _ in range(2))
    else:
        for name in ("k", "v"):
            x = randn(pool, G, ps, D)
            if c["cache"] == "bf16":
                s[name + "p"] = x
            else:
                a = x.abs().amax(-1, keepdim=True).float()
                y = x.float() * (QMAX[c["cache"]] / a)
                s[name + "p"] = (y.to(torch.float8_e4m3fn).view(torch.uint8) if c["cache"] == "e4m3"
                                 else y.round().to(torch.int8))
                s[name + "_scale"] = (a / QMAX[c["cache"]]).squeeze(-1)
    if c["op"] == "attention":
        s["q"] = randn(rows, c["heads"], D)
    return s


# -------------------------------------------------------------- plain forms
def _token_slots(s):
    """Sequence, position, page and row of every new token."""
    cu, lens, ps = s["cu"].long(), s["lens"].long(), s["case"]["page"]
    i = torch.arange(s["rows"], device=DEV)
    b = torch.searchsorted(cu[1:], i, right=True)
    pos = lens[b] - cu[b + 1] + i
    return b, pos, s["table"][b, pos // ps].long(), pos % ps


def _codes(x, cache, wide):
    """Codes (as stored) and scales of rows [..., D]."""
    a = x.to(wide).abs().amax(-1, keepdim=True).clamp(min=2.0 ** -100)
    y = x.to(wide) * QMAX[cache] / a
    y = y.to(torch.float8_e4m3fn).view(torch.uint8) if cache == "e4m3" else y.round().to(torch.int8)
    return y, (a / QMAX[cache]).squeeze(-1)


def _values(codes, scale, cache, wide):
    if cache == "bf16":
        return codes.to(wide)
    if cache == "e4m3":
        codes = codes.view(torch.float8_e4m3fn)
    return codes.to(wide) * scale.to(wide).unsqueeze(-1)


def _write(s):
    _, _, page, row = _token_slots(s)
    for name in ("k", "v"):
        x, cache = s[name], s["case"]["cache"]
        if cache == "bf16":
            s[name + "p"][page, :, row] = x
        else:
            codes, scale = _codes(x, cache, torch.float32)
            s[name + "p"][page, :, row] = codes
            s[name + "_scale"][page, :, row] = scale


def _read(s):
    _, _, page, row = _token_slots(s)
    out = []
    for name in ("k", "v"):
        scale = s[name + "_scale"]
        out.append(_values(s[name + "p"][page, :, row], None if scale is None else scale[page, :, row],
                           s["case"]["cache"], torch.float32).to(torch.bfloat16))
    return out


def _written(s):
    c = s["case"]["cache"]
    if c == "bf16":
        return [s["kp"], s["vp"]]
    if c == "int8":  # the values the codes stand for
        return [_values(s["kp"], s["k_scale"], c, torch.float32), _values(s["vp"], s["v_scale"], c, torch.float32)]
    return [s["kp"].view(torch.float8_e4m3fn), s["k_scale"], s["vp"].view(torch.float8_e4m3fn), s["v_scale"]]


def _softmax_sum(q, k, v, keep, scale):
    """softmax over kept keys of q [.., R, D], k and v [.., L, D]; rows that keep nothing give zeros."""
    x = torch.where(keep, torch.matmul(q, k.transpose(-1, -2)) * scale, -math.inf)
    m = x.amax(-1, keepdim=True).clamp(min=-1e30)
    p = torch.exp(x - m)
    return torch.matmul(p, v) / p.sum(-1, keepdim=True).clamp(min=1e-30)


def _attention(s):
    c = s["case"]
    B, G, H, ps = c["seqs"], c["kv_heads"], c["heads"], c["page"]
    page = s["table"].long()

    def gathered(name):
        scale = s[name + "_scale"]
        x = _values(s[name + "p"][page], None if scale is None else scale[page], c["cache"], torch.float32)
        return x.transpose(1, 2).reshape(B, G, -1, D)[:, :, :s["max_len"]]

    lens, cu = s["lens"].long(), s["cu"].long()
    n = cu[1:] - cu[:-1]
    at = torch.arange(s["max_new"], device=DEV)
    q = s["q"][(cu[:-1, None] + at).clamp(max=s["rows"] - 1)].float()  # [B, Q, H, D]
    q = q.view(B, -1, G, H // G, D).permute(0, 2, 3, 1, 4).reshape(B, G, -1, D)
    pos = (lens - n)[:, None] + at  # [B, Q]
    hi = torch.minimum(lens[:, None], (pos // c["block"] + 1) * c["block"]) if c["block"] else lens[:, None].expand_as(pos)
    key = torch.arange(s["max_len"], device=DEV)
    keep = key < hi[..., None]
    if c["window"]:
        keep = keep & ((key >= hi[..., None] - c["window"]) | (key < c["sink"]))
    keep = keep[:, None, None].expand(B, 1, H // G, -1, -1).reshape(B, 1, -1, s["max_len"])
    o = _softmax_sum(q, gathered("k"), gathered("v"), keep, D ** -0.5)
    o = o.view(B, G, H // G, -1, D).permute(0, 3, 1, 2, 4).reshape(B, -1, H, D).to(torch.bfloat16)
    b, p, _, _ = _token_slots(s)
    return o[b, p - (lens - n)[b]]


def _cross(s):
    c = s["case"]
    B, G, H, Lk = c["seqs"], c["kv_heads"], c["heads"], c["context"]
    q = s["q"].float().view(B, -1, G, H // G, D).permute(0, 2, 3, 1, 4).reshape(B, G, -1, D)
    keep = torch.ones((B, Lk), dtype=torch.bool, device=DEV)
    if s["lens"] is not None:
        keep = torch.arange(Lk, device=DEV) < s["lens"][:, None]
    if s["mask"] is not None:
        keep = keep & s["mask"]
    o = _softmax_sum(q, s["k"].float().transpose(1, 2), s["v"].float().transpose(1, 2), keep[:, None, None], D ** -0.5)
    return o.view(B, G, H // G, -1, D).permute(0, 3, 1, 2, 4).reshape(B, -1, H, D).to(torch.bfloat16)


def run(s):
    op = s["case"]["op"]
    if own:
        from waveforcing_b200 import kernels

        if op == "cross":
            return kernels.cross_attention(s["q"], s["k"], s["v"], kv_lens=s["lens"], key_mask=s["mask"])
        pages = kernels.KVPages(s["kp"], s["vp"], s["k_scale"], s["v_scale"])
        plan = (s["table"], s["cu"], s["lens"])
        if op == "attention":
            c = s["case"]
            return kernels.paged_attention(s["q"], pages, *plan, max_new=s["max_new"], max_len=s["max_len"],
                                           block=c["block"], window=c["window"], sink=c["sink"])
        if op in ("write", "roundtrip"):
            kernels.paged_kv_write(pages, s["k"], s["v"], *plan)
        return _written(s) if op == "write" else list(kernels.paged_kv_read(pages, *plan, rows=s["rows"]))
    if op == "cross":
        return _cross(s)
    if op == "attention":
        return _attention(s)
    if op in ("write", "roundtrip"):
        _write(s)
    return _written(s) if op == "write" else _read(s)


# -------------------------------------------------------- 64-bit definition
def exact(c, seed):
    """From the definitions, one sequence and one head at a time, in 64 bits."""
    s = prepare(c, seed)
    G, f8 = c["kv_heads"], torch.float64
    per = c["heads"] // G

    def attend(q, k, v, keep):  # q [n, D], k and v [L, D], keep [n or 1, L]
        x = (q.to(f8) @ k.to(f8).T) / math.sqrt(D)
        x = x.masked_fill(~keep, -math.inf)
        p = torch.exp(x - x.amax(1, keepdim=True).clamp(min=-1e300))
        return (p @ v.to(f8)) / p.sum(1, keepdim=True).clamp(min=1e-300)

    if c["op"] == "cross":
        out = torch.zeros(s["q"].shape, dtype=f8, device=DEV)
        at = torch.arange(c["context"], device=DEV)
        for b, length in enumerate(_cross_lens(c)):
            keep = at < length
            if s["mask"] is not None:
                keep = keep & s["mask"][b]
            for h in range(c["heads"]):
                out[b, :, h] = attend(s["q"][b, :, h], s["k"][b, :, h // per], s["v"][b, :, h // per], keep[None])
        return out
    new, total = _lens(c)
    table, ps = s["table"].cpu().tolist(), c["page"]

    def head(name, pages, h):  # one K/V head's rows, [rows, D]
        x = s[name + "p"][pages, h]
        x = (x.view(torch.float8_e4m3fn) if c["cache"] == "e4m3" else x).to(f8)
        x = x if c["cache"] == "bf16" else x * s[name + "_scale"][pages, h].to(f8)[..., None]
        return x.reshape(-1, D)

    if c["op"] in ("write", "roundtrip"):
        spots = [(table[b][p // ps], p % ps) for b in range(c["seqs"]) for p in range(total[b] - new[b], total[b])]
        page, row = (torch.tensor(x, device=DEV) for x in zip(*spots))
        out = []
        for name in ("k", "v"):
            x = s[name].to(f8)
            if c["cache"] == "bf16":
                codes, scale, val = None, None, x
            else:
                a = x.abs().amax(-1, keepdim=True)
                y = x * QMAX[c["cache"]] / a
                codes = y.float().to(torch.float8_e4m3fn).to(f8) if c["cache"] == "e4m3" else y.round()
                scale = a / QMAX[c["cache"]]
                val = codes * scale
            if c["op"] == "roundtrip":
                out.append(val)
                continue
            whole = torch.zeros(s[name + "p"].shape, dtype=f8, device=DEV)
            whole[page, :, row] = codes if c["cache"] == "e4m3" else val
            out.append(whole)
            if c["cache"] == "e4m3":
                scales = torch.zeros(s[name + "p"].shape[:3], dtype=f8, device=DEV)
                scales[page, :, row] = scale.squeeze(-1)
                out.append(scales)
        return out
    if c["op"] == "read":
        k, v = [], []
        for b in range(c["seqs"]):
            pages = torch.tensor(table[b][:-(-total[b] // ps)], device=DEV)
            for name, to in (("k", k), ("v", v)):
                x = torch.stack([head(name, pages, h)[total[b] - new[b]:total[b]] for h in range(G)], 1)
                to.append(x)
        return [torch.cat(k), torch.cat(v)]
    out = torch.zeros(s["q"].shape, dtype=f8, device=DEV)
    first = 0
    for b in range(c["seqs"]):
        n, t = new[b], total[b]
        pages = torch.tensor(table[b][:-(-t // ps)], device=DEV)
        seen = torch.tensor(list(_hi_lo(c, n, t)), device=DEV)
        at = torch.arange(t, device=DEV)
        keep = ((at < seen[:, :1]) & (at >= seen[:, 1:2])) | (at < seen[:, 2:])
        for h in range(G):
            k, v = head("k", pages, h)[:t], head("v", pages, h)[:t]
            for e in range(per):
                out[first:first + n, h * per + e] = attend(s["q"][first:first + n, h * per + e], k, v, keep)
        first += n
    return out

