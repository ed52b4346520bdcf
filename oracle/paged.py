"""Paged K/V cache and cross attention, from their definitions in float64.

These operators have no code of their own in the reference: it copies pages
into a contiguous context (wave_rt/denoiser/exchange/paged.py:191-255), scales
whole tensors (common.py:143-150) and attends to padded text
(naive_rt/rolling_forcing/wan/modules/model.py:158-196).  The statement here is
the formulas of include/wfk.h, one row at a time.
"""

from __future__ import annotations

import torch

QMAX = {torch.uint8: 448.0, torch.int8: 127.0}
MIN_AMAX = 2.0 ** -100


def quant_rows(x: torch.Tensor, dtype: torch.dtype):
    """Rows [..., 128] -> (values of the codes, scales) in f64; NaN scale and
    zero codes for rows that are not finite."""
    xd = x.double()
    a = xd.abs().amax(-1, keepdim=True)
    ok = torch.isfinite(a)
    a = torch.where(ok, a, torch.ones_like(a)).clamp(min=MIN_AMAX)
    y = torch.where(ok, xd, torch.zeros_like(xd)) * QMAX[dtype] / a
    # the f32 step before e4m3 moves no quotient of two bf16 across a midpoint
    codes = y.float().to(torch.float8_e4m3fn).double() if dtype == torch.uint8 else y.round()
    scale = torch.where(ok, a / QMAX[dtype], torch.full_like(a, float("nan"))).squeeze(-1)
    return codes, scale


def code_values(codes: torch.Tensor) -> torch.Tensor:
    """Stored codes (uint8 e4m3, int8 or bf16) as f64."""
    return (codes.view(torch.float8_e4m3fn) if codes.dtype == torch.uint8 else codes).double()


def slots(table, cu, lens, page_size, n_pages):
    """(packed row, sequence, page, row in page) of every packed row that has a slot."""
    out = []
    for b in range(len(lens)):
        n = cu[b + 1] - cu[b]
        for i in range(n):
            p = lens[b] - n + i
            if p < 0 or p // page_size >= len(table[b]):
                continue
            page = table[b][p // page_size]
            if 0 <= page < n_pages:
                out.append((cu[b] + i, b, page, p % page_size))
    return out


def softmax_rows(q, k, v, keep, scale):
    """One head: q [n, D], k and v [L, D], keep bool [n, L] -> (o [n, D], lse [n]) in f64.
    Keys that no row keeps do not enter, whatever they hold."""
    used = keep.any(0)
    k, v, keep = k[used].double(), v[used].double(), keep[:, used]
    if k.shape[0] == 0:
        return torch.zeros(q.shape, dtype=torch.float64), torch.full((q.shape[0],), -float("inf"), dtype=torch.float64)
    x = (q.double() @ k.T * scale).masked_fill(~keep, -float("inf"))
    lse = torch.logsumexp(x, 1)
    p = torch.exp(x - torch.where(torch.isinf(lse), torch.zeros_like(lse), lse)[:, None])
    return p @ v, lse


def visible(pos: int, length: int, block: int, window: int, sink: int) -> torch.Tensor:
    """Mask [length] of the keys that the row at position pos sees."""
    hi = min(length, (pos // block + 1) * block) if block else length
    hi = 0 if pos < 0 else hi
    k = torch.arange(length)
    keep = k < hi
    if window:
        keep &= (k < sink) | (k >= hi - window)
    return keep


def paged_attention(q, pages_k, pages_v, table, cu, lens, block, window, sink, scale):
    """q [rows, H, D]; pages as f64 values [P, G, ps, D] (NaN allowed where unseen)
    -> (o, lse, written rows)."""
    rows, H, D = q.shape
    P, G, ps, _ = pages_k.shape
    o = torch.zeros((rows, H, D), dtype=torch.float64)
    lse = torch.zeros((rows, H), dtype=torch.float64)
    written = torch.zeros(rows, dtype=torch.bool)
    for b in range(len(lens)):
        n, L = cu[b + 1] - cu[b], max(0, min(lens[b], len(table[b]) * ps))
        if n == 0:
            continue
        sl = slice(cu[b], cu[b + 1])
        written[sl] = True
        ids = [table[b][j] for j in range(-(-L // ps))]
        good = torch.tensor([0 <= i < P for i in ids], dtype=torch.bool).repeat_interleave(ps)[:L]
        take = [i if 0 <= i < P else 0 for i in ids]
        keep = torch.stack([visible(lens[b] - n + i, L, block, window, sink) & good for i in range(n)])
        for h in range(H):
            g = h // (H // G)
            k = torch.cat([pages_k[i, g] for i in take] or [torch.zeros(0, D)])[:L]
            v = torch.cat([pages_v[i, g] for i in take] or [torch.zeros(0, D)])[:L]
            o[sl, h], lse[sl, h] = softmax_rows(q[sl, h], k, v, keep, scale)
    return o, lse, written


def cross_attention(q, k, v, kv_lens, key_mask, kv_index, scale):
    B, Lq, H, D = q.shape
    N, Lk, G, _ = k.shape
    o = torch.zeros(q.shape, dtype=torch.float64)
    lse = torch.zeros((B, Lq, H), dtype=torch.float64)
    for b in range(B):
        n = kv_index[b] if kv_index is not None else (0 if N == 1 else b)
        keep = torch.zeros(Lk, dtype=torch.bool)
        if 0 <= n < N:
            keep = torch.arange(Lk) < (kv_lens[n] if kv_lens is not None else Lk)
            if key_mask is not None:
                keep = keep & key_mask[n]
        else:
            n = 0
        for h in range(H):
            g = h // (H // G)
            o[b, :, h], lse[b, :, h] = softmax_rows(q[b, :, h], k[n, :, g], v[n, :, g],
                                                    keep[None].expand(Lq, Lk), scale)
    return o, lse
