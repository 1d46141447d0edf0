"""Plain 64-bit forms of the paged-cache operators, sequence by sequence, for the tests."""
from __future__ import annotations

import math

import torch


def rotate(x, cos_sin, positions, interleaved=False, inverse=False):
    R = cos_sin.shape[1]
    out = x.double().clone()
    c, s = cos_sin[positions, : R // 2].double()[:, None], cos_sin[positions, R // 2:].double()[:, None]
    if inverse:
        s = -s
    ia = torch.arange(0, R, 2) if interleaved else torch.arange(R // 2)
    ib = ia + 1 if interleaved else ia + R // 2
    a, b = x.double()[..., ia], x.double()[..., ib]
    out[..., ia], out[..., ib] = a * c - b * s, b * c + a * s
    return out


def rotate_f32(x, cos_sin, positions, interleaved=False):
    """The same in f32 with every product and sum rounded: the values that are quantised."""
    R = cos_sin.shape[1]
    out = x.float().clone()
    c, s = cos_sin[positions, : R // 2][:, None], cos_sin[positions, R // 2:][:, None]
    ia = torch.arange(0, R, 2) if interleaved else torch.arange(R // 2)
    ib = ia + 1 if interleaved else ia + R // 2
    a, b = x.float()[..., ia], x.float()[..., ib]
    out[..., ia], out[..., ib] = a * c - b * s, b * c + a * s
    return out


def append(codes, scale, x, tables, lengths, starts):
    """codes [pages, H, P, D] and scale [pages, H] (CPU copies, changed in place); x f32 [T, H, D]."""
    P = codes.shape[2]
    for b, length in enumerate(lengths):
        first, n = starts[b], starts[b + 1] - starts[b]
        if length == 0:
            continue
        for block in range((length - n) // P, -(-length // P)):
            page, lo, hi = tables[b][block], max(block * P, length - n), min(block * P + P, length)
            if hi <= lo:
                continue
            old = lo - block * P
            rows = x[first + lo - (length - n): first + hi - (length - n)]  # [new, H, D]
            amax = rows.abs().amax((0, 2))
            before = scale[page] if old else torch.zeros_like(scale[page])
            bad = ~torch.isfinite(amax) | torch.isnan(before)
            s = torch.maximum(torch.maximum(before, amax / torch.tensor(127.0)), torch.tensor(1e-12))
            if old:
                grown = (codes[page, :, :old].float() * (before / s)[:, None, None]).round().nan_to_num(0)
                keep = (bad | (before == s))[:, None, None]
                codes[page, :, :old] = torch.where(keep, codes[page, :, :old], grown.to(torch.int8))
            q = (rows / s[:, None]).round().clamp(-127, 127).nan_to_num(0).masked_fill(bad[:, None], 0.0)
            codes[page, :, old: old + hi - lo] = q.to(torch.int8).transpose(0, 1)
            scale[page] = torch.where(bad, torch.full_like(s, float("nan")), s)


def attend(q, k_codes, k_scale, v_codes, v_scale, tables, lengths, starts, scale=None, causal=True, window=0):
    """out, sum of p |v| (for bounds) and lse in 64 bits; pools [pages, H, P, D], [pages, H]."""
    T, heads, D = q.shape
    H, P = k_codes.shape[1], k_codes.shape[2]
    G = heads // H
    scale = D ** -0.5 if scale is None else scale
    out = torch.zeros(T, heads, D, dtype=torch.float64, device=q.device)
    mag, lse = torch.zeros_like(out), torch.full((T, heads), -math.inf, dtype=torch.float64, device=q.device)
    for b, length in enumerate(lengths):
        first, n = starts[b], starts[b + 1] - starts[b]
        if length == 0 or n == 0:
            continue
        pages = torch.tensor(tables[b][: -(-length // P)], device=q.device)
        # held pages of a windowed sequence may be gone: nothing in them is seen
        gone = (pages < 0) | (pages >= k_codes.shape[0])
        pages = torch.where(gone, 0, pages)

        def values(codes, scales):
            x = codes[pages].double() * scales[pages].double()[..., None, None]
            x[gone] = 0
            return x.transpose(0, 1).reshape(H, -1, D)[:, :length]

        k, v = values(k_codes, k_scale), values(v_codes, v_scale)
        key = torch.arange(length, device=q.device)
        for lo in range(0, n, 256):
            pos = torch.arange(length - n + lo, length - n + min(n, lo + 256), device=q.device)
            hidden = torch.zeros(len(pos), length, dtype=torch.bool, device=q.device)
            if causal:
                hidden |= key > pos[:, None]
            if window:
                hidden |= key <= pos[:, None] - window
            rows = slice(first + lo, first + lo + len(pos))
            qd = q[rows].double().view(-1, H, G, D)
            y = torch.einsum("thgd,hkd->hgtk", qd, k) * scale
            y = y.masked_fill(hidden, -math.inf)
            top = y.amax(-1, keepdim=True)
            top = torch.where(top == -math.inf, torch.zeros_like(top), top)
            p = (y - top).exp()
            total = p.sum(-1, keepdim=True)
            safe = torch.where(total == 0, torch.ones_like(total), total)
            vv = torch.nan_to_num(v, 0.0)  # a NaN value counts where it is seen, not where its weight is 0
            seen_nan = torch.isnan(v).any(-1).double() @ (~hidden).double().T > 0  # [H, t]
            total = torch.where(seen_nan[:, None, :, None], math.nan, total)
            safe = torch.where(seen_nan[:, None, :, None], math.nan, safe)
            out[rows] = torch.einsum("hgtk,hkd->thgd", p / safe, vv).reshape(-1, heads, D)
            mag[rows] = torch.einsum("hgtk,hkd->thgd", p / safe, vv.abs()).reshape(-1, heads, D)
            lse[rows] = (top + total.log())[..., 0].permute(2, 0, 1).reshape(-1, heads)
    return out, mag, lse


def fork(tables, lengths, parents, extra, n_pages, P, width):
    """Tables, lengths and copies (src, dst) of the next batch, or None where pages are short."""
    rows, out_len, copies = [], [], []
    whole, openers = set(), {}
    for i, p in enumerate(parents):
        L = lengths[p] if p >= 0 else 0
        whole.update(tables[p][: L // P] if p >= 0 else [])
        if p >= 0 and L % P:
            openers.setdefault(tables[p][L // P], i)
    kept = {page: i for page, i in openers.items() if page not in whole}
    used = whole | set(kept)
    free = iter([x for x in range(n_pages) if x not in used])
    try:
        for i, (p, e) in enumerate(zip(parents, extra)):
            L = lengths[p] if p >= 0 else 0
            row = list(tables[p][: L // P]) if p >= 0 else []
            if L % P:
                page = tables[p][L // P]
                if kept.get(page) == i:
                    row.append(page)
                else:
                    row.append(next(free))
                    copies.append((page, row[-1]))
            while len(row) < -(-(L + e) // P):
                row.append(next(free))
            rows.append(row + [-1] * (width - len(row)))
            out_len.append(L + e)
    except StopIteration:
        return None
    return rows, out_len, copies


def compact(tables, lengths, P):
    held = sorted({x for t, n in zip(tables, lengths) for x in t[: -(-n // P)]})
    U = len(held)
    move = dict(zip([x for x in held if x >= U], [x for x in range(U) if x not in set(held)]))
    rows = [[move.get(x, x) if w < -(-n // P) else -1 for w, x in enumerate(t)] for t, n in zip(tables, lengths)]
    return rows, move
