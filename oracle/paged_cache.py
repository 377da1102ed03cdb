"""Paged 8-bit cache, its pages and sink attention -- TEST INFRASTRUCTURE ONLY.

The operators' definitions, token by token and page by page in Python and fp64,
written for reading rather than speed.  The reference has no counterpart of them;
they are pinned by ``tests/test_oracle_paged_cache.py`` (hand-computed scales,
roundings and tables; attention against ``oracle.attention`` where the two meet;
gradients against differences).
"""

from __future__ import annotations

import math

import torch

BLOCK = 32
FLOOR = -64


def e4m3_values() -> torch.Tensor:
    """The 127 non-negative finite e4m3 values in the order of their codes."""
    out = []
    for code in range(127):
        e, m = code >> 3, code & 7
        out.append(m * 2.0 ** -9 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7))
    return torch.tensor(out, dtype=torch.float64)


def to_e4m3(x: torch.Tensor) -> torch.Tensor:
    """fp64 values to the nearest e4m3 value, ties to the even code; NaN to 0,
    anything past 448 to 448."""
    table = e4m3_values()
    a = torch.nan_to_num(x.double().abs(), nan=0.0, posinf=448.0).clamp(max=448.0)
    hi = torch.searchsorted(table, a).clamp(max=126)
    lo = (hi - 1).clamp(min=0)
    up, down = table[hi] - a, a - table[lo]
    code = torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    value = table[code]
    return torch.where(torch.isnan(x), torch.zeros_like(value), torch.copysign(value, x.double()))


def block_scale(amax: float) -> float:
    """The smallest power of two s >= 2^-64 with amax / s <= 448."""
    s = 2.0 ** FLOOR
    while amax / s > 448.0:
        s *= 2.0
    return s


def append(values, scale, rows, page_table, seq_lens, cu) -> None:
    """In place: ``values`` fp64 (pages, heads, page_size, d) e4m3 values, ``scale`` fp64
    (pages, heads, page_size / 32), ``rows`` (T, heads, d)."""
    num_pages, heads, page_size, _ = values.shape
    for b, length in enumerate(seq_lens):
        n = cu[b + 1] - cu[b]
        first = length - n
        touched = {}
        for t in range(max(first, 0), length):
            touched.setdefault(t // BLOCK, []).append(t)
        for block, tokens in touched.items():
            w = block * BLOCK // page_size
            page = page_table[b][w] if w < len(page_table[b]) else -1
            if not 0 <= page < num_pages:
                continue
            blk, r0 = block * BLOCK % page_size // BLOCK, block * BLOCK % page_size
            held = tokens[0] - block * BLOCK  # earlier tokens of the block
            for h in range(heads):
                x = torch.stack([rows[cu[b] + t - first, h].double() for t in tokens])
                fin = x[torch.isfinite(x)].abs()
                s = block_scale(fin.max().item() if fin.numel() else 0.0)
                if held:
                    old = scale[page, h, blk].item()
                    s = max(s, old)
                    values[page, h, r0:r0 + held] = to_e4m3(
                        values[page, h, r0:r0 + held] * (old / s))
                values[page, h, r0 + held:r0 + held + len(tokens)] = to_e4m3(x / s)
                scale[page, h, blk] = s


def read(values, scale, page_row, length):
    """Tokens [0, length) of one sequence, fp64 (length, heads, d), and which have a page."""
    num_pages, heads, page_size, d = values.shape
    out = torch.zeros(length, heads, d, dtype=torch.float64)
    there = torch.zeros(length, dtype=torch.bool)
    for t in range(length):
        w = t // page_size
        page = page_row[w] if w < len(page_row) else -1
        if 0 <= page < num_pages:
            at = t % page_size
            out[t] = values[page, :, at] * scale[page, :, at // BLOCK, None]
            there[t] = True
    return out, there


def sinks_mask(lq: int, lk: int, window: int, sinks: int) -> torch.Tensor:
    """(lq, lk) bool; queries are the last lq of lk positions."""
    a = torch.arange(lk - lq, lk)[:, None]
    j = torch.arange(lk)[None, :]
    ok = j <= a
    if window:
        ok &= (j > a - window) | (j < sinks)
    return ok


def masked_attention(q, k, v, mask):
    """One sequence in fp64: q (lq, hq, d), k / v (lk, hkv, d); O (lq, hq, d), LSE (hq, lq)."""
    grp = q.shape[1] // k.shape[1]
    q, k, v = q.double(), k.double(), v.double()
    s = torch.einsum("qhd,khd->hqk", q, k.repeat_interleave(grp, 1))
    s = s.masked_fill(~mask, -math.inf)
    lse = torch.logsumexp(s, -1) if k.shape[0] else torch.full(s.shape[:2], -math.inf).double()
    p = torch.exp(s - torch.where(torch.isinf(lse), 0.0, lse)[..., None])
    return torch.einsum("hqk,khd->qhd", p, v.repeat_interleave(grp, 1)), lse


def sinks_fwd_bwd(q, k, v, cu_q, cu_k, window, sinks, do=None, dlse=None):
    """Packed sink attention in fp64 with explicit gradients; lists as cumulative lengths."""
    o, lse = torch.zeros_like(q, dtype=torch.float64), torch.zeros(
        q.shape[1], q.shape[0], dtype=torch.float64, device=q.device)
    dq, dk, dv = (torch.zeros_like(t, dtype=torch.float64) for t in (q, k, v))
    grp = q.shape[1] // k.shape[1]
    for q0, q1, k0, k1 in zip(cu_q, cu_q[1:], cu_k, cu_k[1:]):
        if q1 == q0:
            continue
        mask = sinks_mask(q1 - q0, k1 - k0, window, sinks).to(q.device)
        for h in range(q.shape[1]):
            n = h // grp
            qh, kh, vh = q[q0:q1, h].double(), k[k0:k1, n].double(), v[k0:k1, n].double()
            s = (qh @ kh.T).masked_fill(~mask, -math.inf)
            z = torch.logsumexp(s, 1)
            p = torch.exp(s - z[:, None])
            o[q0:q1, h], lse[h, q0:q1] = p @ vh, z
            if do is None:
                continue
            g = do[q0:q1, h].double()
            delta = (g * o[q0:q1, h]).sum(1)
            if dlse is not None:
                delta = delta - dlse[h, q0:q1].double()
            ds = p * (g @ vh.T - delta[:, None])
            dq[q0:q1, h] = ds @ kh
            dk[k0:k1, n] += ds.T @ qh
            dv[k0:k1, n] += p.T @ g
    return o, lse, dq, dk, dv


# ---- pages: lists of lists, changed in place --------------------------------


def pages_of(length: int, page_size: int) -> int:
    return -(-length // page_size)


def _count(refs, page, by):
    if 0 <= page < len(refs):
        refs[page] += by


def fork(table, lens, refs, parents, page_size) -> None:
    old, old_lens = [list(r) for r in table], list(lens)
    width = len(table[0])
    for b, p in enumerate(parents):
        if p == b:
            continue
        for w in range(min(pages_of(old_lens[b], page_size), width)):
            _count(refs, old[b][w], -1)
        row, length = [-1] * width, 0
        if 0 <= p < len(table):
            length = old_lens[p]
            for w in range(min(pages_of(length, page_size), width)):
                row[w] = old[p][w]
                _count(refs, row[w], 1)
        table[b], lens[b] = row, length


def reserve(table, lens, refs, new_lens, page_size):
    width, n = len(table[0]), len(refs)
    at_entry = list(refs)
    free = [i for i in range(n) if at_entry[i] == 0]
    src, dst, granted = [-1] * len(table), [-1] * len(table), [1] * len(table)

    def last_page(b):
        cur = lens[b]
        if new_lens[b] <= cur or cur % page_size == 0 or pages_of(new_lens[b], page_size) > width:
            return -1
        page = table[b][cur // page_size]
        return page if 0 <= page < n and at_entry[page] > 1 else -1

    writers = {}
    for b in range(len(table)):
        if last_page(b) >= 0:
            writers.setdefault(last_page(b), []).append(b)
    asked = 0
    for b in range(len(table)):
        cur, new = lens[b], new_lens[b]
        if new <= cur:
            continue
        have, need = pages_of(cur, page_size), pages_of(new, page_size)
        if need > width:
            granted[b] = 0
            continue
        page = last_page(b)
        copy = page >= 0 and (len(writers[page]) < at_entry[page] or writers[page][0] != b)
        begin, asked = asked, asked + need - have + copy
        if asked > len(free):
            granted[b] = 0
            continue
        if copy:
            src[b], dst[b] = page, free[begin]
            table[b][cur // page_size] = dst[b]
            refs[page] -= 1
            refs[dst[b]] += 1
        for i in range(need - have):
            table[b][have + i] = free[begin + copy + i]
            refs[free[begin + copy + i]] += 1
        lens[b] = new
    return src, dst, granted


def release(table, lens, refs, keep_lens, page_size, window=0, sinks=0) -> None:
    width = len(table[0])
    for b, asked in enumerate(keep_lens):
        keep = min(lens[b], max(asked, 0))
        for w in range(min(pages_of(lens[b], page_size), width)):
            tokens = range(w * page_size, (w + 1) * page_size)
            gone = tokens[0] >= keep
            if window:
                gone |= all(t >= sinks and t <= keep - window for t in tokens)
            if gone:
                _count(refs, table[b][w], -1)
                table[b][w] = -1
        lens[b] = keep


def compact(table, refs):
    n = len(refs)
    live = sum(r > 0 for r in refs)
    move = [i for i in range(live, n) if refs[i] > 0]
    hole = [i for i in range(live) if refs[i] <= 0]
    to = dict(zip(move, hole))
    for row in table:
        for w, page in enumerate(row):
            row[w] = to.get(page, page)
    for s, d in to.items():
        refs[d], refs[s] = refs[s], 0
    pad = [-1] * (max(n // 2, 1) - len(move))
    return move + pad, hole + pad
