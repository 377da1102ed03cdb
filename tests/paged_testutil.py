"""Paged caches for the tests: random tables, and the cache's tensors as the oracle sees them."""

from __future__ import annotations

import numpy as np
import torch

import gemma4_fa4_amd as g4

DEV = "cuda"
E4M3 = torch.float8_e4m3fn


def ints(values, device=DEV):
    return torch.tensor(values, dtype=torch.int32, device=device)


def cu_of(lengths):
    return [0, *np.cumsum(lengths).tolist()]


def random_table(seed, lens, page, *, spare_pages=3, spare_width=1):
    """A page table of random distinct pages (-1 past each row's end) and the pages' number."""
    rng = np.random.default_rng(seed)
    used = [-(-n // page) for n in lens]
    count = sum(used) + spare_pages
    ids = rng.permutation(count)
    table = np.full((len(lens), max(max(used) + spare_width, 1)), -1, np.int32)
    at = 0
    for b, n in enumerate(used):
        table[b, :n] = ids[at:at + n]
        at += n
    return table.tolist(), count


def empty_cache(pages, heads, page, d):
    return g4.PagedKVCache.empty(pages, num_kv_heads=heads, head_dim=d, page_size=page, device=DEV)


def as_oracle(cache):
    """fp64 CPU (values, scales) of K and of V."""
    return [(t.cpu().double(), s.cpu().double())
            for t, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale))]


def filled_cache(seed, lens, heads, page, d, *, std_k=1.0, std_v=1.0, **kw):
    """A cache that holds random rows for `lens` tokens, its table, and the fp32 rows' sizes."""
    table, count = random_table(seed, lens, page, **kw)
    cache = empty_cache(count, heads, page, d)
    g = torch.Generator().manual_seed(seed)
    total = sum(lens)
    k = (torch.randn(total, heads, d, generator=g) * std_k).to(torch.bfloat16).to(DEV)
    v = (torch.randn(total, heads, d, generator=g) * std_v).to(torch.bfloat16).to(DEV)
    g4.paged_cache_append(cache, k, v, ints(table), ints(lens), ints(cu_of(lens)))
    return cache, table


def check_attention(q, cache, table, lens, new, out, lse, *, window=0, sinks=0):
    """O and LSE against fp64 on the exact cached values, within derived bounds.

    O: P is rounded to bf16 (2^-8 of each weight: 2^-8 sum p |v|) and O itself (2^-8 |O|);
    the rest is fp32: scores off by at most d 2^-24 sum |q k| (t below), so weights by that
    and about 2^-21 of exp2, twice (numerator and sum).  LSE: t, and 2^-20 (1 + |LSE|) for
    exp2, the sum and log2.
    """
    from oracle.paged_cache import sinks_mask

    cu_k, cu_q = cu_of(lens), cu_of(new)
    k, v = g4.paged_cache_gather(cache, ints(table), ints(lens), ints(cu_k), cu_k[-1])
    hkv, d = cache.num_kv_heads, cache.head_dim
    grp = q.shape[1] // hkv
    assert lse.dtype == torch.float32 and out.dtype == torch.bfloat16
    for b, (n, f) in enumerate(zip(lens, new)):
        if f == 0:
            continue
        mask = sinks_mask(f, n, window, sinks).to(DEV)
        for h in range(hkv):
            qb = q[cu_q[b]:cu_q[b + 1], h * grp:(h + 1) * grp].double().transpose(0, 1)
            kb, vb = (x[cu_k[b]:cu_k[b + 1], h].double() for x in (k, v))
            s = (qb @ kb.T).masked_fill(~mask, -torch.inf)
            z = torch.logsumexp(s, -1) if n else torch.full(s.shape[:2], -torch.inf, device=DEV,
                                                            dtype=torch.float64)
            p = torch.exp(s - torch.where(torch.isinf(z), 0.0, z)[..., None])
            o = p @ vb
            size = p @ vb.abs()
            t = d * 2.0 ** -24 * (qb.abs() @ kb.abs().T).masked_fill(~mask, 0).amax(-1) \
                if n else torch.zeros_like(z)
            got = out[cu_q[b]:cu_q[b + 1], h * grp:(h + 1) * grp].double().transpose(0, 1)
            bound = 2.0 ** -8 * (size + o.abs()) * 1.01 + (2 * t[..., None] + 2.0 ** -20) * size
            assert torch.isfinite(got).all(), (b, h)
            worst = ((got - o).abs() - bound).max().item()
            assert worst <= 1e-30, (b, h, worst)
            gl = lse[h * grp:(h + 1) * grp, cu_q[b]:cu_q[b + 1]].double()
            seen = ~torch.isinf(z)
            assert torch.equal(torch.isinf(gl), ~seen)
            worst = ((gl - z).abs() - t - 2.0 ** -20 * (1 + z.abs()))[seen]
            assert worst.numel() == 0 or worst.max().item() <= 0, (b, h, worst.max().item())


def queries(seed, total, heads, d, scale=1.5):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(total, heads, d, generator=g) * scale * d ** -0.5).to(torch.bfloat16).to(DEV)
