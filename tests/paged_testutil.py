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
