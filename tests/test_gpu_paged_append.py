"""paged_cache_append and paged_cache_gather against their definitions, bit for bit.

Scales are powers of two and roundings are to the nearest, so the stored values are exact
functions of the rows: no tolerance."""

import math

import pytest
import torch

import gemma4_fa4_amd as g4
from oracle import paged_cache as pc
from paged_testutil import DEV, as_oracle, cu_of, empty_cache, ints, random_table

pytestmark = pytest.mark.gpu


def rows(seed, total, heads, d):
    """bf16 rows over many binades, with outliers, zeros, subnormals."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(total, heads, d, generator=g)
    x *= torch.exp2(torch.randint(-6, 7, (total, heads, 1), generator=g).float())
    x[torch.rand(total, heads, generator=g) < 0.05] = 0.0
    return x.to(torch.bfloat16)


def check(cache, table, steps, seed, widen=None):
    """Append the steps (lists of new tokens per sequence), compare after each."""
    heads, d = cache.num_kv_heads, cache.head_dim
    want = as_oracle(cache)
    now = [0] * len(table)
    for i, new in enumerate(steps):
        now = [n + f for n, f in zip(now, new)]
        cu = cu_of(new)
        k, v = rows(seed + 2 * i, cu[-1] + 3, heads, d), rows(seed + 2 * i + 1, cu[-1] + 3, heads, d)
        if widen:
            k, v = widen(k), widen(v)
        g4.paged_cache_append(cache, k.to(DEV), v.to(DEV), ints(table), ints(now), ints(cu))
        for (values, scale), x in zip(want, (k, v)):
            pc.append(values, scale, x, table, now, cu)
        for (values, scale), (got, got_scale) in zip(want, as_oracle(cache)):
            assert torch.equal(torch.nan_to_num(scale, 7e7), torch.nan_to_num(got_scale, 7e7)), i
            assert torch.equal(torch.nan_to_num(values, 7e7), torch.nan_to_num(got, 7e7)), i
    return now, want


@pytest.mark.parametrize("d,heads,page", [(256, 3, 32), (512, 1, 64), (256, 1, 256), (512, 2, 128)])
def test_append_in_steps_of_any_size(d, heads, page):
    steps = [[1, 0, 33, 70], [1, 31, 1, 5], [1, 2, 64, 0], [40, 1, 3, 129]]
    lens = [sum(s[b] for s in steps) for b in range(4)]
    table, count = random_table(d + page, lens, page)
    cache = empty_cache(count, heads, page, d)
    now, want = check(cache, table, steps, 11 * d + page)
    # read back: exact, zero rows past the lengths
    ask = [n + 2 for n in now]
    k, v = g4.paged_cache_gather(cache, ints(table), ints(now), ints(cu_of(ask)), sum(ask))
    for (values, scale), got in zip(want, (k, v)):
        for b, n in enumerate(now):
            out, _ = pc.read(values, scale, table[b], n)
            at = cu_of(ask)[b]
            assert torch.equal(got[at:at + n].cpu().double(), out)
            assert not got[at + n:at + n + 2].any()


def test_gather_leaves_rows_behind_the_last_sequence():
    table, count = random_table(1, [40, 7], 32)
    cache = empty_cache(count, 2, 32, 256)
    check(cache, table, [[40, 7]], 5)
    k, v = g4.paged_cache_gather(cache, ints(table), ints([40, 7]), ints([0, 10, 17]), 30)
    assert k[17:].isnan().all() and not k[:17].isnan().any()  # (the fixture fills with NaN)
    assert v[17:].isnan().all() and not v[:17].isnan().any()


def test_hundreds_of_sequences():
    # more than 64: the wave's search for a slot's sequence takes two rounds
    new = [(7 * b) % 45 for b in range(300)]
    table, count = random_table(2, new, 32)
    cache = empty_cache(count, 1, 32, 256)
    check(cache, table, [new], 77)


def test_infinities_and_nan():
    def widen(x):
        x[1, :, 3], x[2, :, 4], x[3, :, 5] = math.inf, -math.inf, math.nan
        x[4] = math.nan  # a whole row
        return x

    table, count = random_table(3, [40], 64)
    cache = empty_cache(count, 2, 64, 512)
    check(cache, table, [[34], [6]], 91, widen)
    k, v = g4.paged_cache_gather(cache, ints(table), ints([40]), ints([0, 40]), 40)
    assert torch.isfinite(k).all() and torch.isfinite(v).all()


def test_extreme_scales():
    def widen(x):
        x[0] *= 2.0 ** 110
        x[1:5] *= 2.0 ** -100  # below the smallest scale's steps: zero
        x[33:] *= 2.0 ** -75
        return x

    table, count = random_table(4, [64], 32)
    cache = empty_cache(count, 1, 32, 256)
    check(cache, table, [[64]], 17, widen)


def test_tokens_without_a_page_are_dropped():
    # row 0: a hole, an ID past the pages, a negative one; row 1: longer than the table is wide
    cache = empty_cache(6, 2, 32, 256)
    for t in (cache.k, cache.v):
        t.view(torch.uint8).fill_(3)
    cache.k_scale.fill_(1.0), cache.v_scale.fill_(1.0)
    table = [[4, -1, 6, -2147483648], [1, 2147483647, 0, 5]]
    check(cache, table, [[128, 150]], 23)
    k, v = g4.paged_cache_gather(cache, ints(table), ints([128, 150]), ints([0, 128, 278]), 278)
    assert not k[32:128].any() and not k[256:].any() and k[:32].any()


def test_more_new_tokens_than_tokens():
    # seq_lens below the rows given: the rows before position 0 are dropped
    cache = empty_cache(2, 1, 32, 256)
    k = rows(1, 40, 1, 256).to(DEV)
    g4.paged_cache_append(cache, k, k, ints([[1, 0]]), ints([10]), ints([0, 40]))
    got, _ = g4.paged_cache_gather(cache, ints([[1, 0]]), ints([10]), ints([0, 10]), 10)
    values = torch.zeros(2, 1, 32, 256, dtype=torch.float64)
    scale = torch.ones(2, 1, 1, dtype=torch.float64)
    pc.append(values, scale, k.cpu()[30:], [[1, 0]], [10], [0, 10])
    assert torch.equal(got.cpu().double(), pc.read(values, scale, [1, 0], 10)[0])


def test_strided_rows_another_stream_and_a_graph():
    table, count = random_table(6, [100], 64)
    cache = empty_cache(count, 4, 64, 256)
    other = empty_cache(count, 4, 64, 256)
    wide = rows(3, 100, 12, 256).to(DEV)  # K and V as slices of a fused projection
    k, v = wide[:, :4], wide[:, 8:]
    tab, lens, cu = ints(table), ints([100]), ints([0, 100])
    g4.paged_cache_append(other, k.contiguous(), v.contiguous(), tab, lens, cu)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        g4.paged_cache_append(cache, k, v, tab, lens, cu)
    torch.cuda.current_stream().wait_stream(stream)
    for a, b in ((cache.k, other.k), (cache.v, other.v)):
        a, b = (g4.paged_cache_gather(c, tab, lens, cu, 100) for c in (cache, other))
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    # one token a step in a captured graph, lengths moving on the device
    lens.fill_(90)
    one = ints([0, 1])
    kt, vt = torch.zeros_like(k[:1]).contiguous(), torch.zeros_like(v[:1]).contiguous()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        lens.add_(1)
        g4.paged_cache_append(cache, kt, vt, tab, lens, one)
    lens.fill_(90)
    eager_lens = ints([90])
    for i in range(8):
        kt.copy_(4 * k[i:i + 1]), vt.copy_(4 * v[i:i + 1])
        graph.replay()
        eager_lens.add_(1)
        g4.paged_cache_append(other, kt, vt, tab, eager_lens, one)
        a, b = (g4.paged_cache_gather(c, tab, ints([98]), ints([0, 98]), 98) for c in (cache, other))
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
