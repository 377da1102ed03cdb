"""paged_cache_attention against fp64 over the exact cached values, within derived bounds
(paged_testutil.check_attention)."""

import numpy as np
import pytest
import torch

import gemma4_fa4_amd as g4
from paged_testutil import DEV, check_attention, cu_of, empty_cache, filled_cache, ints, queries

pytestmark = pytest.mark.gpu


def attend(q, cache, table, lens, new, *, window=0, sinks=0, max_q=None, max_k=None):
    return g4.paged_cache_attention(
        q, cache, ints(table), ints(lens), ints(cu_of(new)), max_seqlen_q=max_q or max(new),
        max_seqlen_k=max_k or max(max(lens), 1), sliding_window=window or None, num_sinks=sinks)


def run(seed, d, hkv, grp, page, lens, new, window=0, sinks=0, **kw):
    print(seed, d, hkv, grp, page, lens[:8], new[:8], window, sinks, flush=True)
    cache, table = filled_cache(seed, lens, hkv, page, d)
    q = queries(seed, sum(new), hkv * grp, d)
    out, lse = attend(q, cache, table, lens, new, window=window, sinks=sinks, **kw)
    check_attention(q, cache, table, lens, new, out, lse, window=window, sinks=sinks)


@pytest.mark.parametrize("d,hkv,grp,page,lens,new", [
    (512, 4, 8, 64, [1], [1]),
    (512, 4, 8, 64, [33], [1]),
    (512, 4, 8, 32, [700, 31, 2049, 64], [1, 1, 1, 1]),
    (512, 1, 8, 256, [5000], [1]),
    (512, 2, 1, 128, [100, 257], [1, 1]),  # GQA 1
    (512, 1, 2, 64, [300], [8]),  # a whole group of 16 rows
    (512, 1, 4, 64, [300, 90], [7, 3]),  # two groups, the second part full
    (512, 4, 8, 64, [515, 12, 200], [5, 0, 8]),  # three groups, none, a set of four
    (512, 2, 8, 64, [4000, 33, 7], [3, 4, 1]),  # sets of two, one group of one empty
    (512, 2, 4, 32, [2000, 3, 90, 77], [16, 3, 9, 1]),
    (256, 2, 1, 64, [900, 64], [64, 20]),
    (256, 2, 8, 128, [300, 1, 40], [4, 1, 2]),
    (256, 16, 2, 64, [900], [1]),
    (256, 3, 2, 32, [130, 1, 500], [3, 1, 17]),
    (256, 2, 8, 128, [77, 40], [40, 40]),
])
def test_over_everything(d, hkv, grp, page, lens, new):
    run(d + page + sum(lens), d, hkv, grp, page, lens, new)


@pytest.mark.parametrize("window,sinks,lens,new", [
    (1024, 4, [3000], [1]),
    (1024, 0, [3000, 500, 1025], [1, 1, 1]),
    (1024, 31, [1500, 1056, 1023], [5, 1, 9]),
    (100, 32, [400, 131, 132, 133], [1, 1, 1, 1]),  # the window's first tile holds sinks too
    (33, 5, [500, 37, 38, 39, 70], [20, 1, 1, 1, 2]),
    (1, 1, [64, 2, 1], [4, 1, 1]),
    (1, 0, [64, 2, 1], [33, 2, 1]),
    (40, 32, [20, 400], [20, 300]),
])
@pytest.mark.parametrize("page", [32, 128])
def test_windows_and_sinks(window, sinks, lens, new, page):
    run(window + sinks, 256, 2, 2, page, lens, new, window, sinks)


@pytest.mark.parametrize("seed", range(24))
def test_random_batches(seed):
    rng = np.random.default_rng(1000 + seed)
    d = int(rng.choice([256, 512]))
    hkv, grp = int(rng.integers(1, 5)), int(rng.choice([1, 2, 4, 8]))
    batch = int(rng.integers(1, 12))
    top = int(rng.choice([40, 300, 2500]))
    lens = [int(x) for x in rng.integers(1, top, batch)]
    most = int(rng.choice([1, 3, 30]))
    new = [min(n, int(x)) for n, x in zip(lens, rng.integers(0, most + 1, batch))]
    new[0] = max(new[0], 1)
    window = int(rng.choice([0, 17, 64, 1024])) if d == 256 else 0
    sinks = int(rng.integers(0, 33)) if window else 0
    run(seed, d, hkv, grp, int(rng.choice([32, 64, 128, 256])), lens, new, window, sinks,
        max_q=max(new) + int(rng.integers(0, 3)), max_k=max(lens) + int(rng.integers(0, 200)))


def test_hundreds_of_sequences():
    # more than a workgroup's threads: the batch's prefix sums take several rounds
    rng = np.random.default_rng(3)
    lens = [int(x) for x in rng.integers(1, 90, 600)]
    run(5, 256, 1, 2, 32, lens, [1] * 600, 64, 3)


# Chunks: more than 448 query rows per KV head (192 at head dim 256, 320 of one or two
# sequences) are attended over bf16 rows in the workspace; shorter ones in several sets of rows.
@pytest.mark.parametrize("d,hkv,grp,page,lens,new,window,sinks", [
    (512, 4, 8, 64, [900, 9, 300], [500, 9, 0], 0, 0),
    (512, 4, 8, 64, [6000, 20], [17, 1], 0, 0),  # a prompt's end and a step in one batch
    (512, 4, 8, 64, [600, 20, 50], [16, 1, 9], 0, 0),  # two sets
    (512, 1, 1, 32, [400], [400], 0, 0),
    (256, 1, 1, 32, [400, 193], [400, 193], 100, 3),
    (512, 2, 4, 256, [2100, 700], [150, 33], 0, 0),
    (256, 16, 2, 64, [3000, 1500], [700, 33], 1024, 4),
    (256, 2, 2, 64, [3000, 1500, 40], [33, 200, 40], 1024, 0),
    (256, 2, 2, 64, [3000, 1500, 40], [33, 90, 40], 1024, 5),
    (256, 2, 8, 32, [900, 70], [200, 70], 100, 32),
    (256, 4, 2, 128, [500, 77], [60, 33], 64, 17),
    (256, 4, 2, 128, [500, 77], [97, 33], 64, 17),
    (256, 1, 4, 64, [333, 1], [40, 1], 0, 0),
])
def test_chunks(d, hkv, grp, page, lens, new, window, sinks):
    run(d + page + sum(lens), d, hkv, grp, page, lens, new, window, sinks)
    run(d + page + sum(lens), d, hkv, grp, page, lens, new, window, sinks, max_q=max(new) + 40,
        max_k=max(lens) + 100)


def test_chunks_of_hundreds_of_sequences():
    lens = [(37 * b) % 150 + 40 for b in range(300)]
    run(16, 256, 1, 8, 32, lens, [33 + b % 7 for b in range(300)], 64, 3)


def test_one_long_sequence_among_short_ones():
    run(6, 512, 2, 8, 64, [40, 20000, 7, 300], [1, 1, 1, 1])


def test_large_scores():
    # maxima that rise by far more than what the softmax absorbs without rescaling
    cache, table = filled_cache(8, [2000], 1, 64, 512, std_k=4.0)
    q = queries(8, 1, 8, 512, scale=30.0)
    out, lse = attend(q, cache, table, [2000], [1])
    check_attention(q, cache, table, [2000], [1], out, lse)


@pytest.mark.parametrize("more", [2, 100])  # read as they lie, and laid out
@pytest.mark.parametrize("d,window,sinks", [(256, 0, 0), (256, 16, 2), (512, 0, 0)])
def test_queries_that_see_nothing(d, window, sinks, more):
    # no tokens at all, and more queries than tokens: 0 and -inf
    cache, table = filled_cache(9, [3, 40], 2, 32, d)
    q = queries(9, more + 7, 8, d)
    out, lse = attend(q, cache, table, [3, 0], [more + 3, 4], window=window, sinks=sinks)
    seen = slice(more, more + 3)
    nothing = torch.ones(more + 7, dtype=torch.bool, device=DEV)
    nothing[seen] = False
    assert not out[nothing].any() and lse[:, nothing].eq(-torch.inf).all()
    check_attention(q[seen], cache, table[:1], [3], [3], out[seen], lse[:, seen], window=window,
                    sinks=sinks)


@pytest.mark.parametrize("new", [2, 45])
def test_rows_behind_the_last_sequence_stay(new):
    cache, table = filled_cache(10, [50], 2, 32, 256)
    q = queries(10, new + 4, 16, 256)
    out, lse = g4.paged_cache_attention(q, cache, ints(table), ints([50]), ints([0, new]),
                                        max_seqlen_q=new, max_seqlen_k=50)
    check_attention(q[:new], cache, table, [50], [new], out[:new], lse[:, :new])
    assert out[new:].isnan().all() and lse[:, new:].isnan().all()  # (the fixture's fill)


@pytest.mark.parametrize("new", [[2, 1], [70, 3]])
def test_what_lies_past_the_end_and_in_other_pages_is_not_seen(new):
    # NaN bytes everywhere but in the tokens: past the last row, in free pages, and in the
    # pages between the sinks and the window, which are gone from the table
    lens, window, sinks = [333, 61], 64, 3
    clean, table = filled_cache(11, lens, 2, 32, 256)
    q = queries(11, sum(new), 8, 256)
    want = attend(q, clean, table, lens, new, window=window, sinks=sinks)
    cache, _ = filled_cache(11, lens, 2, 32, 256)
    used = torch.zeros(cache.num_pages, 32, dtype=torch.bool)
    for b, n in enumerate(lens):
        for t in range(n):
            used[table[b][t // 32], t % 32] = True
    for t in range(sinks // 32 * 32 + 32, (lens[0] - new[0] - window + 1) // 32 * 32, 32):
        used[table[0][t // 32]] = False
        table[0][t // 32] = -1
    for t in (cache.k, cache.v):
        t.view(torch.uint8).masked_fill_(~used.to(DEV)[:, None, :, None], 0x7F)
    gone = ~used.any(1).to(DEV)
    for t in (cache.k_scale, cache.v_scale):
        t.masked_fill_(gone[:, None, None], float("nan"))
    got = attend(q, cache, table, lens, new, window=window, sinks=sinks)
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])


@pytest.mark.parametrize("entry", [-1, 6000, -2147483648, 2147483647])
def test_a_visible_token_without_a_page_gives_nan(entry):
    lens, new = [200, 100, 70], [1, 1, 4]
    cache, table = filled_cache(12, lens, 2, 32, 512)
    q = queries(12, 6, 4, 512)
    want, want_lse = attend(q, cache, table, lens, new)
    table[0][3] = entry
    table[2][2] = entry  # tokens 64 .. 69: seen by all four queries (positions 66 .. 69)
    got, lse = attend(q, cache, table, lens, new)
    assert got[0].isnan().all() and got[2:].isnan().all()
    assert torch.equal(got[1], want[1]) and torch.equal(lse[:, 1], want_lse[:, 1])


@pytest.mark.parametrize("d", [256, 512])
def test_a_chunk_and_a_token_without_a_page(d):
    lens, new = [200, 100], [80, 70]
    cache, table = filled_cache(17, lens, 2, 32, d)
    q = queries(17, 150, 8, d)
    want, want_lse = attend(q, cache, table, lens, new)
    table[0][4] = -1  # tokens 128 .. 159, of the chunk itself: seen from position 128 on
    got, lse = attend(q, cache, table, lens, new)
    assert torch.equal(got[:8], want[:8]) and got[8:80].isnan().all()
    assert torch.equal(got[80:], want[80:]) and torch.equal(lse[:, 80:], want_lse[:, 80:])


def test_a_captured_chunk():
    lens, new = [400, 300], [90, 60]
    cache, table = filled_cache(18, lens, 2, 64, 256)
    q = queries(18, 150, 8, 256)
    tab, ln, cu = ints(table), ints(lens), ints(cu_of(new))

    def call():
        return g4.paged_cache_attention(q, cache, tab, ln, cu, max_seqlen_q=90, max_seqlen_k=400,
                                        sliding_window=64, num_sinks=4)

    call()  # (launch attributes are set outside the capture)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    for i in range(5):
        q.copy_(queries(40 + i, 150, 8, 256))
        ln.copy_(ints([400 - 7 * i, 300 - i]))
        graph.replay()
        want = call()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    check_attention(q, cache, table, [372, 296], new, *got, window=64, sinks=4)


def test_a_table_narrower_than_the_lengths():
    cache, table = filled_cache(13, [64, 64], 1, 32, 256)
    q = queries(13, 2, 1, 256)
    out, _ = attend(q, cache, [row[:2] for row in table], [64, 97], [1, 1])
    assert torch.isfinite(out[0]).all() and out[1].isnan().all()


def test_a_cache_past_4_gib():
    # offsets past 32 bits: the sequences lie in a cache's last pages
    pages, hkv, page, d = 41000, 4, 64, 512
    cache = empty_cache(pages, hkv, page, d)
    assert cache.k.numel() > 5 << 30
    lens, new = [200, 70], [1, 1]
    table = [[pages - 1, pages - 7, pages - 2, 5], [pages - 3, 33000, -1, -1]]
    k, v = (queries(60 + i, 270, hkv, d, 20.0) for i in range(2))
    g4.paged_cache_append(cache, k, v, ints(table), ints(lens), ints(cu_of(lens)))
    q = queries(62, 2, 32, d)
    out, lse = attend(q, cache, table, lens, new)
    check_attention(q, cache, table, lens, new, out, lse)
    got, _ = g4.paged_cache_gather(cache, ints(table), ints(lens), ints(cu_of(lens)), 270)
    assert (got.float() - k.float()).abs().max() <= 2.0 ** -4 * k.float().abs().max()
    g4.copy_pages(cache, ints([pages - 1, 33000]), ints([40000, 0]))
    table[0][0], table[1][1] = 40000, 0
    again = attend(q, cache, table, lens, new)
    assert torch.equal(again[0], out) and torch.equal(again[1], lse)


@pytest.mark.parametrize("bound", [1, 300])
def test_a_batch_without_queries(bound):
    cache, table = filled_cache(21, [50, 60], 2, 32, 256)
    q = queries(21, 4, 16, 256)
    out, lse = g4.paged_cache_attention(q, cache, ints(table), ints([50, 60]), ints([0, 0, 0]),
                                        max_seqlen_q=bound, max_seqlen_k=60)
    assert out.isnan().all() and lse.isnan().all()  # (the fixture's fill: nothing is written)


def test_chunks_of_more_sequences_than_fit_at_once():
    # a generous bound of the lengths: 8 GiB hold the rows of 3 sequences of 700000 tokens
    lens, new = [300, 40, 180, 260, 90, 150, 70], [50, 40, 33, 1, 0, 60, 35]
    cache, table = filled_cache(22, lens, 4, 64, 256)
    q = queries(22, sum(new), 32, 256)
    out, lse = attend(q, cache, table, lens, new, max_k=700000)
    check_attention(q, cache, table, lens, new, out, lse)


def test_strided_queries_and_another_stream():
    lens, new = [400, 77], [1, 3]
    cache, table = filled_cache(14, lens, 2, 64, 256)
    wide = queries(14, 4, 12, 256)
    q = wide[:, 4:8]
    want = attend(q.contiguous(), cache, table, lens, new)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = attend(q, cache, table, lens, new)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_repeats_bitwise():
    lens, new = [3000, 700, 1], [1, 1, 1]
    cache, table = filled_cache(15, lens, 4, 64, 512)
    q = queries(15, 3, 32, 512)
    first = attend(q, cache, table, lens, new)
    for _ in range(3):
        again = attend(q, cache, table, lens, new)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_a_captured_decode_loop():
    """Reserve, append and attend in one graph, replayed over 44 tokens with eager work
    between; every replay against the same calls made eagerly on a second cache."""
    page, hkv, grp, d, window, sinks = 32, 2, 2, 256, 48, 4
    lens = [70, 5]
    table = torch.full((2, 6), -1, dtype=torch.int32, device=DEV)
    state = [(table.clone(), ints([0, 0]), torch.zeros(12, dtype=torch.int32, device=DEV),
              empty_cache(12, hkv, page, d)) for _ in range(2)]
    k, v = (queries(20 + i, sum(lens), hkv, d, 16.0) for i in range(2))
    for t, l, r, cache in state:
        g4.reserve_pages(t, l, r, ints(lens), page_size=page)
        g4.paged_cache_append(cache, k, v, t, l, ints(cu_of(lens)))
    one = ints([0, 1, 2])
    q, kn, vn = (torch.zeros(2, h, d, dtype=torch.bfloat16, device=DEV) for h in (hkv * grp, hkv, hkv))

    def step(t, l, r, cache, want):
        src, dst, _ = g4.reserve_pages(t, l, r, want, page_size=page)
        g4.copy_pages(cache, src, dst)
        g4.paged_cache_append(cache, kn, vn, t, l, one)
        out = g4.paged_cache_attention(q, cache, t, l, one, max_seqlen_q=1, max_seqlen_k=192,
                                       sliding_window=window, num_sinks=sinks)
        g4.release_pages(t, l, r, want, page_size=page, sliding_window=window, num_sinks=sinks)
        return out

    target = ints(lens)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        target.add_(1)
        got = step(*state[0], target)
    target.copy_(ints(lens))
    for i in range(44):
        for j, x in enumerate((q, kn, vn)):
            x.copy_(queries(100 + 3 * i + j, 2, x.shape[1], d, 16.0 if j else 1.5))
        graph.replay()
        want = step(*state[1], ints([n + i + 1 for n in lens]))
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), i
        assert torch.equal(state[0][0], state[1][0]) and torch.equal(state[0][2], state[1][2])
        # page 1 (tokens 32 .. 63) goes once 63 <= 70 + i + 1 - 48; page 0 holds the sinks
        assert (state[0][0][0, 1].item() >= 0) == (i < 40)
    assert state[0][1].tolist() == [n + 44 for n in lens]
    assert (state[0][0][0] >= 0).tolist() == [True, False, True, True, False, False]


@pytest.mark.parametrize("window", [2**31 - 1, 2**32 + 1, 400])
def test_a_window_past_every_length(window):
    """As no window, also for more new tokens than the sequence has."""
    for lens, new in (([300, 5, 60], [2, 9, 60]), ([300, 5, 60], [120, 100, 60])):
        cache, table = filled_cache(30, lens, 2, 64, 256)
        q = queries(30, sum(new), 8, 256)
        want = attend(q, cache, table, lens, new)
        got = attend(q, cache, table, lens, new, window=window)
        check_attention(q, cache, table, lens, new, *got)
        got = attend(q, cache, table, lens, new, window=window, sinks=3)
        check_attention(q, cache, table, lens, new, *got)
        assert torch.equal(torch.isneginf(got[1]), torch.isneginf(want[1]))


# Sets of 2, 3 and 4 groups of 16 rows a workgroup, each with a last one that is part full,
# steps of two tiles that end inside one and in the first, and several sets.
@pytest.mark.parametrize("hkv,grp,page,lens,new", [
    (1, 8, 32, [700, 100], [6, 2]),
    (2, 8, 64, [500], [56]),  # 448 rows, the most that are read as they lie
    (2, 8, 64, [500], [57]),
    (1, 2, 64, [300, 64], [24, 9]),
    (1, 1, 64, [200, 33], [48, 17]),
    (4, 8, 128, [3001, 70, 5], [10, 2, 5]),
    (2, 4, 256, [90000], [13]),
    (1, 8, 32, [31 + b for b in range(70)], [1 + b % 4 for b in range(70)]),
])
def test_sets_of_rows_at_head_dim_512(hkv, grp, page, lens, new):
    run(lens[0] + new[0], 512, hkv, grp, page, lens, new)
    run(lens[0] + new[0], 512, hkv, grp, page, lens, new, max_q=max(new) + 3, max_k=max(lens) + 9)


def test_large_scores_of_a_set():
    cache, table = filled_cache(31, [2000], 1, 64, 512, std_k=4.0)
    q = queries(31, 7, 8, 512, scale=30.0)
    out, lse = attend(q, cache, table, [2000], [7])
    check_attention(q, cache, table, [2000], [7], out, lse)


@pytest.mark.parametrize("new", [[1, 1], [9, 2], [40, 61]])
def test_what_lies_past_the_end_is_not_seen_at_head_dim_512(new):
    lens = [333, 61]
    clean, table = filled_cache(32, lens, 2, 32, 512)
    q = queries(32, sum(new), 8, 512)
    want = attend(q, clean, table, lens, new)
    cache, _ = filled_cache(32, lens, 2, 32, 512)
    used = torch.zeros(cache.num_pages, 32, dtype=torch.bool)
    for b, n in enumerate(lens):
        for t in range(n):
            used[table[b][t // 32], t % 32] = True
    for t in (cache.k, cache.v):
        t.view(torch.uint8).masked_fill_(~used.to(DEV)[:, None, :, None], 0x7F)
    for t in (cache.k_scale, cache.v_scale):
        t.masked_fill_(~used.any(1).to(DEV)[:, None, None], float("nan"))
    got = attend(q, cache, table, lens, new)
    assert torch.equal(want[0], got[0]) and torch.equal(want[1], got[1])


def test_a_set_and_a_token_without_a_page():
    lens, new = [200, 100], [20, 9]
    cache, table = filled_cache(33, lens, 2, 32, 512)
    q = queries(33, 29, 8, 512)
    want, want_lse = attend(q, cache, table, lens, new)
    table[0][6] = -1  # tokens 192 .. 199: seen from position 192 on, query 12 of 20
    got, lse = attend(q, cache, table, lens, new)
    assert torch.equal(got[:12], want[:12]) and got[12:20].isnan().all()
    assert torch.equal(got[20:], want[20:]) and torch.equal(lse[:, 20:], want_lse[:, 20:])


@pytest.mark.parametrize("new", [160, 161])  # 320 rows, the most that are read as they lie
def test_a_chunk_of_one_local_conversation(new):
    run(34, 256, 2, 2, 64, [3000], [new], 1024, 4)


def test_sets_with_strided_queries_a_narrow_table_and_another_stream():
    lens, new = [400, 77], [9, 3]
    cache, table = filled_cache(35, lens, 2, 64, 512)
    wide = queries(35, 12, 24, 512)
    q = wide[:, 8:24]
    want = attend(q.contiguous(), cache, table, lens, new)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = attend(q, cache, table, lens, new)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    out, _ = attend(q, cache, [row[:2] for row in table], lens, new)  # 128 tokens of 400
    assert out[:9].isnan().all() and torch.equal(out[9:], want[0][9:])


def test_sets_repeat_bitwise_in_a_graph():
    lens, new = [3000, 500], [6, 4]
    cache, table = filled_cache(36, lens, 4, 64, 512)
    q = queries(36, 10, 32, 512)
    tab, ln, cu = ints(table), ints(lens), ints(cu_of(new))

    def call():
        return g4.paged_cache_attention(q, cache, tab, ln, cu, max_seqlen_q=6, max_seqlen_k=3000)

    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    for i in range(4):
        q.copy_(queries(70 + i, 10, 32, 512))
        ln.copy_(ints([3000 - 70 * i, 500 - i]))
        graph.replay()
        want = call()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
