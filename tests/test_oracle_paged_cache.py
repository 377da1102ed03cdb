"""What pins oracle/paged_cache.py: hand-computed roundings, scales and tables, the dense
oracle where the two meet, and gradients against differences."""

import math

import pytest
import torch

from oracle import paged_cache as pc
from oracle.attention import attention_fwd_bwd


def test_e4m3_roundings_by_hand():
    x = [0.0, -0.0, 2.0 ** -9, 2.0 ** -10, 1.5 * 2.0 ** -10, 3 * 2.0 ** -10, 1.0625, 1.1875,
         -1.1875, 17.0, 19.0, 447.0, 448.0, 1e9, -math.inf, math.nan]
    want = [0.0, 0.0, 2.0 ** -9, 0.0, 2.0 ** -9, 2.0 ** -8, 1.0, 1.25, -1.25, 16.0, 20.0, 448.0,
            448.0, 448.0, -448.0, 0.0]
    got = pc.to_e4m3(torch.tensor(x, dtype=torch.float64))
    assert got.tolist() == want
    # every finite code stands for itself, and torch's type agrees on all of them
    codes = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    assert torch.equal(codes, pc.e4m3_values())
    assert torch.equal(pc.to_e4m3(-codes), -codes)
    g = torch.Generator().manual_seed(1)
    r = torch.randn(20000, generator=g) * torch.exp2(torch.randint(-12, 9, (20000,), generator=g))
    r = r.clamp(-448, 448)
    assert torch.equal(pc.to_e4m3(r.double()), r.to(torch.float8_e4m3fn).double())


def test_scales_by_hand():
    assert pc.block_scale(448.0) == 1.0
    assert pc.block_scale(450.0) == 2.0
    assert pc.block_scale(224.0) == 0.5
    assert pc.block_scale(0.0) == 2.0 ** -64
    assert pc.block_scale(1.0) == 2.0 ** -8  # 1 / 2^-8 = 256, 1 / 2^-9 = 512


def test_append_and_read_by_hand():
    values = torch.full((3, 1, 32, 2), math.nan, dtype=torch.float64)
    scale = torch.full((3, 1, 1), math.nan, dtype=torch.float64)
    rows = torch.zeros(33, 1, 2)
    rows[:, 0, 0] = 1.0
    rows[32, 0, 1] = 100.0
    table = [[2, 0]]
    pc.append(values, scale, rows[:31], table, [31], [0, 31])
    assert scale[2, 0, 0] == 2.0 ** -8 and scale[0, 0, 0].isnan()
    pc.append(values, scale, rows[31:], table, [33], [0, 2])
    out, there = pc.read(values, scale, table[0], 33)
    assert there.all()
    # 100 in a block of scale 2^-2 (400 <= 448): steps of 32 x 2^-2 = 8, a tie at 100 -> even code
    assert scale[0, 0, 0] == 0.25 and out[32, 0, 1] == 96.0
    assert out[:32, 0, 0].eq(1).all()
    # a larger row in the first block: earlier rows are rounded again, 1 stays exact
    big = torch.tensor([[[300.0, 0.0009]]])
    values2, scale2 = values.clone(), scale.clone()
    pc.append(values2, scale2, big, [[2]], [32], [0, 1])  # token 31 again
    assert scale2[2, 0, 0] == 1.0
    assert torch.equal(pc.read(values2, scale2, [2], 31)[0][:, 0, 0], torch.ones(31).double())
    assert pc.read(values2, scale2, [2], 32)[0][31, 0].tolist() == [288.0, 0.0]  # 288 | 320
    assert not pc.read(values, scale, [7, -1], 33)[1].any()


@pytest.mark.parametrize("lq,lk,window", [(5, 5, 0), (3, 40, 0), (40, 40, 16), (7, 60, 16)])
def test_masked_attention_is_the_dense_oracle_without_sinks(lq, lk, window):
    g = torch.Generator().manual_seed(3)
    q, k, v = (torch.randn(n, h, 8, generator=g) for n, h in ((lq, 4), (lk, 2), (lk, 2)))
    o, lse = pc.masked_attention(q, k, v, pc.sinks_mask(lq, lk, window, 0))
    o_ref, l_ref, *_ = attention_fwd_bwd(q, k, v, [0, lq], [0, lk], sliding_window=window or None)
    torch.testing.assert_close(o, o_ref.double())
    torch.testing.assert_close(lse, l_ref.double())


def test_sinks_mask_by_hand():
    m = pc.sinks_mask(3, 8, 2, 1).int().tolist()
    assert m == [[1, 0, 0, 0, 1, 1, 0, 0], [1, 0, 0, 0, 0, 1, 1, 0], [1, 0, 0, 0, 0, 0, 1, 1]]


def test_sinks_gradients_against_differences():
    g = torch.Generator().manual_seed(5)
    cu_q, cu_k = [0, 6, 6, 8], [0, 9, 12, 20]
    q, k, v = (torch.randn(n, h, 4, generator=g).double() for n, h in ((8, 2), (20, 1), (20, 1)))
    do, dlse = torch.randn(8, 2, 4, generator=g).double(), torch.randn(2, 8, generator=g).double()

    def loss(q, k, v):
        o, lse, *_ = pc.sinks_fwd_bwd(q, k, v, cu_q, cu_k, 3, 2)
        return ((o * do).sum() + (lse * dlse).sum()).item()

    o, lse, *grads = pc.sinks_fwd_bwd(q, k, v, cu_q, cu_k, 3, 2, do, dlse)
    args = [q, k, v]
    for i, grad in enumerate(grads):
        for at in [(0, 0, 0), (5, 0, 1), (7, 0, 3)]:
            moved = []
            for step in (1e-5, -1e-5):
                x = [t.clone() for t in args]
                x[i][at] += step
                moved.append(loss(*x))
            assert abs((moved[0] - moved[1]) / 2e-5 - grad[at].item()) < 1e-8


def test_pages_by_hand():
    table, lens, refs = [[3, 5, -1], [1, -1, -1], [-1, -1, -1]], [40, 20, 0], [0, 1, 0, 1, 0, 1, 0]
    pc.fork(table, lens, refs, [0, 0, 0], 32)
    assert table == [[3, 5, -1]] * 3 and lens == [40] * 3 and refs == [0, 0, 0, 3, 0, 3, 0]
    # all three write into page 5: the first keeps it, the others copy; row 2 needs a third page
    src, dst, ok = pc.reserve(table, lens, refs, [41, 41, 70], 32)
    assert (src, dst, ok) == ([-1, 5, 5], [-1, 0, 1], [1, 1, 1])
    assert table == [[3, 5, -1], [3, 0, -1], [3, 1, 2]] and lens == [41, 41, 70]
    assert refs == [1, 1, 1, 3, 0, 1, 0]
    # two pages left: row 0 asks for one, row 2 for more columns than there are, row 1 for none
    assert pc.reserve(table, lens, refs, [65, 41, 100], 32)[2] == [1, 1, 0]
    assert table[0] == [3, 5, 4] and lens == [65, 41, 70]
    # a window of 7: behind token 41 tokens 0 .. 34 have passed, behind token 70 0 .. 63
    pc.release(table, lens, refs, [0, 41, 70], 32, window=7, sinks=0)
    assert table == [[-1, -1, -1], [-1, 0, -1], [-1, -1, 2]] and lens == [0, 41, 70]
    assert refs == [1, 0, 1, 0, 0, 0, 0]
    assert pc.compact(table, refs) == ([2, -1, -1], [1, -1, -1])
    assert table == [[-1, -1, -1], [-1, 0, -1], [-1, -1, 1]] and refs == [1, 1, 0, 0, 0, 0, 0]


def test_one_sharer_that_does_not_grow_makes_all_writers_copy():
    table, lens, refs = [[0, -1], [0, -1], [0, -1]], [5, 5, 5], [3, 0, 0]
    src, dst, ok = pc.reserve(table, lens, refs, [6, 5, 6], 32)
    assert (src, dst, ok) == ([0, -1, 0], [1, -1, 2], [1, 1, 1]) and refs == [1, 1, 1]
