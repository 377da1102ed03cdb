"""Local attention with a window and sinks (forward, backward, single tokens) against fp64.

Bounds.  The forward's are paged_testutil.check_attention's: P is rounded to bf16 before P V
and O at the end.  The backward rounds P and dS to bf16, O (in delta) and each result once,
dQ of rows with sinks behind their window twice; with half steps of 2^-8 and independent
signs over many terms the results' relative Frobenius errors stay near 2^-8 / sqrt(3) times
the square root of the number of roundings: the repository's 2e-2 bound, and its
upstream-relative rule (twice the error of a bf16 attention) element by element, hold for the
window alone and are kept here, with the bf16 attention's rounding points applied to the sink
mask."""

import numpy as np
import pytest
import torch

import gemma4_fa4_amd as g4
from g4_testutil import check_gradients, cu, qkv
from oracle import paged_cache as pc

pytestmark = pytest.mark.gpu
DEV = "cuda"


def forward_bound(q, k, v, mask):
    """(O, LSE, O's bound, LSE's bound) of one sequence and query head in fp64."""
    s = (q @ k.T).masked_fill(~mask, -torch.inf)
    z = torch.logsumexp(s, 1)
    p = torch.exp(s - z[:, None])
    o, size = p @ v, p @ v.abs()
    t = q.shape[1] * 2.0 ** -24 * (q.abs() @ k.abs().T).masked_fill(~mask, 0).amax(1)
    bound = 2.0 ** -8 * (size + o.abs()) * 1.01 + (2 * t[:, None] + 2.0 ** -20) * size
    return o, z, bound, t + 2.0 ** -20 * (1 + z.abs())


def check_forward(q, k, v, lq, lk, window, sinks, o, lse, heads=None):
    cq, ck = cu(lq).tolist(), cu(lk).tolist()
    grp = q.shape[1] // k.shape[1]
    for b in range(len(lq)):
        if lq[b] == 0:
            continue
        mask = pc.sinks_mask(lq[b], lk[b], window, sinks).to(DEV)
        for h in heads or range(q.shape[1]):
            args = (x[i:j, n].to(DEV).double() for x, i, j, n in (
                (q, cq[b], cq[b + 1], h), (k, ck[b], ck[b + 1], h // grp),
                (v, ck[b], ck[b + 1], h // grp)))
            want, z, bound, zb = forward_bound(*args, mask)
            got = o[cq[b]:cq[b + 1], h].double()
            assert ((got - want).abs() <= bound).all(), (b, h)
            assert ((lse[h, cq[b]:cq[b + 1]].double() - z).abs() <= zb).all(), (b, h)


def baseline(q, k, v, cq, ck, window, sinks, do, dlse):
    """Gradients of a plain bf16 attention: scores, P, dP and dS rounded, as a user's own code."""
    r = lambda x: x.to(torch.bfloat16).float()  # noqa: E731
    dq, dk, dv = (torch.zeros_like(t, dtype=torch.float32) for t in (q, k, v))
    grp = q.shape[1] // k.shape[1]
    for q0, q1, k0, k1 in zip(cq, cq[1:], ck, ck[1:]):
        if q0 == q1:
            continue
        mask = pc.sinks_mask(q1 - q0, k1 - k0, window, sinks).to(q.device)
        for h in range(q.shape[1]):
            n = h // grp
            qh, kh, vh, g = (t.float() for t in (q[q0:q1, h], k[k0:k1, n], v[k0:k1, n], do[q0:q1, h]))
            s = r(qh @ kh.T).masked_fill(~mask, -torch.inf)
            p = torch.softmax(s, 1)
            o = r(r(p) @ vh)
            delta = (g * o).sum(1) - dlse[h, q0:q1]
            ds = r(p * (r(g @ vh.T) - delta[:, None]))
            dq[q0:q1, h] = r(ds @ kh)
            dk[k0:k1, n] += ds.T @ qh
            dv[k0:k1, n] += r(p).T @ g
    return dq, r(dk), r(dv)


def stages(q, k, v, lq, lk, window, sinks, do, dlse, ds_budget=0):
    """Forward and backward through the library, for head counts the adapter does not take."""
    from gemma4_fa4_amd import ops

    plan = ops.make_plan(
        num_seqs=len(lq), seqlen_q=max(lq), seqlen_k=max(lk), num_q_heads=q.shape[1],
        num_kv_heads=k.shape[1], head_dim=256, window=window, cu_q=cu(lq).to(DEV),
        cu_k=cu(lk).to(DEV), total_q=sum(lq), total_k=sum(lk), ds_budget=ds_budget)
    plan.num_sinks = sinks
    o, lse = plan.forward(q, k, v)
    return (o, lse, *plan.backward(q, k, v, o, do, lse, dlse))


CASES = [  # hkv, grp, window, sinks, lq, lk
    (2, 2, 64, 4, [300], [300]),
    (1, 1, 32, 32, [257, 40, 33], [257, 40, 33]),  # the window ends in the sinks' tile
    (1, 4, 100, 7, [130, 0, 1, 64], [400, 50, 101, 64]),  # suffixes, an empty one, no far pair
    (2, 8, 64, 1, [90], [1000]),
    (1, 2, 1, 3, [70], [70]),  # a window of the query alone
    (3, 2, 40, 20, [20, 500], [45, 500]),  # fewer queries than a tile
    (2, 2, 1024, 4, [1100, 2500], [1100, 2500]),
    (16, 2, 1024, 16, [3000, 100, 1025, 1024], [3000, 100, 1025, 1024]),
]


@pytest.mark.parametrize("hkv,grp,window,sinks,lq,lk", CASES)
@pytest.mark.parametrize("ds_budget", [0, -1])
def test_against_fp64(hkv, grp, window, sinks, lq, lk, ds_budget):
    print(hkv, grp, window, sinks, lq, lk, flush=True)
    q, k, v, do, dlse = (t.to(DEV) for t in qkv(sum(lk) + sinks, sum(lq), sum(lk), hkv * grp, hkv, 256))
    o, lse, *grads = stages(q, k, v, lq, lk, window, sinks, do, dlse, ds_budget)
    check_forward(q, k, v, lq, lk, window, sinks, o, lse)
    cq, ck = cu(lq).tolist(), cu(lk).tolist()
    *_, dq, dk, dv = pc.sinks_fwd_bwd(q, k, v, cq, ck, window, sinks, do, dlse)
    base = baseline(q, k, v, cq, ck, window, sinks, do, dlse)
    check_gradients(grads, [t.cpu() for t in (dq, dk, dv)], [t.cpu() for t in base])


def test_many_sequences_of_which_few_are_longer_than_the_window():
    lk = [20, 90, 5, 64, 65, 30, 200] * 20 + [64] * 30
    q, k, v, do, dlse = (t.to(DEV) for t in qkv(77, sum(lk), sum(lk), 4, 2, 256))
    o, lse, *grads = stages(q, k, v, lk, lk, 64, 5, do, dlse)
    c = cu(lk).tolist()
    *_, dq, dk, dv = pc.sinks_fwd_bwd(q, k, v, c, c, 64, 5, do, dlse)
    base = baseline(q, k, v, c, c, 64, 5, do, dlse)
    check_gradients(grads, [t.cpu() for t in (dq, dk, dv)], [t.cpu() for t in base])


@pytest.mark.parametrize("lq,lk", [(300, 300), (50, 400)])
def test_the_library_takes_fixed_layouts(lq, lk):
    # (B, S, H, D) with strides, bitwise as the packed call on the same rows
    from gemma4_fa4_amd import ops

    b, hkv, grp, window, sinks = 3, 2, 2, 64, 6
    q, k, v, do, dlse = (t.to(DEV) for t in qkv(9, b * lq, b * lk, hkv * grp, hkv, 256))
    want = stages(q, k, v, [lq] * b, [lk] * b, window, sinks, do, dlse)
    plan = ops.make_plan(num_seqs=b, seqlen_q=lq, seqlen_k=lk, num_q_heads=hkv * grp,
                         num_kv_heads=hkv, head_dim=256, window=window)
    plan.num_sinks = sinks
    q4, k4, v4, do4 = (t.view(b, -1, t.shape[1], 256) for t in (q, k, v, do))
    k4 = torch.cat((k4, k4), 2)[:, :, :hkv]  # strided
    o, lse = plan.forward(q4, k4, v4)
    dlse4 = dlse.view(hkv * grp, b, lq).transpose(0, 1).contiguous()
    grads = plan.backward(q4, k4, v4, o, do4, lse, dlse4)
    assert torch.equal(o.flatten(0, 1), want[0])
    assert torch.equal(lse.transpose(0, 1).reshape(hkv * grp, -1), want[1])
    for x, y in zip(grads, want[2:]):
        assert torch.equal(x.flatten(0, 1), y)


def adapter(q, k, v, lq, lk, sinks):
    return g4.fa4_local_sinks_varlen_forward(
        q, k, v, cu(lq).to(DEV), cu(lk).to(DEV), max_seqlen_q=max(lq), max_seqlen_k=max(lk),
        num_sinks=sinks)


@pytest.mark.parametrize("lq,lk,sinks", [
    ([1], [3000], 4), ([1, 1, 1], [1024, 1025, 40], 1), ([3, 16], [1040, 2000], 32),
    ([17], [1500], 5), ([700], [1800], 4), ([1200, 3], [1200, 1500], 31)])
def test_the_adapter_forward(lq, lk, sinks):
    q, k, v, *_ = (t.to(DEV) for t in qkv(sum(lk), sum(lq), sum(lk), 32, 16, 256))
    o, lse = adapter(q, k, v, lq, lk, sinks)
    check_forward(q, k, v, lq, lk, 1024, sinks, o, lse, heads=[0, 1, 13, 31])


def test_no_sinks_is_the_local_adapter():
    lq = [1300, 40]
    q, k, v, do, _ = (t.to(DEV) for t in qkv(3, 1340, 1340, 32, 16, 256))
    outs = []
    for call in (lambda *a: adapter(*a, lq, lq, 0),
                 lambda *a: g4.fa4_local_varlen_forward(
                     *a, cu(lq).to(DEV), cu(lq).to(DEV), max_seqlen_q=1300, max_seqlen_k=1300)):
        args = [t.clone().requires_grad_(True) for t in (q, k, v)]
        o, lse = call(*args)
        outs.append([o, lse, *torch.autograd.grad(o, args, do)])
    for a, b in zip(*outs):
        assert torch.equal(a, b)


def test_autograd_strides_gradient_of_lse_and_repeats():
    lq = [1500, 200]
    q, k, v, do, dlse = (t.to(DEV) for t in qkv(5, 1700, 1700, 32, 16, 256))
    wide = torch.zeros(1700, 64, 256, dtype=torch.bfloat16, device=DEV)
    wide[:, :32], wide[:, 32:48], wide[:, 48:] = q, k, v
    args = [t.clone().requires_grad_(True) for t in (q, k, v)]
    o, lse = adapter(*args, lq, lq, 6)
    want = torch.autograd.grad([o, lse], args, [do, dlse])
    leaf = wide.requires_grad_(True)
    views = leaf[:, :32], leaf[:, 32:48].clone(), leaf[:, 48:]
    o2, lse2 = adapter(*views, lq, lq, 6)
    g, = torch.autograd.grad([o2, lse2], leaf, [do.transpose(0, 1).contiguous().transpose(0, 1), dlse])
    assert torch.equal(o, o2) and torch.equal(lse, lse2)
    for a, b in zip(want, (g[:, :32], g[:, 32:48], g[:, 48:])):
        assert torch.equal(a, b)
    # a broadcast gradient, and LSE's alone
    a = torch.autograd.grad(adapter(*args, lq, lq, 6)[0].sum(), args)
    b = torch.autograd.grad(adapter(*args, lq, lq, 6)[0], args, torch.ones_like(o))
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    c = torch.autograd.grad(adapter(*args, lq, lq, 6)[1], args, dlse)
    *_, dq, dk, dv = pc.sinks_fwd_bwd(q, k, v, [0, 1500, 1700], [0, 1500, 1700], 1024, 6,
                                      torch.zeros_like(do), dlse)
    for x, y in zip(c[:2], (dq, dk)):
        assert (x.double() - y).norm() <= 1e-2 * y.norm()
    assert not c[2].any()


def test_differences_along_random_directions():
    # the loss in fp64 from the forward's own formula; the gradient from the kernels
    lq = [1100]
    q, k, v, do, _ = (t.to(DEV) for t in qkv(8, 1100, 1100, 32, 16, 256))
    args = [t.clone().requires_grad_(True) for t in (q, k, v)]
    grads = torch.autograd.grad(adapter(*args, lq, lq, 8)[0], args, do)
    g = torch.Generator().manual_seed(2)
    for i, grad in enumerate(grads):
        step = torch.randn(grad.shape, generator=g).to(DEV).double()
        losses = []
        for e in (1e-4, -1e-4):
            x = [t.double() for t in (q, k, v)]
            x[i] = x[i] + e * step
            losses.append((pc.sinks_fwd_bwd(*x, [0, 1100], [0, 1100], 1024, 8)[0] * do.double()).sum())
        slope = ((losses[0] - losses[1]) / 2e-4).item()
        # bf16 gradients: each element off by 2^-8 of itself and as much of its roundings inside,
        # summed over random signs
        size = (grad.double() * step).norm().item()
        assert abs((grad.double() * step).sum().item() - slope) <= 8 * 2.0 ** -8 * size


def test_two_adapter_calls_side_by_side_on_two_streams():
    lq = [1400]
    sets = [[t.to(DEV) for t in qkv(30 + i, 1400, 1400, 32, 16, 256)] for i in range(2)]
    want = []
    for q, k, v, do, _ in sets:
        a = [t.clone().requires_grad_(True) for t in (q, k, v)]
        want.append(torch.autograd.grad(adapter(*a, lq, lq, 4)[0], a, do))
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for st, (q, k, v, do, _) in zip(streams, sets):
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            a = [t.clone().requires_grad_(True) for t in (q, k, v)]
            got.append(torch.autograd.grad(adapter(*a, lq, lq, 4)[0], a, do))
    torch.cuda.synchronize()
    for x, y in zip(want, got):
        assert all(torch.equal(a, b) for a, b in zip(x, y))


def test_a_captured_single_token_step():
    # the library call in a graph (the adapter reads cu_seqlens on the host)
    from gemma4_fa4_amd import ops

    lk = [1500, 1300]
    q, k, v, *_ = (t.to(DEV) for t in qkv(9, 2, 2800, 32, 16, 256))
    plan = ops.make_plan(num_seqs=2, seqlen_q=1, seqlen_k=1500, num_q_heads=32, num_kv_heads=16,
                         head_dim=256, window=1024, cu_q=cu([1, 1]).to(DEV), cu_k=cu(lk).to(DEV),
                         total_q=2, total_k=2800)
    plan.num_sinks = 4
    plan.forward(q, k, v)  # (launch attributes are set outside the capture)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = plan.forward(q, k, v)
    for i in range(4):
        q.copy_(qkv(50 + i, 2, 1, 32, 16, 256)[0])
        graph.replay()
        want = plan.forward(q, k, v)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    check_forward(q, k, v, [1, 1], lk, 1024, 4, *got, heads=[0, 31])


@pytest.mark.parametrize("ds_budget", [0, -1])
def test_a_captured_backward(ds_budget):
    from gemma4_fa4_amd import ops

    n = [200, 90]
    q, k, v, do, dlse = (t.to(DEV) for t in qkv(12, 290, 290, 4, 2, 256))
    plan = ops.make_plan(num_seqs=2, seqlen_q=200, seqlen_k=200, num_q_heads=4, num_kv_heads=2,
                         head_dim=256, window=64, cu_q=cu(n).to(DEV), cu_k=cu(n).to(DEV),
                         total_q=290, total_k=290, ds_budget=ds_budget)
    plan.num_sinks = 4

    def step():
        o, lse = plan.forward(q, k, v)
        return (o, lse, *plan.backward(q, k, v, o, do, lse, dlse))

    step()  # (launch attributes are set outside the capture)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for i in range(4):
        q.copy_(qkv(60 + i, 290, 1, 4, 2, 256)[0])
        graph.replay()
        want = step()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    check_forward(q, k, v, n, n, 64, 4, *got[:2])
