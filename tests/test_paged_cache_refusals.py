"""Refusals of the paged cache's calls, on the CPU: each wrong argument is named before a launch."""

import ctypes

import pytest
import torch

import gemma4_fa4_amd as g4
from gemma4_fa4_amd import _lib
from gemma4_fa4_amd import paged_cache as pcm

E4M3 = torch.float8_e4m3fn


def tensors(pages=4, heads=2, page=64, d=256):
    z = dict(dtype=torch.uint8)
    return [torch.zeros(pages, heads, page, d, **z).view(E4M3),
            torch.zeros(pages, heads, page, d, **z).view(E4M3),
            torch.ones(pages, heads, page // 32), torch.ones(pages, heads, page // 32)]


@pytest.fixture
def cache(monkeypatch):
    monkeypatch.setattr(pcm, "_require_gfx950", lambda device: None)
    return g4.PagedKVCache(*tensors())


def test_a_cpu_cache_is_refused():
    with pytest.raises(g4.UnsupportedMI355XPath, match="GPU tensors"):
        g4.PagedKVCache(*tensors())


@pytest.mark.parametrize("change,error,match", [
    (lambda t: t.__setitem__(0, t[0].view(torch.uint8)), ValueError, "float8_e4m3fn"),
    (lambda t: t.__setitem__(1, t[1][0]), ValueError, "rank-4"),
    (lambda t: t.__setitem__(1, t[1][:2]), ValueError, "same shape"),
    (lambda t: t.__setitem__(1, t[0]), ValueError, "distinct"),
    (lambda t: t.__setitem__(2, t[2].double()), ValueError, "k_scale"),
    (lambda t: t.__setitem__(3, t[3][:, :, :1]), ValueError, "v_scale"),
])
def test_cache_tensors(change, error, match, monkeypatch):
    monkeypatch.setattr(pcm, "_require_gfx950", lambda device: None)
    t = tensors()
    change(t)
    with pytest.raises(error, match=match):
        g4.PagedKVCache(*t)


@pytest.mark.parametrize("page,d", [(16, 256), (48, 256), (512, 256), (64, 128)])
def test_page_sizes_and_head_dims(page, d, monkeypatch):
    monkeypatch.setattr(pcm, "_require_gfx950", lambda device: None)
    with pytest.raises(g4.UnsupportedMI355XPath, match="page sizes"):
        g4.PagedKVCache(*tensors(page=page, d=d))


def test_non_contiguous_pages(monkeypatch):
    monkeypatch.setattr(pcm, "_require_gfx950", lambda device: None)
    t = tensors(pages=8)
    with pytest.raises(ValueError, match="contiguous"):
        g4.PagedKVCache(t[0][::2], t[1][::2], t[2][::2], t[3][::2])


def append_args():
    k = torch.zeros(5, 2, 256, dtype=torch.bfloat16)
    i = dict(dtype=torch.int32)
    return dict(k=k, v=k.clone(), page_table=torch.zeros(3, 4, **i), seq_lens=torch.zeros(3, **i),
                cu_seqlens=torch.zeros(4, **i))


@pytest.mark.parametrize("name,value,error,match", [
    ("k", torch.zeros(5, 2, 256), ValueError, "BF16"),
    ("k", torch.zeros(5, 1, 256, dtype=torch.bfloat16), ValueError, "heads and head dim"),
    ("v", torch.zeros(4, 2, 256, dtype=torch.bfloat16), ValueError, "heads and head dim"),
    ("v", torch.zeros(5, 2, 512, dtype=torch.bfloat16)[..., ::2], ValueError, "unit last"),
    ("k", torch.zeros(5, 2, 257, dtype=torch.bfloat16)[..., :256], ValueError, "16-byte"),
    ("k", torch.zeros(5, 2, 256, dtype=torch.bfloat16, requires_grad=True),
     g4.UnsupportedMI355XPath, "autograd"),
    ("page_table", torch.zeros(3, 4, dtype=torch.int64), ValueError, "page_table"),
    ("page_table", torch.zeros(12, dtype=torch.int32), ValueError, "rank-2"),
    ("page_table", torch.zeros(3, 0, dtype=torch.int32), ValueError, "rank-2"),
    ("page_table", torch.zeros(4, 3, dtype=torch.int32).t(), ValueError, "contiguous"),
    ("seq_lens", torch.zeros(2, dtype=torch.int32), ValueError, "seq_lens"),
    ("cu_seqlens", torch.zeros(3, dtype=torch.int32), ValueError, "cu_seqlens"),
])
def test_append_arguments(cache, name, value, error, match):
    args = append_args() | {name: value}
    with pytest.raises(error, match=match):
        g4.paged_cache_append(cache, **args)


def test_gather_arguments(cache):
    a = append_args()
    for total in (-1, 2.0, True):
        with pytest.raises(ValueError, match="total"):
            g4.paged_cache_gather(cache, a["page_table"], a["seq_lens"], a["cu_seqlens"], total)
    with pytest.raises(ValueError, match="cu_seqlens"):
        g4.paged_cache_gather(cache, a["page_table"], a["seq_lens"], a["seq_lens"], 1)


def library_args(**change):
    """Descriptors for calls that must return before they touch the device."""
    t = torch.zeros(64, dtype=torch.uint8).data_ptr()
    t += -t % 16
    c = dict(k=t, v=t, k_scale=t, v_scale=t, num_pages=4, num_kv_heads=2, head_dim=256, page_size=64)
    p = dict(pages=t, seq_lens=t, batch=3, width=4)
    for name, value in change.items():
        (c if name in c else p)[name] = value
    return _lib.G4PagedCache(**c), _lib.G4PageTable(**p), t


@pytest.mark.parametrize("change,rc", [
    (dict(head_dim=128), _lib.G4_ERR_UNSUPPORTED), (dict(page_size=48), _lib.G4_ERR_UNSUPPORTED),
    (dict(num_pages=0), _lib.G4_ERR_INVALID), (dict(num_kv_heads=0), _lib.G4_ERR_INVALID),
    (dict(k=None), _lib.G4_ERR_INVALID), (dict(k_scale=None), _lib.G4_ERR_INVALID),
    (dict(batch=0), _lib.G4_ERR_INVALID), (dict(width=0), _lib.G4_ERR_INVALID),
    (dict(pages=None), _lib.G4_ERR_INVALID), (dict(seq_lens=None), _lib.G4_ERR_INVALID),
])
def test_the_library_refuses(change, rc):
    lib = _lib.load()
    cache, table, t = library_args(**change)
    lay = _lib.G4Layout(0, 512, 256)
    args = [ctypes.byref(cache), ctypes.byref(table), t, 5, t, lay, t, lay, None]
    assert lib.g4_cache_append(*args) == rc and lib.g4_last_error()
    assert lib.g4_cache_gather(*args) == rc


def test_the_library_refuses_operands():
    lib = _lib.load()
    cache, table, t = library_args()
    good, bad = _lib.G4Layout(0, 512, 256), _lib.G4Layout(0, 512, 4)
    for call in (lib.g4_cache_append, lib.g4_cache_gather):
        head = [ctypes.byref(cache), ctypes.byref(table)]
        assert call(*head, None, 5, t, good, t, good, None) == _lib.G4_ERR_INVALID
        assert call(*head, t, -1, t, good, t, good, None) == _lib.G4_ERR_INVALID
        assert call(*head, t, 5, t + 8, good, t, good, None) == _lib.G4_ERR_INVALID
        assert call(*head, t, 5, t, good, t, bad, None) == _lib.G4_ERR_INVALID
        assert call(*head, t, 0, None, good, None, good, None) == _lib.G4_OK  # nothing to do


def pool_args():
    i = dict(dtype=torch.int32)
    return dict(page_table=torch.zeros(3, 4, **i), seq_lens=torch.zeros(3, **i),
                ref_counts=torch.zeros(6, **i))


ROWS = {g4.fork_pages: "parents", g4.reserve_pages: "new_lens", g4.release_pages: "keep_lens"}


@pytest.mark.parametrize("call", list(ROWS), ids=lambda c: c.__name__)
@pytest.mark.parametrize("name,value,error,match", [
    ("page_table", torch.zeros(3, 4), ValueError, "page_table"),
    ("seq_lens", torch.zeros(4, dtype=torch.int32), ValueError, "seq_lens"),
    ("ref_counts", torch.zeros(6, dtype=torch.int64), ValueError, "ref_counts"),
    ("ref_counts", torch.zeros(0, dtype=torch.int32), ValueError, "ref_counts"),
    ("rows", torch.zeros(2, dtype=torch.int32), ValueError, "must be an INT32 tensor"),
    ("page_size", 48, g4.UnsupportedMI355XPath, "page_size"),
    (None, None, g4.UnsupportedMI355XPath, "GPU tensors"),
])
def test_pool_arguments(call, name, value, error, match):
    args = pool_args() | {"rows": torch.zeros(3, dtype=torch.int32), "page_size": 64}
    if name:
        args[name] = value
    args[ROWS[call]] = args.pop("rows")
    with pytest.raises(error, match=match):
        call(**args)


def test_pool_tensors_may_not_be_one():
    a = pool_args()
    with pytest.raises(ValueError, match="distinct"):
        g4.reserve_pages(**a, new_lens=a["seq_lens"], page_size=64)


def test_release_window_compact_and_copy_arguments(cache):
    a = pool_args()
    keep = torch.zeros(3, dtype=torch.int32)
    for bad in (dict(sliding_window=0), dict(num_sinks=-1)):
        with pytest.raises(ValueError):
            g4.release_pages(**a, keep_lens=keep, page_size=64, **bad)
    with pytest.raises(ValueError, match="ref_counts"):
        g4.compact_pages(a["page_table"], a["ref_counts"].long())
    with pytest.raises(g4.UnsupportedMI355XPath, match="GPU tensors"):
        g4.compact_pages(a["page_table"][:1].contiguous(), a["ref_counts"])
    i = torch.zeros(3, dtype=torch.int32)
    for src, dst in ((i.long(), i), (i, i[:2]), (i[None], i)):
        with pytest.raises(ValueError, match="src|dst"):
            g4.copy_pages(cache, src, dst)


def test_the_library_refuses_pool_calls():
    lib = _lib.load()
    _, table, t = library_args()
    t += -t % 256
    assert lib.g4_pages_workspace_bytes(0, 1, 1) == 0 and lib.g4_last_error()
    need = lib.g4_pages_workspace_bytes(6, 3, 4)
    assert need >= 3 * 6 * 4
    ref = ctypes.byref(table)
    assert lib.g4_pages_fork(ref, t, 6, 64, t, t, need - 1, None) == _lib.G4_ERR_WORKSPACE
    assert lib.g4_pages_fork(ref, t, 6, 64, t, t + 4, need, None) == _lib.G4_ERR_WORKSPACE
    assert lib.g4_pages_fork(ref, t, 6, 64, None, t, need, None) == _lib.G4_ERR_INVALID
    assert lib.g4_pages_fork(ref, None, 6, 64, t, t, need, None) == _lib.G4_ERR_INVALID
    assert lib.g4_pages_reserve(ref, t, 6, 64, t, None, t, t, t, need, None) == _lib.G4_ERR_INVALID
    assert lib.g4_pages_reserve(ref, t, 6, 40, t, t, t, t, t, need, None) == _lib.G4_ERR_UNSUPPORTED
    assert lib.g4_pages_release(ref, t, 6, 64, t, -1, 0, None) == _lib.G4_ERR_INVALID
    assert lib.g4_pages_compact(ref, t, 0, t, t, t, need, None) == _lib.G4_ERR_INVALID
    cache, _, _ = library_args()
    assert lib.g4_pages_copy(ctypes.byref(cache), t, t, -1, None) == _lib.G4_ERR_INVALID
    assert lib.g4_pages_copy(ctypes.byref(cache), None, t, 1, None) == _lib.G4_ERR_INVALID
    assert lib.g4_pages_copy(ctypes.byref(cache), None, None, 0, None) == _lib.G4_OK


def attention_args(d=256, heads=4):
    i = dict(dtype=torch.int32)
    return dict(q=torch.zeros(5, heads, d, dtype=torch.bfloat16), page_table=torch.zeros(3, 4, **i),
                seq_lens=torch.zeros(3, **i), cu_seqlens_q=torch.zeros(4, **i),
                max_seqlen_q=2, max_seqlen_k=100)


@pytest.mark.parametrize("change,error,match", [
    (dict(q=torch.zeros(5, 4, 256)), ValueError, "BF16"),
    (dict(q=torch.zeros(5, 4, 512, dtype=torch.bfloat16)), ValueError, "head dim"),
    (dict(q=torch.zeros(5, 3, 256, dtype=torch.bfloat16)), ValueError, "multiple"),
    (dict(q=torch.zeros(5, 6, 256, dtype=torch.bfloat16)), g4.UnsupportedMI355XPath, "GQA"),
    (dict(q=torch.zeros(5, 4, 256, dtype=torch.bfloat16, requires_grad=True)),
     g4.UnsupportedMI355XPath, "autograd"),
    (dict(q=torch.zeros(5, 4, 512, dtype=torch.bfloat16)[..., ::2]), ValueError, "unit last"),
    (dict(max_seqlen_q=0), ValueError, "max_seqlen"),
    (dict(max_seqlen_k=(1 << 30) + 1), ValueError, "max_seqlen"),
    (dict(max_seqlen_k=True), TypeError, "integers"),
    (dict(max_seqlen_q=torch.tensor(2)), TypeError, "integers"),
    (dict(sliding_window=0), ValueError, "sliding_window"),
    (dict(num_sinks=4), ValueError, "needs a sliding_window"),
    (dict(sliding_window=64, num_sinks=33), g4.UnsupportedMI355XPath, "num_sinks"),
    (dict(sliding_window=64, num_sinks=-1), g4.UnsupportedMI355XPath, "num_sinks"),
    (dict(cu_seqlens_q=torch.zeros(3, dtype=torch.int32)), ValueError, "cu_seqlens_q"),
    (dict(seq_lens=torch.zeros(3)), ValueError, "seq_lens"),
])
def test_attention_arguments(cache, change, error, match):
    args = attention_args() | change
    with pytest.raises(error, match=match):
        g4.paged_cache_attention(args.pop("q"), cache, **args)


def test_attention_of_head_dim_512_takes_no_window(monkeypatch):
    monkeypatch.setattr(pcm, "_require_gfx950", lambda device: None)
    cache = g4.PagedKVCache(*tensors(d=512))
    args = attention_args(d=512)
    with pytest.raises(g4.UnsupportedMI355XPath, match="512"):
        g4.paged_cache_attention(args.pop("q"), cache, **args, sliding_window=64)


def test_the_library_refuses_attention():
    lib = _lib.load()
    cache, table, t = library_args()
    t += -t % 256
    lay = _lib.G4Layout(0, 1024, 256)

    def call(rows=5, ws=None, nbytes=None, q=t, lse=t, **change):
        p = _lib.G4CacheAttn(cache, table, t, rows, 4, 2, 100, 0, 0)
        for name, value in change.items():
            setattr(p, name, value)
        need = lib.g4_cache_attn_workspace_bytes(ctypes.byref(p))
        return lib.g4_cache_attn_fwd(ctypes.byref(p), q, lay, t, lay, lse, t if ws is None else ws,
                                     need if nbytes is None else nbytes, None)

    assert call(num_q_heads=3) == _lib.G4_ERR_INVALID
    assert call(num_q_heads=32) == _lib.G4_ERR_UNSUPPORTED
    assert call(max_seqlen_q=0) == _lib.G4_ERR_INVALID
    assert call(max_seqlen_k=-1) == _lib.G4_ERR_INVALID
    assert call(window=-1) == _lib.G4_ERR_INVALID
    assert call(num_sinks=2) == _lib.G4_ERR_INVALID
    assert call(window=64, num_sinks=33) == _lib.G4_ERR_UNSUPPORTED
    assert call(cu_seqlens_q=None) == _lib.G4_ERR_INVALID
    assert call(q=t + 8) == _lib.G4_ERR_INVALID
    assert call(lse=None) == _lib.G4_ERR_INVALID
    assert call(nbytes=255) == _lib.G4_ERR_WORKSPACE
    assert call(ws=t + 16) == _lib.G4_ERR_WORKSPACE
    assert call(rows=0, q=None, lse=None) == _lib.G4_OK


def test_a_cache_whose_tensors_share_memory(monkeypatch):
    monkeypatch.setattr(pcm, "_require_gfx950", lambda device: None)
    k, v, ks, vs = tensors()
    with pytest.raises(ValueError, match="memory in common"):
        g4.PagedKVCache(k, v, ks, ks)
    pool = torch.zeros(7, 2, 64, 256, dtype=torch.uint8).view(E4M3)
    with pytest.raises(ValueError, match="memory in common"):
        g4.PagedKVCache(pool[:4], pool[3:], ks, vs)
    pool = torch.zeros(2, 4, 2, 64, 256, dtype=torch.uint8).view(E4M3)
    assert g4.PagedKVCache(pool[0], pool[1], ks, vs).num_pages == 4  # two parts of one tensor


def test_a_cache_whose_memory_changes(cache):
    old = cache.descriptor()
    assert cache.descriptor() is old
    cache.k, cache.v, cache.k_scale, cache.v_scale = tensors(pages=9, d=512)
    assert cache.descriptor().num_pages == 9 and cache.descriptor().k == cache.k.data_ptr()
    cache.v = tensors()[1]
    with pytest.raises(ValueError, match="same shape"):
        g4.paged_cache_append(cache, **append_args())
    with pytest.raises(ValueError, match="same shape"):
        g4.copy_pages(cache, *torch.zeros(2, 3, dtype=torch.int32))


@pytest.mark.parametrize("window", [64.0, True, torch.tensor(64)])
def test_windows_and_sinks_are_integers(cache, window):
    args = attention_args()
    with pytest.raises(TypeError, match="sliding_window"):
        g4.paged_cache_attention(args["q"], cache, **{k: v for k, v in args.items() if k != "q"},
                                 sliding_window=window)
    with pytest.raises(TypeError, match="num_sinks"):
        g4.paged_cache_attention(args["q"], cache, **{k: v for k, v in args.items() if k != "q"},
                                 sliding_window=64, num_sinks=window)
    pool = pool_args() | dict(keep_lens=torch.zeros(3, dtype=torch.int32), page_size=64)
    with pytest.raises(TypeError, match="sliding_window"):
        g4.release_pages(**pool, sliding_window=window)
    with pytest.raises(TypeError, match="num_sinks"):
        g4.release_pages(**pool, sliding_window=64, num_sinks=window)


def test_a_window_past_32_bits_is_not_cut_to_its_low_ones():
    assert pcm._window(2**32 + 1) == pcm._window(2**31 - 1) == 2**31 - 1
    assert pcm._window(None) == 0 and pcm._window(5) == 5


def test_tables_pools_and_lists_past_32_bits():
    i = dict(dtype=torch.int32, device="meta")
    pool = dict(page_table=torch.zeros(3, 4, **i), seq_lens=torch.zeros(3, **i),
                ref_counts=torch.zeros(6, **i))
    with pytest.raises(g4.UnsupportedMI355XPath, match="2\\^31"):
        pcm._table(torch.zeros(2**16, 2**15, **i), None, torch.device("meta"))
    from gemma4_fa4_amd import cache_pages

    with pytest.raises(g4.UnsupportedMI355XPath, match="2\\^31"):
        cache_pages._pool(pool["page_table"], None, torch.zeros(2**31, **i))
