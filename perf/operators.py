"""The serving cache's operators and sink attention, as timed cases.

Four kinds of work, each over the range that programs on one MI355X meet:

* ``attend``: attention of new tokens over a paged cache held in 8 bits (e4m3), with one
  power-of-two scale for each block of 32 tokens and KV head: decode steps, drafted tokens to
  verify, chunks of a prompt; sliding layers with a window and a few first tokens that stay
  visible (sinks), global layers over everything;
* ``append``: the new tokens' K and V rounded into the cache's pages;
* ``pages``: the pages' tables and reference counts: conversations forked and grown with copies
  of shared pages, passed pages released, live pages moved to the front;
* ``sinks``: bf16 attention with a sliding window and sinks, packed: single tokens, and forward
  and backward of training batches.

Where ``own`` is false ``run`` computes the same in plain torch operations.  Lengths and tables
follow from a case's own ``shape`` number, values from the seed given to ``prepare``.
"""

import math
import os
import sys

import numpy as np
import torch

own = False

DEVICE = "cuda"
WINDOW = 1024  # sliding layers
Q_HEADS = 32
KV_HEADS = {"local": 16, "global": 4}
HEAD_DIM = {"local": 256, "global": 512}
BLOCK = 32  # tokens that share a scale
TOP = 448.0  # largest e4m3 value
FLOOR = -64  # exponent of the smallest scale
E4M3 = torch.float8_e4m3fn


def listed():
    return [
        # One conversation on a sliding layer, past its window: the smallest call, 50 of a
        # generated token's 60 layers.  The pages between the sinks and the window are gone.
        {"name": "attend_local_1", "kind": "attend", "layer": "local", "batch": 1, "cache": 2500,
         "new": 1, "sinks": 4, "page": 64, "shape": 0},
        # A serving step on a global layer: 16 conversations of 4K to 8K tokens.
        {"name": "attend_global_16", "kind": "attend", "layer": "global", "batch": 16,
         "cache": 8192, "new": 1, "sinks": 0, "page": 64, "shape": 1},
        # Two long documents being answered on a global layer.
        {"name": "attend_global_100k", "kind": "attend", "layer": "global", "batch": 2,
         "cache": 100000, "new": 1, "sinks": 0, "page": 128, "shape": 2},
        # Up to five drafted tokens of eight conversations verified on a sliding layer.
        {"name": "attend_verify_8", "kind": "attend", "layer": "local", "batch": 8, "cache": 4000,
         "new": 5, "sinks": 4, "page": 32, "shape": 3},
        # A 500-token message appended to a 12K conversation (chunked prefill), global layer.
        {"name": "attend_500_after_12k", "kind": "attend", "layer": "global", "batch": 1,
         "cache": 12500, "new": 500, "sinks": 0, "page": 64, "shape": 4},
        # The new token of 64 conversations stored, global layer.
        {"name": "append_step_64", "kind": "append", "layer": "global", "batch": 64,
         "cache": 700, "new": 1, "page": 64, "shape": 5},
        # Prompts of up to 6000 tokens stored behind earlier turns, sliding layer.
        {"name": "append_prompts", "kind": "append", "layer": "local", "batch": 4,
         "cache": 7000, "new": 6000, "page": 64, "shape": 6},
        # A beam search step over 24 beams: rows replaced by their parents, one page each made
        # their own again for the next token.
        {"name": "pages_beam_24", "kind": "pages", "way": "fork", "layer": "global", "batch": 24,
         "width": 130, "pages": 1500, "page": 64, "shape": 7},
        # A large pool after a quarter of its conversations ended: released, moved together.
        {"name": "pages_compact", "kind": "pages", "way": "compact", "layer": "local",
         "batch": 256, "width": 64, "pages": 16000, "page": 32, "shape": 8},
        # A single token of eight conversations over a bf16 cache, sliding layer with sinks.
        {"name": "sinks_step_8", "kind": "sinks", "batch": 8, "cache": 4000, "new": 1, "sinks": 4,
         "train": False, "shape": 9},
        # Fine-tuning on one sample of 2500 tokens, sliding layer with sinks.
        {"name": "sinks_train_2500", "kind": "sinks", "batch": 1, "cache": 2500, "new": 2500,
         "sinks": 4, "train": True, "shape": 10},
        # A packed training batch of 32K tokens.
        {"name": "sinks_train_32k", "kind": "sinks", "batch": 6, "cache": 32768, "new": 32768,
         "sinks": 16, "train": True, "shape": 11},
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "append", "pages", "sinks"])
    layer = rng.choice(["local", "global"])
    page = rng.choice([32, 64, 128, 256])
    shape = rng.randrange(1 << 30)
    if kind == "attend":
        way = rng.choice(["step", "step", "verify", "chunk"])
        new = 1 if way == "step" else rng.randint(2, 16) if way == "verify" else \
            _log_uniform(rng, 17, 1500)
        batch = _log_uniform(rng, 1, 2 if way == "chunk" else 64)
        most = 12000 if way == "chunk" else 200000 // batch
        return {"kind": kind, "layer": layer, "batch": batch, "cache": new + _log_uniform(rng, 1, most),
                "new": new, "sinks": rng.choice([0, 1, 4, 31]) if layer == "local" else 0,
                "page": page, "shape": shape}
    if kind == "append":
        batch = _log_uniform(rng, 1, 128)
        new = 1 if rng.random() < 0.4 else _log_uniform(rng, 2, 16000 // batch)
        return {"kind": kind, "layer": layer, "batch": batch, "cache": new + rng.randint(0, 500),
                "new": new, "page": page, "shape": shape}
    if kind == "pages":
        batch = _log_uniform(rng, 2, 256)
        width = rng.randint(4, max(4, min(200, 12000 // batch)))
        return {"kind": kind, "way": rng.choice(["fork", "compact"]), "layer": layer,
                "batch": batch, "width": width, "page": rng.choice([32, 64]),
                "pages": batch * (width + 2) + rng.randint(1, 2000), "shape": shape}
    if rng.random() < 0.4:
        batch = _log_uniform(rng, 1, 64)
        return {"kind": kind, "batch": batch, "cache": _log_uniform(rng, 40, 100000 // batch),
                "new": rng.randint(1, 4), "sinks": rng.randint(1, 32), "train": False,
                "shape": shape}
    tokens = _log_uniform(rng, 100, 30000)
    return {"kind": kind, "batch": _log_uniform(rng, 1, max(1, tokens // 1000)), "cache": tokens,
            "new": tokens, "sinks": rng.randint(1, 32), "train": True, "shape": shape}


# ---------------------------------------------------------------------------
# geometry of a case
# ---------------------------------------------------------------------------


def _lengths(case):
    """Tokens of every sequence, the new ones among them, and how many are new."""
    rng = np.random.default_rng(case["shape"])
    n, top, new = case["batch"], case["cache"], case["new"]
    if case["kind"] == "sinks" and case["train"]:  # `cache` tokens in all
        if n == 1:
            return [top], [top]
        shares = rng.uniform(0.1, 1.0, n)
        lengths = np.maximum(1, np.floor(shares / shares.sum() * top)).astype(int)
        lengths[int(np.argmax(lengths))] += top - int(lengths.sum())
        return [int(x) for x in lengths], [int(x) for x in lengths]
    lengths = [top] + [int(x) for x in rng.integers(max(1, top // 2), top + 1, n - 1)]
    fresh = [new] + [int(x) for x in rng.integers(max(1, new // 2), new + 1, n - 1)]
    return lengths, [min(f, x) for f, x in zip(fresh, lengths)]


def _window(case):
    return WINDOW if case["kind"] == "sinks" or case["layer"] == "local" else 0


def _visible(case):
    """(allowed (query, key) pairs of one head, keys that any query sees)."""
    window, sinks, pairs, keys = _window(case), case["sinks"], 0, 0
    for length, new in zip(*_lengths(case)):
        at = np.arange(length - new, length, dtype=np.int64)
        if window:
            far = np.maximum(at + 1 - window, 0)  # keys behind the window
            pairs += int((at + 1 - far + np.minimum(far, sinks)).sum())
            keys += length - int(far[0]) + min(int(far[0]), sinks)
        else:
            pairs += int((at + 1).sum())
            keys += length
    return pairs, keys


def work(case):
    if case["kind"] == "pages":
        h, d, page = KV_HEADS[case["layer"]], HEAD_DIM[case["layer"]], case["page"]
        moved = case["batch"] if case["way"] == "fork" else _compact_moves(case)
        tables = case["batch"] * case["width"] * 4 * (4 if case["way"] == "fork" else 3)
        one = 2 * h * (page * d + page // BLOCK * 4)
        return {"bytes": tables + 2 * 4 * case["pages"] + 2 * moved * one, "flops": 0}
    lengths, new = _lengths(case)
    layer = case.get("layer", "local")
    h, d = KV_HEADS[layer], HEAD_DIM[layer]
    rows = sum(new)
    if case["kind"] == "append":
        old = sum((n - f) % BLOCK for n, f in zip(lengths, new))  # rounded again at worst
        blocks = sum(-(-n // BLOCK) - (n - f) // BLOCK for n, f in zip(lengths, new))
        return {"bytes": 2 * h * (rows * d * 3 + min(old, rows) * d + blocks * 4), "flops": 0}
    pairs, keys = _visible(case)
    forward = 4.0 * Q_HEADS * pairs * d
    qo, lse = rows * Q_HEADS * d * 2, rows * Q_HEADS * 4
    if case["kind"] == "attend":
        return {"bytes": 2 * qo + lse + 2 * keys * h * (d + 4 / BLOCK), "flops": forward}
    kv = keys * h * d * 2
    if not case["train"]:
        return {"bytes": 2 * qo + lse + 2 * kv, "flops": forward}
    return {"bytes": 4 * qo + lse + 4 * kv, "flops": 3.5 * forward}


# ---------------------------------------------------------------------------
# what a program has in hand
# ---------------------------------------------------------------------------


class _Values:
    def __init__(self, seed):
        self.g = torch.Generator(device=DEVICE).manual_seed(seed)

    def normal(self, *shape, std=1.0):
        return torch.randn(*shape, generator=self.g, device=DEVICE).mul_(std)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _cu(lengths):
    return _ints([0, *np.cumsum(lengths).tolist()])


def _scale(amax):
    """The smallest power of two s with amax / s <= 448, at least 2^-64."""
    m, e = torch.frexp(amax)  # amax = m 2^e, m in [0.5, 1)
    return torch.ldexp(torch.ones_like(amax), (e - 9 + (m > 0.875).int()).clamp_min(FLOOR))


def _filled(r, pages, h, page, d, std):
    """Pages of random rows in 8 bits, and their blocks' scales."""
    x = r.normal(pages, h, page // BLOCK, BLOCK, d, std=std)
    s = _scale(x.abs().amax((-1, -2)))
    return (x / s[..., None, None]).to(E4M3).view(pages, h, page, d), s


def _cache(case, r, lengths, fresh, spare=1):
    """Pages in random order; those that no query sees any more are gone from the table."""
    page, h, d = case["page"], KV_HEADS[case["layer"]], HEAD_DIM[case["layer"]]
    rng = np.random.default_rng(case["shape"] + 1)
    table = np.full((len(lengths), max(-(-n // page) for n in lengths) + spare), -1, np.int32)
    for b, (n, f) in enumerate(zip(lengths, fresh)):
        at = np.arange(-(-n // page))
        passed = (at * page >= case.get("sinks", 0)) & ((at + 1) * page <= n - f - WINDOW + 1)
        at = at[~passed] if case["kind"] == "attend" and case["layer"] == "local" else at
        table[b, at] = 0
    count = int((table == 0).sum())
    table[table == 0] = rng.permutation(count)
    st = {"page_table": torch.from_numpy(table).to(DEVICE), "seq_lens": _ints(lengths),
          "cu": _cu(fresh)}
    st["k"], st["k_scale"] = _filled(r, count, h, page, d, 1.0)
    st["v"], st["v_scale"] = _filled(r, count, h, page, d, 0.5)
    return st


def _compact_moves(case):
    table, ends, _ = _pool(case)
    live = np.unique(table[~ends][table[~ends] >= 0])
    return int((live >= live.size).sum())


def _pool(case):
    """A pool in use: rows of random lengths on random pages, which rows end, lengths."""
    rng = np.random.default_rng(case["shape"] + 1)
    b, w, page = case["batch"], case["width"], case["page"]
    lens = rng.integers(1, (w - 1) * page, b)
    used = -(-lens // page)
    table = np.full((b, w), -1, np.int32)
    ids = rng.permutation(case["pages"])[: int(used.sum())]
    table[np.arange(w)[None, :] < used[:, None]] = ids
    return table, rng.random(b) < 0.25, lens


def prepare(case, seed):
    r = _Values(seed)
    if case["kind"] == "pages":
        table, ends, lens = _pool(case)
        h, d, page, n = KV_HEADS[case["layer"]], HEAD_DIM[case["layer"]], case["page"], case["pages"]
        refs = np.zeros(n, np.int32)
        refs[table[table >= 0]] = 1
        st = {"page_table": torch.from_numpy(table).to(DEVICE), "seq_lens": _ints(lens.tolist()),
              "ref_counts": torch.from_numpy(refs).to(DEVICE)}
        rng = np.random.default_rng([case["shape"], seed])
        if case["way"] == "fork":  # the beams' parents of this step
            st["parents"] = _ints(rng.integers(0, case["batch"], case["batch"]).tolist())
        else:
            st["keep_lens"] = _ints(np.where(ends, 0, lens).tolist())
        for name in ("k", "v"):  # any finite values
            raw = torch.randint(0, 252, (n, h, page, d), generator=r.g, device=DEVICE,
                                dtype=torch.uint8)
            st[name] = raw.add_((raw >= 126) * 2).view(E4M3)
        st["k_scale"] = torch.ldexp(torch.ones(n, h, page // BLOCK, device=DEVICE),
                                    torch.randint(-9, -3, (n, h, page // BLOCK), generator=r.g,
                                                  device=DEVICE, dtype=torch.int32))
        st["v_scale"] = st["k_scale"] * 0.5
        return {"case": case, **st}
    lengths, fresh = _lengths(case)
    layer = case.get("layer", "local")
    h, d = KV_HEADS[layer], HEAD_DIM[layer]
    st = {"case": case, "max_q": max(fresh), "max_k": max(lengths)}
    if case["kind"] == "append":
        st |= _cache(case, r, lengths, fresh)
        # (some tokens larger than what their block holds, as outlying tokens are)
        st["new_k"], st["new_v"] = (
            (r.normal(sum(fresh), h, d, std=std) * (1 + 3 * (r.normal(sum(fresh), 1, 1) > 1)))
            .to(torch.bfloat16) for std in (1.0, 0.5))
        return st
    st["q"] = r.normal(sum(fresh), Q_HEADS, d, std=1.5 / math.sqrt(d)).to(torch.bfloat16)
    if case["kind"] == "attend":
        return st | _cache(case, r, lengths, fresh)
    st["k"] = r.normal(sum(lengths), h, d).to(torch.bfloat16)
    st["v"] = r.normal(sum(lengths), h, d).to(torch.bfloat16)
    st["cu_q"], st["cu_k"] = _cu(fresh), _cu(lengths)
    if case["train"]:
        st["dout"] = r.normal(sum(fresh), Q_HEADS, d).to(torch.bfloat16)
        for name in ("q", "k", "v"):
            st[name].requires_grad_(True)
    return st


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------


def _package():
    path = os.path.join(os.getcwd(), "gemma4-fa4-kernels_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import gemma4_fa4_amd

    return gemma4_fa4_amd


def _handle(g4, st):
    if "handle" not in st:  # a program keeps its cache's handle
        st["handle"] = g4.PagedKVCache(st["k"], st["v"], st["k_scale"], st["v_scale"])
    return st["handle"]


def run(st):
    kind = st["case"]["kind"]
    if kind == "attend":
        return _run_attend(st)
    if kind == "append":
        return _run_append(st)
    if kind == "pages":
        return _run_fork(st) if st["case"]["way"] == "fork" else _run_compact(st)
    return _run_sinks(st)


def _run_attend(st):
    case = st["case"]
    window = _window(case)
    if own:
        g4 = _package()
        out, lse = g4.paged_cache_attention(
            st["q"], _handle(g4, st), st["page_table"], st["seq_lens"], st["cu"],
            max_seqlen_q=st["max_q"], max_seqlen_k=st["max_k"],
            sliding_window=window or None, num_sinks=case["sinks"])
    else:
        out, lse = _plain_attend(st, window, case["sinks"])
    return {"out": out, "lse": lse}


def _plain_attend(st, window, sinks):
    q, table, cu, lens = st["q"], st["page_table"], st["cu"].long(), st["seq_lens"].long()
    b, w = table.shape
    _, h, page, d = st["k"].shape
    grp, most, total = Q_HEADS // h, st["max_q"], q.shape[0]
    # the sequences' rows side by side
    at = torch.arange(most, device=DEVICE)
    new = cu[1:] - cu[:-1]
    rows = (cu[:-1, None] + at).clamp_max(total - 1)
    qs = q[rows].float().view(b, most, h, grp, d).permute(0, 2, 3, 1, 4).reshape(b, h, grp * most, d)
    # the pages that the batch has, in 32 bits
    ids = table.clamp_min(0).long()
    keys = w * page

    def read(x, s):
        x = x.view(torch.uint8)[ids].view(E4M3).float().view(b, w, h, page // BLOCK, BLOCK, d)
        x = x * s[ids][..., None, None]
        return x.view(b, w, h, page, d).permute(0, 2, 1, 3, 4).reshape(b, h, keys, d)

    scores = torch.matmul(qs, read(st["k"], st["k_scale"]).transpose(-1, -2))
    j = torch.arange(keys, device=DEVICE)
    a = (lens - new)[:, None] + at  # the queries' places
    ok = j <= a[..., None]
    if window:
        ok &= (j > a[..., None] - window) | (j < sinks)
    ok &= (table >= 0).repeat_interleave(page, 1)[:, None, :]
    scores = scores.view(b, h * grp, most, keys).masked_fill_(~ok[:, None], -math.inf)
    top = scores.amax(-1, keepdim=True).clamp_min(-1e30)
    p = scores.sub_(top).exp_()
    total_p = p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(b, h, grp * most, keys), read(st["v"], st["v_scale"]))
    out = out.view(b, h * grp, most, d) / total_p.clamp_min(1e-30)
    lse = (total_p.log() + top)[..., 0]
    # back to packed rows
    row = torch.arange(total, device=DEVICE)
    seq = torch.bucketize(row, cu[1:], right=True)
    i = row - cu[seq]
    return out[seq, :, i].to(torch.bfloat16), lse[seq, :, i].t().contiguous()


def _run_append(st):
    if own:
        g4 = _package()
        g4.paged_cache_append(_handle(g4, st), st["new_k"], st["new_v"], st["page_table"],
                              st["seq_lens"], st["cu"])
    else:
        _plain_append(st, "k")
        _plain_append(st, "v")
    return {name: st[name] for name in ("k", "v", "k_scale", "v_scale")}


def _plain_append(st, name):
    x, cache, scale = st["new_" + name], st[name], st[name + "_scale"]
    table, cu, lens = st["page_table"].long(), st["cu"].long(), st["seq_lens"].long()
    n, h, page, d = cache.shape
    per = page // BLOCK
    raw = cache.view(torch.uint8).view(n, h, per, BLOCK, d)
    row = torch.arange(x.shape[0], device=DEVICE)
    seq = torch.bucketize(row, cu[1:], right=True)
    first = lens - (cu[1:] - cu[:-1])  # the first new token's place
    at = first[seq] + row - cu[seq]
    pg, blk, slot = table[seq, at // page], at % page // BLOCK, at % BLOCK
    x = x.float()
    amax = torch.zeros(n * per, h, device=DEVICE).scatter_reduce(
        0, (pg * per + blk)[:, None].expand(-1, h), x.abs().amax(-1), "amax")
    fresh = _scale(amax).view(n, per, h).transpose(1, 2)
    # a sequence's first block may hold earlier tokens: the larger scale, and they rounded again
    hp, hb, kept = table[torch.arange(len(lens), device=DEVICE), first // page], \
        first % page // BLOCK, first % BLOCK
    old = scale[hp, :, hb]
    now = torch.where((kept > 0)[:, None], torch.maximum(fresh[hp, :, hb], old), fresh[hp, :, hb])
    was = raw[hp, :, hb]
    again = (was.view(E4M3).float() * (old / now)[..., None, None]).to(E4M3).view(torch.uint8)
    earlier = torch.arange(BLOCK, device=DEVICE)[None, :] < kept[:, None]
    raw[hp, :, hb] = torch.where(earlier[:, None, :, None], again, was)
    fresh[hp, :, hb] = now
    scale[pg, :, blk] = fresh[pg, :, blk]
    raw[pg, :, blk, slot] = (x / fresh[pg, :, blk][..., None]).to(E4M3).view(torch.uint8)


def _run_fork(st):
    """Every beam takes its parent's row, and is made ready for one more token."""
    page = st["case"]["page"]
    # (the calls change tables and counts in place: each pass starts from copies)
    table, lens, refs = st["page_table"].clone(), st["seq_lens"].clone(), st["ref_counts"].clone()
    if own:
        g4 = _package()
        cache = _handle(g4, st)
        g4.fork_pages(table, lens, refs, st["parents"], page_size=page)
        src, dst, granted = g4.reserve_pages(table, lens, refs, lens + 1, page_size=page)
        g4.copy_pages(cache, src, dst)
        granted = granted.bool()
    else:
        _plain_fork(table, lens, refs, st["parents"].long(), page)
        src, dst, granted = _plain_reserve(table, lens, refs, lens + 1, page)
        _plain_copy(st, src, dst)
    return {"page_table": table, "seq_lens": lens, "ref_counts": refs, "src": src, "dst": dst,
            "granted": granted, "k": st["k"], "v": st["v"], "k_scale": st["k_scale"],
            "v_scale": st["v_scale"]}


def _counted(refs, ids, by):
    refs.index_add_(0, ids.clamp_min(0).long().view(-1), (by * (ids >= 0)).int().view(-1))


def _plain_fork(table, lens, refs, parents, page):
    b, w = table.shape
    at = torch.arange(w, device=DEVICE)
    own_row = (parents == torch.arange(b, device=DEVICE))[:, None]
    used = at < (lens[:, None] + page - 1) // page
    new_table, new_lens = table[parents], lens[parents]
    new_used = at < (new_lens[:, None] + page - 1) // page
    _counted(refs, torch.where(used & ~own_row, table, -1), -1)
    _counted(refs, torch.where(new_used & ~own_row, new_table, -1), 1)
    table.copy_(torch.where(own_row, table, torch.where(new_used, new_table, -1)))
    lens.copy_(new_lens)


def _plain_reserve(table, lens, refs, new_lens, page):
    b, w = table.shape
    n = refs.shape[0]
    rows, at = torch.arange(b, device=DEVICE), torch.arange(w, device=DEVICE)
    free = refs == 0
    rank = torch.cumsum(free, 0) - 1
    found = torch.zeros(n + 1, dtype=torch.int32, device=DEVICE)
    found.scatter_(0, torch.where(free, rank, n), torch.arange(n, dtype=torch.int32, device=DEVICE))
    have, need = (lens + page - 1) // page, (new_lens + page - 1) // page
    grows = (new_lens > lens) & (need <= w)
    last = table[rows, ((lens - 1).clamp_min(0) // page).long()]
    # a shared page that a row writes into becomes its own copy, but for the first such row
    # where nobody else has the page
    held = last.clamp_min(0).long()
    part = grows & (lens % page != 0) & (last >= 0) & (refs[held] > 1)
    writers = torch.zeros_like(refs).index_add_(0, held, part.int())
    first = torch.full_like(refs, b).scatter_reduce(
        0, held, torch.where(part, rows, b).int(), "amin")
    shared = part & ((writers[held] < refs[held]) | (rows > first[held]))
    asked = torch.where(grows, need - have, 0) + shared.int()
    end = torch.cumsum(asked, 0)
    begin = end - asked
    granted = (need <= w) & (end <= free.sum())
    own_copy = shared & granted
    dst = torch.where(own_copy, found[begin.long().clamp_max(n)], -1)
    src = torch.where(own_copy, last, -1)
    k = begin[:, None] + shared[:, None].int() + at - have[:, None]
    fresh = (granted & grows)[:, None] & (at >= have[:, None]) & (at < need[:, None])
    table.copy_(torch.where(fresh, found[k.long().clamp(0, n)], table))
    column = at == ((lens - 1).clamp_min(0) // page)[:, None]
    table.copy_(torch.where(column & own_copy[:, None], dst[:, None], table))
    _counted(refs, torch.where(fresh, table, -1), 1)
    _counted(refs, dst, 1)
    _counted(refs, src, -1)
    lens.copy_(torch.where(granted & grows, new_lens, lens))
    return src, dst, granted


def _plain_copy(st, src, dst):
    # (a pair that is none copies page 0 onto itself: nothing moves page 0 in the same call)
    ok = dst >= 0
    f, t = torch.where(ok, src, 0).long(), torch.where(ok, dst, 0).long()
    for name in ("k", "v", "k_scale", "v_scale"):
        x = st[name].view(torch.uint8) if name in ("k", "v") else st[name]
        x.index_copy_(0, t, x[torch.where(t == 0, 0 * f + _origin(f, t), f)])


def _origin(f, t):
    """What page 0 takes: the pair that writes it, if there is one, else itself."""
    return torch.where((t == 0) & (f > 0), f, 0).amax()


def _run_compact(st):
    """The pages of ended conversations given back, the live ones moved to the front."""
    page = st["case"]["page"]
    # (tables and counts are changed in place, and the pages' moves with them: each pass starts
    # from copies of all that it changes)
    table, lens, refs = st["page_table"].clone(), st["seq_lens"].clone(), st["ref_counts"].clone()
    if own:
        g4 = _package()
        cache = _handle(g4, st)
        g4.release_pages(table, lens, refs, st["keep_lens"], page_size=page)
        src, dst = g4.compact_pages(table, refs)
        g4.copy_pages(cache, src, dst)
    else:
        _plain_release(table, lens, refs, st["keep_lens"], page)
        src, dst = _plain_compact(table, refs)
        _plain_copy(st, src, dst)
    return {"page_table": table, "seq_lens": lens, "ref_counts": refs, "src": src, "dst": dst,
            "k": st["k"], "v": st["v"], "k_scale": st["k_scale"], "v_scale": st["v_scale"]}


def _plain_release(table, lens, refs, keep, page):
    at = torch.arange(table.shape[1], device=DEVICE)
    used = at < (lens[:, None] + page - 1) // page
    gone = used & (at >= (keep[:, None] + page - 1) // page)
    _counted(refs, torch.where(gone, table, -1), -1)
    table.masked_fill_(gone, -1)
    lens.copy_(torch.minimum(lens, keep))


def _plain_compact(table, refs):
    n = refs.shape[0]
    ids = torch.arange(n, dtype=torch.int32, device=DEVICE)
    live = refs > 0
    count = live.sum()
    move, hole = live & (ids >= count), ~live & (ids < count)
    most = max(n // 2, 1)
    src = torch.full((most + 1,), -1, dtype=torch.int32, device=DEVICE)
    dst = src.clone()
    src.scatter_(0, torch.where(move, torch.cumsum(move, 0) - 1, most), torch.where(move, ids, -1))
    dst.scatter_(0, torch.where(hole, torch.cumsum(hole, 0) - 1, most), torch.where(hole, ids, -1))
    src, dst = src[:most], dst[:most]
    to = torch.cat((ids, ids[:1]))
    to.scatter_(0, torch.where(src >= 0, src, n).long(), torch.where(src >= 0, dst, 0))
    table.copy_(torch.where(table >= 0, to[table.clamp_min(0).long()], table))
    refs.copy_(torch.zeros_like(refs).scatter_add_(0, to[:n].long(), torch.where(live, refs, 0)))
    return src, dst


def _run_sinks(st):
    case = st["case"]
    if own:
        out, lse = _package().fa4_local_sinks_varlen_forward(
            st["q"], st["k"], st["v"], st["cu_q"], st["cu_k"], max_seqlen_q=st["max_q"],
            max_seqlen_k=st["max_k"], num_sinks=case["sinks"])
    else:
        out, lse = _plain_sinks(st, case["sinks"])
    if not case["train"]:
        return {"out": out, "lse": lse}
    dq, dk, dv = torch.autograd.grad(out, (st["q"], st["k"], st["v"]), st["dout"])
    return {"out": out.detach(), "lse": lse.detach(), "dq": dq, "dk": dk, "dv": dv}


def _plain_sinks(st, sinks):
    """Blocks of queries against the keys that their window reaches, and the sinks."""
    q, k, v, cu_q, cu_k = st["q"], st["k"], st["v"], st["cu_q"].long(), st["cu_k"].long()
    total, hq, d = q.shape
    h, b = k.shape[1], cu_q.shape[0] - 1
    grp = hq // h
    rows = min(WINDOW, st["max_q"])
    per = -(-st["max_q"] // rows)  # blocks of a sequence
    seq = torch.arange(b, device=DEVICE).repeat_interleave(per)
    start = torch.arange(per, device=DEVICE).repeat(b) * rows
    lq, lk = (cu_q[1:] - cu_q[:-1])[seq], (cu_k[1:] - cu_k[:-1])[seq]
    if per > 1:  # (the blocks that exist: `max_q` and the batch are the host's)
        most = total // rows + b
        keep = torch.argsort((start >= lq).int(), stable=True)[:most]
        seq, start, lq, lk = seq[keep], start[keep], lq[keep], lk[keep]
    i = start[:, None] + torch.arange(rows, device=DEVICE)
    a = i + (lk - lq)[:, None]
    near = min(WINDOW + rows, st["max_k"])
    j = torch.cat((torch.arange(sinks, device=DEVICE).expand(len(seq), -1),
                   (a[:, :1] + rows - near).clamp_min(0) + torch.arange(near, device=DEVICE)), 1)
    first = torch.cat((torch.ones(sinks, dtype=torch.bool, device=DEVICE),
                       torch.zeros(near, dtype=torch.bool, device=DEVICE)))
    far = j[:, None, :] <= a[..., None] - WINDOW
    ok = (j[:, None, :] <= a[..., None]) & (far == first) & (j < lk[:, None])[:, None, :]
    qi = (cu_q[seq][:, None] + i).clamp_max(total - 1)
    ki = (cu_k[seq][:, None] + j).clamp_max(k.shape[0] - 1)
    qs = q.float()[qi].view(-1, rows, h, grp, d).permute(0, 2, 3, 1, 4).reshape(-1, h, grp * rows, d)
    ks, vs = (x.float()[ki].permute(0, 2, 1, 3).contiguous() for x in (k, v))
    s = torch.matmul(qs, ks.transpose(-1, -2)).view(-1, h, grp, rows, j.shape[1])
    s = s.masked_fill(~ok[:, None, None], -math.inf)
    top = s.detach().amax(-1, keepdim=True).clamp_min(-1e30)
    p = (s - top).exp()
    sums = p.sum(-1, keepdim=True).clamp_min(1e-30)
    o = torch.matmul((p / sums).view(-1, h, grp * rows, j.shape[1]), vs)
    o = o.view(-1, h, grp, rows, d).permute(0, 3, 1, 2, 4).reshape(-1, hq, d)
    lse = (sums.log() + top)[..., 0].permute(0, 3, 1, 2).reshape(-1, hq)
    # back to packed rows
    row = torch.arange(total, device=DEVICE)
    there = torch.full((total + 1,), 0, device=DEVICE).scatter(
        0, torch.where(i < lq[:, None], cu_q[seq][:, None] + i, total).view(-1),
        torch.arange(i.numel(), device=DEVICE))
    return o[there[row]].to(torch.bfloat16), lse[there[row]].t().contiguous()


# ---------------------------------------------------------------------------
# the same from the definitions, in 64 bits
# ---------------------------------------------------------------------------


def exact(case, seed):
    if case["kind"] == "pages":
        return None  # whole numbers and copied bytes
    st = prepare(case, seed)
    if case["kind"] == "append":
        return _exact_append(st)
    if case["kind"] == "attend":
        return _exact_attend(st)
    return _exact_sinks(st)


def _exact_append(st):
    """Block by block: scales from the largest value, rows to the nearest e4m3 value."""
    cu, lens = st["cu"].tolist(), st["seq_lens"].tolist()
    if sum(-(-n // BLOCK) for n in lens) > 3000:
        return None

    def nearest(x):
        step = torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -6))) - 3)
        return torch.round(x / step) * step

    got = {}
    for name in ("k", "v"):
        cache, scale = st[name].double(), st[name + "_scale"].double()
        page = cache.shape[2]
        for b, n in enumerate(lens):
            x = st["new_" + name][cu[b]:cu[b + 1]].double()
            first = n - x.shape[0]
            for t0 in range(first // BLOCK * BLOCK, n, BLOCK):
                lo, hi = max(first, t0), min(n, t0 + BLOCK)
                pg, blk = int(st["page_table"][b, t0 // page]), t0 % page // BLOCK
                rows = x[lo - first:hi - first].transpose(0, 1)  # (heads, rows, d)
                e = torch.ceil(torch.log2(rows.abs().amax((1, 2)) / TOP)).clamp_min(FLOOR)
                s = torch.exp2(e)
                if lo > t0:
                    s = torch.maximum(s, scale[pg, :, blk])
                    held = cache[pg, :, t0 % page:t0 % page + lo - t0]
                    held.copy_(nearest(held * (scale[pg, :, blk] / s)[:, None, None]))
                cache[pg, :, lo % page:lo % page + hi - lo] = nearest(rows / s[:, None, None])
                scale[pg, :, blk] = s
        got[name], got[name + "_scale"] = cache, scale
    return {name: got[name] for name in ("k", "v", "k_scale", "v_scale")}


def _exact_attend(st):
    case = st["case"]
    pairs, _ = _visible(case)
    if pairs * Q_HEADS * HEAD_DIM[case["layer"]] > 4e13:
        return None
    window, sinks = _window(case), case["sinks"]
    cu, lens, table = st["cu"].tolist(), st["seq_lens"].tolist(), st["page_table"].tolist()
    page, h = case["page"], KV_HEADS[case["layer"]]
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device=DEVICE)
    lse = torch.full((Q_HEADS, st["q"].shape[0]), -math.inf, dtype=torch.float64, device=DEVICE)
    for b, n in enumerate(lens):
        used = [(w, p) for w, p in enumerate(table[b][: -(-n // page)]) if p >= 0]
        at = torch.tensor([w for w, _ in used], device=DEVICE)
        j = (at[:, None] * page + torch.arange(page, device=DEVICE)).view(-1)
        ids = torch.tensor([p for _, p in used], device=DEVICE)
        i = torch.arange(n - (cu[b + 1] - cu[b]), n, device=DEVICE)[:, None]
        ok = (j <= i) & (j < n)
        if window:
            ok = ok & ((i - j < window) | (j < sinks))
        for head in range(h):
            k, v = (x[:, head].view(torch.uint8)[ids].view(E4M3).double().view(len(used), -1, BLOCK, x.shape[-1])
                    * s[:, head][ids].double()[..., None, None]
                    for x, s in ((st["k"], st["k_scale"]), (st["v"], st["v_scale"])))
            k, v = k.reshape(len(j), -1), v.reshape(len(j), -1)
            for g in range(Q_HEADS // h):
                m = head * (Q_HEADS // h) + g
                s = (st["q"][cu[b]:cu[b + 1], m].double() @ k.t()).masked_fill(~ok, -math.inf)
                z = torch.logsumexp(s, 1)
                out[cu[b]:cu[b + 1], m] = torch.exp(s - z[:, None]) @ v
                lse[m, cu[b]:cu[b + 1]] = z
    return {"out": out, "lse": lse}


def _exact_sinks(st):
    case = st["case"]
    if max(_lengths(case)[0]) > 16000 and case["train"]:
        return None
    cu_q, cu_k, sinks = st["cu_q"].tolist(), st["cu_k"].tolist(), case["sinks"]
    q, k, v = (st[n].detach().double() for n in ("q", "k", "v"))
    out, dq, dk, dv = (torch.zeros_like(x) for x in (q, q, k, v))
    lse = torch.full((Q_HEADS, q.shape[0]), -math.inf, dtype=torch.float64, device=DEVICE)
    for b in range(len(cu_q) - 1):
        q0, q1, k0, k1 = cu_q[b], cu_q[b + 1], cu_k[b], cu_k[b + 1]
        i = torch.arange(k1 - k0 - (q1 - q0), k1 - k0, device=DEVICE)[:, None]
        j = torch.arange(k1 - k0, device=DEVICE)
        ok = (j <= i) & ((j + WINDOW > i) | (j < sinks))
        for m in range(Q_HEADS):
            n = m // (Q_HEADS // k.shape[1])
            qm, km, vm = q[q0:q1, m], k[k0:k1, n], v[k0:k1, n]
            s = (qm @ km.t()).masked_fill(~ok, -math.inf)
            z = torch.logsumexp(s, 1)
            p = torch.exp(s - z[:, None])
            o = p @ vm
            out[q0:q1, m], lse[m, q0:q1] = o, z
            if case["train"]:
                do = st["dout"][q0:q1, m].double()
                ds = p * (do @ vm.t() - (do * o).sum(1, keepdim=True))
                dq[q0:q1, m] = ds @ km
                dk[k0:k1, n] += ds.t() @ qm
                dv[k0:k1, n] += p.t() @ do
    if not case["train"]:
        return {"out": out, "lse": lse}
    return {"out": out, "lse": lse, "dq": dq, "dk": dk, "dv": dv}
