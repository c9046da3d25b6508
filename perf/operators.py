"""Cases and plain forms of the serving operators around the paged cache.

The operators, each as a user's program calls it (``own``) and in its plain
form of elementary torch operations:

* ``append``: ``append_quantized``, new tokens into a paged cache held in 8
  bits (e4m3) with one scale for each (block, head);
* ``attend``: ``flash_attn_with_kvcache`` over such a cache (``k_descale`` /
  ``v_descale``), with or without new tokens in the same call;
* ``window``: ``flash_attn_with_kvcache`` with a sliding window and a few first
  tokens that stay visible (``window_size``, ``sink_tokens``), over float and
  8-bit caches; the pages behind the window are freed (-1 in the page table);
* ``prefill``: ``flash_attn_func`` / ``flash_attn_varlen_func`` with the same
  window and first tokens;
* ``copy``: ``copy_blocks``, blocks of every layer's caches copied at once;
* ``compact``: ``compact_blocks``, the blocks in use moved to the front of the
  pool and the page table renumbered.

``listed()`` names the cases, ``draw(rng)`` gives more of their ranges,
``prepare(case, seed)`` makes a state, ``run(state)`` is one pass, ``work(case)``
what a pass cannot do without and ``exact(case, seed)`` the result in 64 bits.
"""

import math
import os
import random
import sys

import torch

own = False

_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "cpu-attention_b200")
_DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}
_F8 = torch.float8_e4m3fn
_F8_MAX = 448.0
_MIN_EXP = -126  # smallest exponent of a block's scale


def listed():
    return [
        # one decode step's new tokens: latency
        dict(name="append one token", op="append", batch=32, new=1, packed=False, lo=17, hi=2047, kv_heads=8, dim=128,
             page=16, dtype="bf16"),
        # prompts of many lengths entering the cache at once
        dict(name="append prompts", op="append", batch=12, new=4099, packed=True, lo=0, hi=37, kv_heads=16, dim=128,
             page=16, dtype="bf16"),
        # the repository's decode workload, its cache held in 8 bits
        dict(name="attend 8-bit", op="attend", cache="8bit", batch=32, heads=16, kv_heads=16, dim=128, page=16, lo=17,
             hi=2047, new=0, dtype="bf16", lse=False, left=-1, sinks=0),
        # grouped heads, engine lengths
        dict(name="attend 8-bit grouped", op="attend", cache="8bit", batch=64, heads=64, kv_heads=8, dim=128, page=16,
             lo=1, hi=8191, new=0, dtype="bf16", lse=False, left=-1, sinks=0),
        # one user with a long document: work has to be split along the cache
        dict(name="attend 8-bit one long", op="attend", cache="8bit", batch=1, heads=32, kv_heads=8, dim=128, page=64,
             lo=131077, hi=131077, new=0, dtype="bf16", lse=True, left=-1, sinks=0),
        # a whole decode step in one call, 32-bit queries, small heads
        dict(name="attend 8-bit step", op="attend", cache="8bit", batch=64, heads=8, kv_heads=8, dim=64, page=32,
             lo=1401, hi=1599, new=1, dtype="fp32", lse=False, left=-1, sinks=0),
        # long conversations behind a window, first tokens kept, pages between them freed
        dict(name="window grouped", op="window", cache="bf16", batch=64, heads=32, kv_heads=8, dim=128, page=16, lo=1,
             hi=32767, new=1, dtype="bf16", lse=False, left=4095, sinks=4),
        # the same on 8-bit caches, few users: latency
        dict(name="window 8-bit small", op="window", cache="8bit", batch=4, heads=16, kv_heads=4, dim=64, page=16,
             lo=100, hi=5000, new=0, dtype="bf16", lse=False, left=511, sinks=4),
        # a long prompt through a windowed layer
        dict(name="prefill window", op="prefill", batch=1, lq=8192, lk=8192, packed=False, heads=16, kv_heads=4,
             dim=128, left=1023, right=0, sinks=4, causal=True, dtype="bf16"),
        # prompts of many lengths packed end to end
        dict(name="prefill window packed", op="prefill", batch=7, lq=1531, lk=1531, packed=True, heads=8, kv_heads=8,
             dim=64, left=255, right=0, sinks=16, causal=True, dtype="bf16"),
        # a beam or a shared prefix forks: its last blocks, in every layer
        dict(name="copy blocks", op="copy", layers=24, blocks=640, pairs=65, kv_heads=8, dim=128, page=16,
             cache="bf16"),
        # a pool that is half free after requests ended, 8-bit caches with their scales
        dict(name="compact blocks", op="compact", layers=12, blocks=2111, batch=24, width=64, lo=1, hi=1023,
             kv_heads=8, dim=128, page=16, cache="8bit", left=-1, sinks=0),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "window", "window", "prefill", "copy", "compact"])
    dim, page = rng.choice([32, 64, 128]), rng.choice([16, 16, 32, 48, 64, 128])
    kv_heads, group = rng.choice([1, 2, 3, 4, 8, 16]), rng.choice([1, 1, 2, 3, 4, 7, 8, 16])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    if op == "append":
        batch = _log(rng, 1, 64)
        packed = rng.random() < 0.5
        new = _log(rng, 1, max(1, 24000 // batch) if packed else max(1, min(400, 12000 // batch)))
        lo = rng.randrange(0, 300)
        return dict(op=op, batch=batch, new=new, packed=packed, lo=lo, hi=lo + rng.randrange(0, 900),
                    kv_heads=kv_heads, dim=dim, page=page, dtype=dtype)
    if op in ("attend", "window"):
        batch = _log(rng, 1, 64)
        most = max(64, min(100000, 1000000 // (batch * kv_heads)))
        hi = _log(rng, 16, most)
        win = op == "window"
        cache = rng.choice(["8bit", "bf16", "fp32"]) if win else "8bit"
        return dict(op=op, cache=cache, batch=batch, heads=kv_heads * group, kv_heads=kv_heads, dim=dim, page=page,
                    lo=rng.randrange(0, hi + 1), hi=hi, new=rng.choice([0, 0, 1]),
                    dtype=dtype if cache == "8bit" else cache, lse=rng.random() < 0.3,
                    left=_log(rng, 1, 4096) if win else -1, sinks=rng.choice([0, 1, 4, 17, 64]) if win else 0)
    if op == "prefill":
        batch = _log(rng, 1, 8)
        lq = _log(rng, 16, (8192 if dtype == "bf16" else 2000) // batch)
        kv_heads = min(kv_heads, 8)
        packed = rng.random() < 0.5
        causal = rng.random() < 0.7
        return dict(op=op, batch=batch, lq=lq, lk=lq if packed else lq + rng.choice([0, 0, 100, 333]), packed=packed,
                    heads=kv_heads * rng.choice([1, 2]), kv_heads=kv_heads, dim=dim, left=_log(rng, 1, 800),
                    right=0 if causal else _log(rng, 1, 200), sinks=rng.choice([0, 1, 4, 30, 150]), causal=causal,
                    dtype=dtype)
    layers, cache = _log(rng, 1, 15), rng.choice(["8bit", "bf16", "fp32"])
    block = kv_heads * page * dim * {"8bit": 1, "bf16": 2, "fp32": 4}[cache]
    blocks = _log(rng, 8, max(9, min(900, 400000000 // (2 * layers * block))))
    if op == "copy":
        return dict(op=op, layers=layers, blocks=blocks, pairs=_log(rng, 1, blocks // 2), kv_heads=kv_heads, dim=dim,
                    page=page, cache=cache)
    batch = _log(rng, 1, min(20, blocks // 2))
    width = max(1, blocks // (2 * batch))
    win = rng.random() < 0.5
    return dict(op=op, layers=layers, blocks=blocks, batch=batch, width=width, lo=0, hi=width * page,
                kv_heads=kv_heads, dim=dim, page=page, cache=cache, left=_log(rng, 1, width * page) if win else -1,
                sinks=rng.choice([0, 4, 40]) if win else 0)


# ---------------------------------------------------------------- inputs ----
def _spread(n, lo, hi):
    """n lengths spread evenly over [lo, hi] (the longest when there is one)."""
    return [hi] if n == 1 else [lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _lens(case, rng):
    lens = _spread(case["batch"], case["lo"], case["hi"])
    rng.shuffle(lens)
    return lens


def _pool_8bit(g, blocks, heads, page, dim):
    """Codes and scales of a pool of blocks whose tokens have a size of their own per (block, head)."""
    x = torch.randn(blocks, heads, page, dim, generator=g, device="cuda")
    x *= torch.exp2(torch.randint(-2, 3, (blocks, heads, 1, 1), generator=g, device="cuda").float())
    m, e = torch.frexp(x.abs().amax((2, 3)))
    scale = torch.exp2((e - 9 + (m > 0.875)).float())
    return (x / scale[:, :, None, None]).to(_F8), scale


def _pool(g, kind, blocks, heads, page, dim):
    if kind == "8bit":
        return _pool_8bit(g, blocks, heads, page, dim)
    return torch.randn(blocks, heads, page, dim, generator=g, device="cuda").to(_DTYPES[kind]), None


def _table(rng, needs, spare):
    """A page table with needs[i] blocks for sequence i in a shuffled order, and the pool's size."""
    total = sum(needs) + spare
    order = list(range(total))
    rng.shuffle(order)
    width = max(1, max(needs))
    rows, at = [], 0
    for n in needs:
        rows.append(order[at:at + n] + [-1] * (width - n))
        at += n
    return torch.tensor(rows, dtype=torch.int32, device="cuda"), max(1, total)


def prepare(case, seed):
    rng = random.Random(seed)
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, s = case["op"], {"case": dict(case)}
    if op == "prefill":
        _prepare_prefill(case, s, rng, g)
        return s
    if op == "copy":
        n = case["blocks"]
        order = list(range(n))
        rng.shuffle(order)
        p = case["pairs"]
        src = [order[rng.randrange(p, n)] for _ in range(p)]
        s["mapping"] = torch.tensor([[a, b] for a, b in zip(src, order[:p])], dtype=torch.int64, device="cuda")
        s["caches"] = _layers(case, g)
        return s
    page = case["page"]
    if op == "compact":
        lens = _lens(case, rng)
        s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        order = list(range(case["blocks"]))
        rng.shuffle(order)
        rows, at = [], 0
        for i, n in enumerate(lens):
            need = -(-n // page)
            row = order[at:at + need]
            at += need
            if i % 4 == 1 and rows:  # a fork: its first blocks are its parent's
                share = min(need, -(-lens[i - 1] // page)) // 2
                row[:share] = rows[-1][:share]
            rows.append(row + [-1] * (case["width"] - need))
        s["table"] = torch.tensor(rows, dtype=torch.int32, device="cuda")
        s["caches"] = _layers(case, g)
        return s
    kv, dim, new = case["kv_heads"], case["dim"], case["new"]
    lens = _lens(case, rng)
    news = _spread(case["batch"], 1, new) if case.get("packed") else [new] * case["batch"]
    if case.get("packed"):
        rng.shuffle(news)
    table, blocks = _decode_table(case, rng, lens, news)
    s["lens"], s["table"] = torch.tensor(lens, dtype=torch.int32, device="cuda"), table
    kind = "8bit" if op == "append" else case["cache"]
    s["k_cache"], s["k_scale"] = _pool(g, kind, blocks, kv, page, dim)
    s["v_cache"], s["v_scale"] = _pool(g, kind, blocks, kv, page, dim)
    dt = _DTYPES[case["dtype"] if kind == "8bit" else kind]
    s["k"] = s["v"] = None
    if new:
        shape = (sum(news), kv, dim) if case.get("packed") else (case["batch"], new, kv, dim)
        grow = torch.exp2(torch.randint(-2, 3, shape[:-1] + (1,), generator=g, device="cuda").float())
        s["k"] = (torch.randn(shape, generator=g, device="cuda") * grow).to(dt)
        s["v"] = torch.randn(shape, generator=g, device="cuda").to(dt)
    if case.get("packed"):
        s["cu"] = torch.tensor([sum(news[:i]) for i in range(len(news) + 1)], dtype=torch.int32, device="cuda")
        s["max_new"] = max(news)
    if op != "append":
        s["q"] = torch.randn(case["batch"], 1, case["heads"], dim, generator=g, device="cuda").to(dt)
    return s


def _decode_table(case, rng, lens, news):
    """Every page of a sequence; with a window, those between the first tokens and the window are freed (-1)."""
    page, left, sinks = case["page"], case.get("left", -1), case.get("sinks", 0)
    ends = [-(-(n + m) // page) for n, m in zip(lens, news)]
    holes = [(0, 0) if left < 0 else (-(-sinks // page), max(0, n + m - 1 - left) // page)
             for n, m in zip(lens, news)]
    needs = [e - max(0, b - a) for e, (a, b) in zip(ends, holes)]
    packed, total = _table(rng, needs, 3)
    if left < 0:
        return packed, total
    packed = packed.tolist()
    width = max(1, max(ends))
    rows = []
    for row, e, (a, b), need in zip(packed, ends, holes, needs):
        ids = row[:need]
        if b > a:
            ids = ids[:a] + [-1] * (b - a) + ids[a:]
        rows.append(ids + [-1] * (width - e))
    return torch.tensor(rows, dtype=torch.int32, device="cuda"), total


def _layers(case, g):
    out = []
    for _ in range(case["layers"]):
        for _ in range(2):
            c, scale = _pool(g, case["cache"], case["blocks"], case["kv_heads"], case["page"], case["dim"])
            out += [c] if scale is None else [c, scale]
    return out


def _prefill_lens(case):
    return _spread(case["batch"], 1, case["lq"]) if case["packed"] else [case["lq"]] * case["batch"]


def _prepare_prefill(case, s, rng, g):
    h, kv, d, dt = case["heads"], case["kv_heads"], case["dim"], _DTYPES[case["dtype"]]
    if case["packed"]:
        lens = _prefill_lens(case)
        rng.shuffle(lens)
        t = sum(lens)
        s["lens"] = lens
        s["cu"] = torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device="cuda")
        shapes = [(t, h, d), (t, kv, d), (t, kv, d)]
    else:
        b = case["batch"]
        shapes = [(b, case["lq"], h, d), (b, case["lk"], kv, d), (b, case["lk"], kv, d)]
    s["q"], s["k"], s["v"] = (torch.randn(x, generator=g, device="cuda").to(dt) for x in shapes)


# ------------------------------------------------------------------ a pass --
def run(s):
    case = s["case"]
    if own:
        return _run_own(case, s)
    return {"append": _plain_append_op, "attend": _plain_decode, "window": _plain_decode, "prefill": _plain_prefill,
            "copy": _plain_copy, "compact": _plain_compact}[case["op"]](case, s)


def _run_own(case, s):
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    import cpu_attention as C
    op = case["op"]
    if op == "append":
        C.append_quantized(s["k"], s["v"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["lens"],
                           s["table"], cu_seqlens_new=s.get("cu"), max_seqlen_new=s.get("max_new"))
        return _cache_state(s)
    if op in ("attend", "window"):
        opts = {}
        if s["k_scale"] is not None:
            opts.update(k_descale=s["k_scale"], v_descale=s["v_scale"])
        if op == "window":
            opts.update(window_size=(case["left"], 0), sink_tokens=case["sinks"])
        got = C.flash_attn_with_kvcache(s["q"], s["k_cache"], s["v_cache"], k=s["k"], v=s["v"],
                                        cache_seqlens=s["lens"], page_table=s["table"],
                                        return_softmax_lse=case["lse"], **opts)
        got = list(got) if case["lse"] else [got]
        return got + (_cache_state(s) if case["new"] else [])
    if op == "prefill":
        opts = dict(causal=case["causal"], window_size=(case["left"], case["right"]), sink_tokens=case["sinks"])
        if case["packed"]:
            return C.flash_attn_varlen_func(s["q"], s["k"], s["v"], s["cu"], s["cu"], case["lq"], case["lk"], **opts)
        return C.flash_attn_func(s["q"], s["k"], s["v"], **opts)
    if op == "copy":
        C.copy_blocks(s["caches"], s["mapping"])
        return s["caches"]
    table, used = C.compact_blocks(s["caches"], s["table"], s["lens"], case["page"],
                                   window_size=(case["left"], 0), sink_tokens=case["sinks"])
    return [table, used] + s["caches"]


def _cache_state(s):
    got = [s["k_cache"], s["v_cache"]]
    return got if s["k_scale"] is None else got + [s["k_scale"], s["v_scale"]]


# ------------------------------------------------------------- plain forms --
def _token_rows(cache, scale, k_side, block, off):
    """The rows of the tokens (block, off), [..., heads, dim] in 32 bits."""
    n, h, page, d = cache.shape
    if scale is not None:
        codes = cache.view(torch.uint8)[block, :, off].view(_F8).float()
        return codes * scale[block][..., None]
    if not k_side:
        return cache[block, :, off].float()
    if cache.dtype == torch.bfloat16:  # dims in pairs, K transposed inside its page
        return cache.view(n, h, d // 2, page, 2)[block, :, :, off].flatten(-2).float()
    return cache.view(n, h, d, page)[block, :, :, off]


def _plain_decode(case, s):
    page, new = case["page"], case["new"]
    if new and s["k_scale"] is not None:
        _plain_append(s, s["k"].flatten(0, 1), s["v"].flatten(0, 1), s["lens"], _dense_tokens(s["lens"], new), new)
    elif new:
        seq, pos = _dense_tokens(s["lens"], new)
        block, off = s["table"][seq, pos // page].long(), pos % page
        _plain_put(s["k_cache"], True, block, off, s["k"].flatten(0, 1))
        _plain_put(s["v_cache"], False, block, off, s["v"].flatten(0, 1))
    lens = s["lens"].long() + new
    left, sinks = case["left"], case["sinks"]
    if left < 0:
        pos = torch.arange(max(1, case["hi"] + new), device="cuda").expand(case["batch"], -1)
        seen = pos < lens[:, None]
    else:
        first = torch.arange(sinks, device="cuda").expand(case["batch"], -1)
        last = lens[:, None] - 1 - left + torch.arange(left + 1, device="cuda")
        pos = torch.cat([first, last], 1)
        seen = torch.cat([first < lens[:, None], last >= sinks], 1)
    pos = pos.clamp(min=0)
    width = s["table"].shape[1]
    rows = torch.arange(case["batch"], device="cuda")[:, None]
    block = torch.where(seen, s["table"][rows, (pos // page).clamp(max=width - 1)].long(), 0)
    off = pos % page
    keys = _token_rows(s["k_cache"], s["k_scale"], True, block, off)
    values = torch.where(seen[:, :, None, None], _token_rows(s["v_cache"], s["v_scale"], False, block, off), 0.0)
    b, h, kv, d = case["batch"], case["heads"], case["kv_heads"], case["dim"]
    q = s["q"].float().view(b, kv, h // kv, d)
    w = torch.matmul(q, keys.permute(0, 2, 3, 1)) * d ** -0.5
    w = torch.where(seen[:, None, None, :], w, -math.inf)
    out, lse = _softmax_rows(w, values.permute(0, 2, 1, 3))
    out = [out.reshape(b, 1, h, d).to(s["q"].dtype)]
    return out + ([lse.reshape(b, h, 1)] if case["lse"] else []) + (_cache_state(s) if new else [])


def _softmax_rows(w, values):
    """softmax(w) @ values and the log-sum-exp; rows that see nothing give 0 and -inf."""
    m = w.amax(-1, keepdim=True)
    safe = torch.where(m == -math.inf, 0.0, m)
    p = torch.exp(w - safe)
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, values) / torch.where(total > 0, total, 1.0)
    return out, (safe + torch.log(total)).squeeze(-1)


def _dense_tokens(lens, new):
    """(sequence, position) of the new tokens of a [batch, new] append."""
    b = lens.shape[0]
    seq = torch.arange(b, device="cuda")[:, None].expand(b, new)
    return seq.flatten(), (lens.long()[:, None] + torch.arange(new, device="cuda")).flatten()


def _plain_put(cache, k_side, block, off, rows):
    n, h, page, d = cache.shape
    if not k_side:
        cache[block, :, off] = rows
    elif cache.dtype == torch.bfloat16:
        cache.view(n, h, d // 2, page, 2)[block, :, :, off] = rows.unflatten(-1, (d // 2, 2))
    else:
        cache.view(n, h, d, page)[block, :, :, off] = rows


def _plain_append_op(case, s):
    if case["packed"]:
        at = torch.arange(s["k"].shape[0], device="cuda")
        seq = torch.searchsorted(s["cu"], at, right=True, out_int32=True).long() - 1
        tokens = (seq, s["lens"].long()[seq] + at - s["cu"].long()[seq])
        _plain_append(s, s["k"], s["v"], s["lens"], tokens, s["max_new"])
    else:
        _plain_append(s, s["k"].flatten(0, 1), s["v"].flatten(0, 1), s["lens"], _dense_tokens(s["lens"], case["new"]),
                      case["new"])
    return _cache_state(s)


def _plain_append(s, k, v, lens, tokens, max_new):
    """The pages that get tokens, as one dense tile each: requantised with the scale that now fits them."""
    seq, pos = tokens
    page, width = s["k_cache"].shape[2], s["table"].shape[1]
    first = lens.long() // page
    most = (max_new + page - 2) // page + 1
    index = first[:, None] + torch.arange(most, device="cuda")
    ids = torch.where(index < width, s["table"].long().gather(1, index.clamp(max=width - 1)), -1)
    tile = pos // page - first[seq]
    got = torch.zeros(ids.shape + (page,), dtype=torch.bool, device="cuda")
    got[seq, tile, pos % page] = True
    ids = torch.where(got.any(-1), ids, -1)
    keep = ids >= 0
    for_pages = (seq, tile, pos % page, got, ids, keep)
    _plain_append_side(s["k_cache"], s["k_scale"], k, *for_pages)
    _plain_append_side(s["v_cache"], s["v_scale"], v, *for_pages)


def _plain_append_side(cache, scale, rows, seq, tile, off, got, ids, keep):
    safe = ids.clamp(min=0)
    b, p, page = got.shape
    h, d = cache.shape[1], cache.shape[3]
    fresh = got[:, :, 0]  # the page's first token is new: what it held is void
    old = torch.where(fresh[:, :, None], 0.0, scale[safe])
    new = torch.zeros(b, p, page, h, d, device="cuda")
    new[seq, tile, off] = rows.float()
    m, e = torch.frexp(new.abs().amax((2, 4)))
    fit = torch.exp2((e - 9 + (m > 0.875)).clamp(min=_MIN_EXP).float())
    now = torch.maximum(old, torch.where(m > 0, fit, 2.0 ** _MIN_EXP))
    codes = cache.view(torch.uint8)[safe]
    moved = (codes.view(_F8).float() * (old / now)[:, :, :, None, None]).to(_F8).view(torch.uint8)
    codes = torch.where((old == now)[:, :, :, None, None] | fresh[:, :, None, None, None], codes, moved)
    put = (new.permute(0, 1, 3, 2, 4) / now[:, :, :, None, None]).to(_F8).view(torch.uint8)
    codes = torch.where(got[:, :, None, :, None], put, codes)
    cache.view(torch.uint8)[ids[keep]] = codes[keep]
    scale[ids[keep]] = now[keep]


def _plain_prefill(case, s):
    h, kv, d = case["heads"], case["kv_heads"], case["dim"]
    lead = (1,) if case["packed"] else ()
    q, k, v = (x.float().view(lead + x.shape) for x in (s["q"], s["k"], s["v"]))
    b, lq, lk = q.shape[0], q.shape[1], k.shape[1]
    q = q.view(b, lq, kv, h // kv, d).permute(0, 2, 3, 1, 4).reshape(b, kv, -1, d)
    w = torch.matmul(q, k.permute(0, 2, 3, 1)).view(b, kv, h // kv, lq, lk) * d ** -0.5
    w = torch.where(_seen(case, s, lq, lk), w, -math.inf)
    out, _ = _softmax_rows(w.flatten(2, 3), v.permute(0, 2, 1, 3))
    out = out.view(b, h, lq, d).transpose(1, 2).to(s["q"].dtype)
    return out.reshape(s["q"].shape)


def _seen(case, s, lq, lk):
    """[lq, lk]: whether row i sees key j."""
    i, j = torch.arange(lq, device="cuda")[:, None], torch.arange(lk, device="cuda")[None]
    same = True
    if case["packed"]:
        si = torch.searchsorted(s["cu"], i, right=True) - 1
        sj = torch.searchsorted(s["cu"], j, right=True) - 1
        same = si == sj
        i, j = i - s["cu"].long()[si], j - s["cu"].long()[sj]
    else:
        i = i + lk - lq
    seen = (j >= i - case["left"]) | (j < case["sinks"])
    return seen & (j <= i + case["right"]) & same


def _bytes_of(c):
    return c.view(torch.uint8) if c.dtype == _F8 else c


def _plain_copy(case, s):
    src, dst = s["mapping"][:, 0], s["mapping"][:, 1]
    [_bytes_of(c).index_copy_(0, dst, _bytes_of(c)[src]) for c in s["caches"]]
    return s["caches"]


def _plain_compact(case, s):
    table, lens, page, n = s["table"].long(), s["lens"].long(), case["page"], case["blocks"]
    at = torch.arange(table.shape[1], device="cuda") * page
    live = at < lens[:, None]
    if case["left"] >= 0:
        live &= (at + page > lens[:, None] - 1 - case["left"]) | (at < case["sinks"])
    used = torch.zeros(n, dtype=torch.bool, device="cuda")
    used[table[live]] = True
    count = used.sum()
    place = torch.arange(n, device="cuda")
    dst, src = place[~used & (place < count)], place[used & (place >= count)]
    dst = dst[:src.shape[0]]
    place[src] = dst
    [_bytes_of(c).index_copy_(0, dst, _bytes_of(c)[src]) for c in s["caches"]]
    new = torch.where(live, place[table.clamp(min=0)], -1).to(torch.int32)
    return [new, count.to(torch.int32).view(1)] + s["caches"]


# -------------------------------------------------------------------- work --
def _visible(case):
    """Keys that the sequences' rows see, and their sum of pages, in a decode."""
    got = []
    for n in _spread(case["batch"], case["lo"], case["hi"]):
        n += case["new"]
        lo = 0 if case["left"] < 0 else max(0, n - 1 - case["left"])
        got.append(n if lo <= case["sinks"] else min(n, case["sinks"]) + n - lo)
    return got


def work(case):
    op, kv, d = case["op"], case["kv_heads"], case["dim"]
    size = {"8bit": 1, "bf16": 2, "fp32": 4}
    if op == "append":
        tokens = sum(_spread(case["batch"], 1, case["new"])) if case["packed"] else case["batch"] * case["new"]
        values = 2 * tokens * kv * d
        return {"bytes": values * (size[case["dtype"]] + 1), "flops": 2 * values}
    if op in ("attend", "window"):
        keys = sum(_visible(case))
        kind = case["cache"]
        act = size[case["dtype"] if kind == "8bit" else kind]
        cells = 2 * keys * kv
        scales = 4 * cells / case["page"] if kind == "8bit" else 0
        rows = case["batch"] * d * (2 * case["heads"] + 2 * kv * case["new"]) * act
        return {"bytes": cells * d * size[kind] + scales + rows, "flops": 4 * keys * case["heads"] * d}
    if op == "prefill":
        pairs = tokens_q = tokens_k = 0
        for n in _prefill_lens(case):
            m = n if case["packed"] else case["lk"]
            tokens_q, tokens_k = tokens_q + n, tokens_k + m
            for i in range(n):
                at = i + m - n
                hi = min(m - 1, at + case["right"])
                lo = max(0, at - case["left"])
                first = min(case["sinks"], lo, hi + 1)
                pairs += max(0, first) + max(0, hi + 1 - lo)
        act = size[case["dtype"]]
        return {"bytes": act * d * (2 * tokens_q * case["heads"] + 2 * tokens_k * kv),
                "flops": 4 * pairs * case["heads"] * d}
    block = kv * case["page"] * d * size[case["cache"]] + (4 * kv if case["cache"] == "8bit" else 0)
    if op == "copy":
        return {"bytes": 2 * case["layers"] * 2 * case["pairs"] * block, "flops": 0}
    # about (blocks - used) / blocks of the used blocks lie past the end of the packed pool
    used = sum(-(-n // case["page"]) for n in _spread(case["batch"], case["lo"], case["hi"]))
    moved = max(1, used * (case["blocks"] - used) // case["blocks"])
    return {"bytes": 2 * case["layers"] * 2 * moved * block + 8 * case["batch"] * case["width"], "flops": 0}


# ------------------------------------------------------------------- exact --
def exact(case, seed):
    """The same outputs in 64 bits, sequence by sequence from the definition."""
    s = prepare(case, seed)
    op = case["op"]
    if op == "copy":
        caches = [c.double() for c in s["caches"]]
        before = [c.clone() for c in caches]
        for a, b in s["mapping"].tolist():
            for c, was in zip(caches, before):
                c[b] = was[a]
        return caches
    if op == "compact":
        return _exact_compact(case, s)
    if op == "prefill":
        return _exact_prefill(case, s)
    lens = s["lens"].tolist()
    table = s["table"].tolist()
    state = None
    if case["new"]:
        state = _exact_append(case, s, lens, table)
        if op == "append":
            return state
    out, lse = [], []
    for i, n in enumerate(lens):
        n += case["new"]
        o, z = _exact_row(case, s, state, i, n, table[i])
        out.append(o)
        lse.append(z)
    got = [torch.stack(out)[:, None]]
    if case["lse"]:
        got.append(torch.stack(lse)[:, :, None])
    return got + (state or [])


def _exact_row(case, s, state, i, n, row):
    h, kv, d, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    low = 0 if case["left"] < 0 else n - 1 - case["left"]
    pages = [p for p in range(-(-n // page)) if (p + 1) * page > low or p * page < case["sinks"]]
    if not pages:
        return (torch.zeros(h, d, dtype=torch.float64, device="cuda"),
                torch.full((h,), -math.inf, dtype=torch.float64, device="cuda"))
    ids = torch.tensor([row[p] for p in pages], device="cuda")
    at = (torch.tensor(pages, device="cuda")[:, None] * page + torch.arange(page, device="cuda")).flatten()
    keep = at < n
    if low > 0:
        keep &= (at >= low) | (at < case["sinks"])
    sides = []
    for k, name in enumerate(("k", "v")):
        if s[name + "_scale"] is not None:
            codes = state[k][ids] if state else s[name + "_cache"].view(torch.uint8)[ids].view(_F8).double()
            x = codes * (state[2 + k] if state else s[name + "_scale"].double())[ids][:, :, None, None]
        else:
            x = (state[k] if state else s[name + "_cache"].double())[ids]
            if k == 0 and case["cache"] == "bf16":
                x = x.reshape(-1, kv, d // 2, page, 2).transpose(2, 3).reshape(-1, kv, page, d)
            elif k == 0:
                x = x.reshape(-1, kv, d, page).transpose(2, 3)
        sides.append(x.transpose(0, 1).reshape(kv, -1, d)[:, keep])
    q = s["q"][i, 0].double().view(kv, h // kv, d)
    w = q @ sides[0].transpose(1, 2) / math.sqrt(d)
    z = torch.logsumexp(w, -1)
    return (torch.exp(w - z[..., None]) @ sides[1]).reshape(h, d), z.reshape(h)


def _exact_append(case, s, lens, table):
    """The caches' codes (or values) and scales after the append."""
    page = case["page"]
    if case.get("packed"):
        cu = s["cu"].tolist()
        new = [[s[x][cu[i]:cu[i + 1]] for x in "kv"] for i in range(len(lens))]
    else:
        new = [[s[x][i] for x in "kv"] for i in range(len(lens))]
    got = []
    scales = []
    for side, name in enumerate(("k", "v")):
        cache, scale = s[name + "_cache"], s[name + "_scale"]
        if scale is None:
            cache = cache.clone()
            for i, n in enumerate(lens):
                for j, row in enumerate(new[i][side]):
                    block, off = cache[table[i][(n + j) // page]], (n + j) % page
                    if side:
                        block[:, off] = row
                    elif cache.dtype == torch.bfloat16:
                        block.view(row.shape[0], -1, page, 2)[:, :, off] = row.reshape(row.shape[0], -1, 2)
                    else:
                        block.view(row.shape[0], -1, page)[:, :, off] = row
            got.append(cache.double())
            continue
        codes, scale = cache.clone().view(torch.uint8).view(_F8).double(), scale.double()
        for i, n in enumerate(lens):
            rows = new[i][side].double()
            for p in range(n // page, -(-(n + rows.shape[0]) // page)):
                a, z = max(n, p * page), min(n + rows.shape[0], (p + 1) * page)
                x = rows[a - n:z - n].transpose(0, 1)
                top = x.abs().amax((1, 2)) / _F8_MAX
                power = torch.ceil(torch.log2(top)).clamp(min=_MIN_EXP)
                # log2 of a power of two itself may be off by its last bit
                power = torch.where(torch.exp2(power - 1) >= top, power - 1, power).clamp(min=_MIN_EXP)
                fit = torch.exp2(torch.where(torch.exp2(power) < top, power + 1, power))
                b = table[i][p]
                if a > p * page:
                    was, fit = scale[b], torch.maximum(scale[b], fit)
                    codes[b] = _round_8bit(codes[b] * (was / fit)[:, None, None])
                scale[b] = fit
                codes[b][:, a - p * page:z - p * page] = _round_8bit(x / fit[:, None, None])
        got.append(codes)
        scales.append(scale)
    return got + scales


def _round_8bit(x):
    """The nearest e4m3 value (ties to even), in 64 bits."""
    _, e = torch.frexp(x)
    step = torch.exp2((e - 4).clamp(min=-9).double())
    return (torch.round(x / step) * step).clamp(-_F8_MAX, _F8_MAX)


def _exact_prefill(case, s):
    h, kv, d = case["heads"], case["kv_heads"], case["dim"]
    starts = s["cu"].tolist() if case["packed"] else None
    out = []
    for i in range(case["batch"]):
        if case["packed"]:
            q, k, v = (s[x][starts[i]:starts[i + 1]].double() for x in "qkv")
        else:
            q, k, v = (s[x][i].double() for x in "qkv")
        lq, lk = q.shape[0], k.shape[0]
        rows = []
        for a in range(0, lq, 1024):
            at = torch.arange(a, min(lq, a + 1024), device="cuda")[:, None] + lk - lq
            j = torch.arange(lk, device="cuda")[None]
            hide = (j > at + case["right"]) | ((j < at - case["left"]) & (j >= case["sinks"]))
            heads = []
            for head in range(h):
                w = q[a:a + 1024, head] @ k[:, head * kv // h].T / math.sqrt(d)
                w = w.masked_fill(hide, -math.inf)
                p = torch.softmax(w, -1).nan_to_num(0.0)
                heads.append(p @ v[:, head * kv // h])
            rows.append(torch.stack(heads, 1))
        out.append(torch.cat(rows))
    return torch.cat(out) if case["packed"] else torch.stack(out)


def _exact_compact(case, s):
    page, left, sinks = case["page"], case["left"], case["sinks"]
    table, lens = s["table"].tolist(), s["lens"].tolist()
    live = set()
    for row, n in zip(table, lens):
        for p in range(-(-n // page)):
            if left < 0 or (p + 1) * page > n - 1 - left or p * page < sinks:
                live.add(row[p])
    free = [b for b in range(len(live)) if b not in live]
    moves = dict(zip(sorted(b for b in live if b >= len(live)), free))
    new = []
    for row, n in zip(table, lens):
        new.append([moves.get(b, b) if p * page < n and (left < 0 or (p + 1) * page > n - 1 - left or p * page < sinks)
                    else -1 for p, b in enumerate(row)])
    caches = [c.double() for c in s["caches"]]
    for a, b in moves.items():
        for c in caches:
            c[b] = c[a]
    return [torch.tensor(new, dtype=torch.int32, device="cuda"),
            torch.tensor([len(live)], dtype=torch.int32, device="cuda")] + caches
