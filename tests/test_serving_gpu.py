"""Caches held in 8 bits, windows with first tokens and block moves on the B200,
against float64 implementations (tests/serving.py) with derived bounds."""

import math

import pytest
import torch

import serving as S

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, FP32 = torch.bfloat16, torch.float32


def api():
    import cpu_attention
    return cpu_attention


def kernel():
    from cpu_attention import _kernel
    return _kernel


def status(reset=True):
    K = kernel()
    return K.status(torch.device("cuda", torch.cuda.current_device()), reset=reset)


def bytes_of(t):
    """The bytes of a tensor [blocks, ...], one row per block."""
    return t.contiguous().reshape(t.shape[0], -1).view(torch.uint8).cpu()


# ------------------------------------------------------------------- append --
def empty_8bit(blocks, heads, page, d, fill=0x7f):
    c = torch.full((blocks, heads, page, d), fill, dtype=torch.uint8, device=DEV).view(S.F8)
    return c, c.clone(), torch.zeros(blocks, heads, device=DEV), torch.zeros(blocks, heads, device=DEV)


def check_append(kc, vc, ks, vs, want):
    for got, ref in ((kc, want[0]), (vc, want[1])):
        g = got.cpu().double()
        assert torch.equal(torch.isnan(g), torch.isnan(ref))
        assert torch.equal(g[~torch.isnan(g)], ref[~torch.isnan(ref)])
    assert torch.equal(ks.cpu().double(), want[2]) and torch.equal(vs.cpu().double(), want[3])


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("d,page", [(128, 16), (64, 32), (32, 48), (128, 128)])
def test_append_matches_definition(dtype, d, page):
    """Appends of several sizes to the same caches, magnitudes growing and shrinking: codes and scales equal the
    definition exactly (powers of two, one rounding)."""
    g = torch.Generator().manual_seed(d + page)
    heads, batch = 3, 4
    width = 5
    table = torch.randperm(batch * width + 2, generator=g)[:batch * width].reshape(batch, width).to(torch.int32)
    blocks = batch * width + 2
    kc, vc, ks, vs = empty_8bit(blocks, heads, page, d, 0)
    want = [torch.zeros(blocks, heads, page, d, dtype=torch.float64) for _ in range(2)] \
        + [torch.zeros(blocks, heads, dtype=torch.float64) for _ in range(2)]
    lens = [0, page - 1, 3, page]
    for n, size in ((1, 1.0), (1, 300.0), (page + 3, 1e-3), (2, 1e4), (1, 1e-30), (page // 2, 7.0)):
        k, v = (torch.randn(batch, n, heads, d, generator=g).mul(size).to(dtype) for _ in range(2))
        api().append_quantized(k.to(DEV), v.to(DEV), kc, vc, ks, vs, torch.tensor(lens, dtype=torch.int32, device=DEV),
                               table.to(DEV))
        for x, r in enumerate((k, v)):
            S.append(want[x], want[2 + x], [t.double() for t in r], lens, table.tolist(), page)
        check_append(kc, vc, ks, vs, want)
        lens = [a + n for a in lens]
    assert status() == 0


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_append_packed_strided_and_left_out(dtype):
    """Packed tokens as views of a fused projection (also at an odd element: no 16-byte loads), a sequence of zero
    tokens, one left out by a negative length; blocks of nobody and slots behind a block's tokens stay as they were."""
    g = torch.Generator().manual_seed(1)
    heads, d, page = 2, 64, 16
    news, lens = [5, 0, 40, 1, 9], [3, 7, 0, 31, -1]
    total = sum(news)
    for odd in (0, 1):
        flat = torch.randn(total * (2 * heads * d + 8) + odd, generator=g).to(dtype).to(DEV)
        fused = flat[odd:].view(total, 2 * heads * d + 8)
        k, v = (fused[:, x * heads * d:(x + 1) * heads * d].view(total, heads, d) for x in range(2))
        cu = torch.tensor([sum(news[:i]) for i in range(6)], dtype=torch.int32, device=DEV)
        table = torch.randperm(24, generator=g)[:20].reshape(5, 4).to(torch.int32)
        kc, vc, ks, vs = empty_8bit(24, heads, page, d, 0x31)
        ks += 0.5
        vs += 0.25
        want = [kc.cpu().double(), vc.cpu().double(), ks.cpu().double(), vs.cpu().double()]
        api().append_quantized(k, v, kc, vc, ks, vs, torch.tensor(lens, dtype=torch.int32, device=DEV), table.to(DEV),
                               cu_seqlens_new=cu, max_seqlen_new=40)
        for x, r in enumerate((k, v)):
            rows = [r[sum(news[:i]):sum(news[:i + 1])].cpu().double() for i in range(5)]
            S.append(want[x], want[2 + x], rows, lens, table.tolist(), page)
        check_append(kc, vc, ks, vs, want)
    # offsets and lengths on the host
    api().append_quantized(k, v, kc, vc, ks, vs, torch.tensor(lens, dtype=torch.int32), table, cu_seqlens_new=cu.cpu())
    for x, r in enumerate((k, v)):
        rows = [r[sum(news[:i]):sum(news[:i + 1])].cpu().double() for i in range(5)]
        S.append(want[x], want[2 + x], rows, lens, table.tolist(), page)
    check_append(kc, vc, ks, vs, want)
    assert status() == 0


def test_append_infinities_nan_and_zeros():
    """An infinity becomes the largest code and sets no scale, NaN stays NaN, zeros alone take the smallest scale."""
    kc, vc, ks, vs = empty_8bit(2, 1, 16, 32, 0)
    k = torch.zeros(1, 2, 1, 32)
    k[0, 0, 0, :4] = torch.tensor([math.inf, -math.inf, math.nan, 3.0])
    v = torch.zeros(1, 2, 1, 32)
    api().append_quantized(k.to(DEV), v.to(DEV), kc, vc, ks, vs, torch.zeros(1, dtype=torch.int32, device=DEV),
                           torch.zeros(1, 1, dtype=torch.int32, device=DEV))
    s = S.fit_scale(torch.tensor([3.0]))
    assert ks[0, 0].item() == s and vs[0, 0].item() == 2.0 ** -126
    row = kc[0, 0, 0].cpu().double()
    assert row[0] == 448 and row[1] == -448 and torch.isnan(row[2]) and row[3] * s == 3.0
    assert (vc[0, 0, :2].cpu().double() == 0).all()


def test_append_out_of_place_is_flagged():
    """Positions past the table and bad entries are skipped and flagged, the rest is written."""
    K = kernel()
    g = torch.Generator().manual_seed(2)
    k, v = (torch.randn(3, 20, 1, 32, generator=g).to(DEV) for _ in range(2))
    kc, vc, ks, vs = empty_8bit(8, 1, 16, 32, 0)
    table = torch.tensor([[0, 1], [2, 99], [-5, 3]], dtype=torch.int32, device=DEV)
    status()
    api().append_quantized(k, v, kc, vc, ks, vs, torch.tensor([16, 0, 0], dtype=torch.int32, device=DEV), table)
    assert status() == K.STATUS_LENS | K.STATUS_TABLE
    want = [torch.zeros(8, 1, 16, 32, dtype=torch.float64) for _ in range(2)] \
        + [torch.zeros(8, 1, dtype=torch.float64) for _ in range(2)]
    for x, r in enumerate((k, v)):
        S.append(want[x], want[2 + x], [t.cpu().double() for t in r], [16, 0, 0], table.tolist(), 16)
    check_append(kc, vc, ks, vs, want)
    # more tokens in a packed sequence than stated: the first ones are stored
    cu = torch.tensor([0, 20], dtype=torch.int32, device=DEV)
    api().append_quantized(k[0], v[0], kc, vc, ks, vs, torch.zeros(1, dtype=torch.int32, device=DEV), table[:1], cu, 4)
    assert status() == K.STATUS_LENS


# ------------------------------------------------------------------- decode --
LENS = [0, 1, 15, 16, 17, 100, 333, 0, 1030]


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("h,hk", [(4, 4), (6, 2), (8, 1), (20, 2)])
def test_decode_8bit(dtype, d, page, h, hk):
    pc = S.Paged("8bit", LENS, hk, d, page, dtype, seed=d + page + h)
    q = torch.randn(len(LENS), 1, h, d, generator=torch.Generator().manual_seed(h)).to(dtype).to(DEV)
    out, lse = api().flash_attn_with_kvcache(q, pc.k_cache, pc.v_cache, cache_seqlens=pc.L, page_table=pc.bt,
                                             return_softmax_lse=True, **pc.opts())
    assert out.shape == q.shape and out.dtype == dtype
    S.check_decode(out, lse, q, pc, h)
    assert status() == 0
    again = api().flash_attn_with_kvcache(q, pc.k_cache, pc.v_cache, cache_seqlens=pc.L, page_table=pc.bt, **pc.opts())
    assert torch.equal(out, again)


@pytest.mark.parametrize("kind", ["8bit", "bf16", "fp32"])
@pytest.mark.parametrize("d,page,h,hk", [(128, 16, 8, 2), (64, 32, 4, 4), (32, 48, 18, 2)])
@pytest.mark.parametrize("left,sinks", [(0, 0), (0, 1), (15, 4), (16, 16), (100, 17), (5000, 3), (64, 0), (-1, 7),
                                        (31, 400)])
def test_decode_window(kind, d, page, h, hk, left, sinks):
    dtype = FP32 if kind == "fp32" else BF16
    pc = S.Paged(kind, LENS, hk, d, page, dtype, seed=left + sinks, left=left, sinks=sinks)
    q = torch.randn(len(LENS), 1, h, d, generator=torch.Generator().manual_seed(h)).to(dtype).to(DEV)
    out, lse = api().flash_attn_with_kvcache(q, pc.k_cache, pc.v_cache, cache_seqlens=pc.L, page_table=pc.bt,
                                             window_size=(left, 0), sink_tokens=sinks, return_softmax_lse=True,
                                             **pc.opts())
    S.check_decode(out, lse, q, pc, h)
    assert status() == 0


@pytest.mark.parametrize("kind", ["8bit", "bf16", "fp32"])
@pytest.mark.parametrize("lens,h,hk", [([40000], 8, 1), ([9000, 1, 0, 12345], 32, 8), ([700] * 40, 4, 4)])
def test_decode_long_and_split(kind, lens, h, hk):
    """Items that many warps and CTAs share: joined in order, the same bits each time."""
    dtype = FP32 if kind == "fp32" else BF16
    pc = S.Paged(kind, lens, hk, 128, 16, dtype, seed=3, left=-1)
    q = torch.randn(len(lens), 1, h, 128, generator=torch.Generator().manual_seed(5)).to(dtype).to(DEV)
    call = lambda: api().flash_attn_with_kvcache(q, pc.k_cache, pc.v_cache, cache_seqlens=pc.L,  # noqa: E731
                                                 page_table=pc.bt, sink_tokens=0, return_softmax_lse=True, **pc.opts())
    out, lse = call()
    S.check_decode(out, lse, q, pc, h)
    for _ in range(3):
        o2, l2 = call()
        assert torch.equal(out, o2) and torch.equal(lse, l2)


def test_decode_large_scores_scales_and_queries():
    """Scores far apart, queries of 2^-120 to 2^100, scales from 2^-100 to 2^20, a negative softmax scale, an explicit
    one, a block of scale 0."""
    lens, h = [200, 37, 64], 4
    for dtype in (BF16, FP32):
        pc = S.Paged("8bit", lens, 2, 64, 16, dtype, seed=4)
        for x in range(2):
            e = torch.randint(-100 if x else -30, 21 if x else 3, pc.scale[x].shape,
                              generator=torch.Generator().manual_seed(x))
            pc.scale[x] = torch.exp2(e.double())
            pc.scale[x][pc.table[0][1]] = 0.0
        pc.k_scale, pc.v_scale = (s.float().to(DEV) for s in pc.scale)
        base = torch.randn(3, 1, h, 64, generator=torch.Generator().manual_seed(9))
        for size, scale in ((1.0, None), (2.0 ** -120, None), (2.0 ** 100, 2.0 ** -100), (1.0, -0.05), (1.0, 0.0)):
            q = (base * size).to(dtype).to(DEV)
            out, lse = api().flash_attn_with_kvcache(q, pc.k_cache, pc.v_cache, cache_seqlens=pc.L, page_table=pc.bt,
                                                     softmax_scale=scale, return_softmax_lse=True, **pc.opts())
            S.check_decode(out, lse, q, pc, h, scale)


@pytest.mark.parametrize("kind", ["8bit", "bf16", "fp32"])
@pytest.mark.parametrize("n", [1, 3, 21])
@pytest.mark.parametrize("window", [None, (20, 4)])
def test_decode_appends(kind, n, window):
    """k/v in the call: the caches afterwards equal the two-step route's, and the row sees its new tokens."""
    dtype = FP32 if kind == "fp32" else BF16
    lens, h, hk, d, page = [0, 15, 16, 100, 31], 4, 2, 64, 16
    left, sinks = window if window else (-1, 0)
    pc = S.Paged(kind, lens, hk, d, page, dtype, seed=n * 2, left=left, sinks=sinks, room=n)
    if kind == "8bit":  # what was never written must be a number: the append keeps what a block holds
        for c in (pc.k_cache, pc.v_cache):
            u = c.view(torch.uint8)
            u[(u & 0x7f) == 0x7f] = 0
    g = torch.Generator().manual_seed(n)
    k, v = (torch.randn(len(lens), n, hk, d, generator=g).to(dtype).to(DEV) for _ in range(2))
    q = torch.randn(len(lens), 1, h, d, generator=g).to(dtype).to(DEV)
    opts = dict(window_size=(left, 0), sink_tokens=sinks) if window else (dict() if kind == "8bit"
                                                                         else dict(sink_tokens=0))
    k2, v2 = pc.k_cache.clone(), pc.v_cache.clone()
    s2 = [None if s is None else s.clone() for s in (pc.k_scale, pc.v_scale)]
    # the call's own route first on the live caches
    out = api().flash_attn_with_kvcache(q, pc.k_cache, pc.v_cache, k=k, v=v, cache_seqlens=pc.L, page_table=pc.bt,
                                        **pc.opts(), **opts)
    if kind == "8bit":
        api().append_quantized(k, v, k2, v2, *s2, pc.L, pc.bt)
        assert torch.equal(s2[0], pc.k_scale) and torch.equal(s2[1], pc.v_scale)
        pc.scale = [s.cpu().double() for s in (pc.k_scale, pc.v_scale)]
    else:
        pos = pc.L.long()[:, None] + torch.arange(n, device=DEV)
        slots = pc.bt.long().gather(1, pos // page) * page + pos % page
        api().reshape_and_cache(k.flatten(0, 1), v.flatten(0, 1), k2, v2, slots.flatten())
    assert torch.equal(bytes_of(k2), bytes_of(pc.k_cache)) and torch.equal(bytes_of(v2), bytes_of(pc.v_cache))
    pc.rows = [S.unpack(c.cpu().double() if kind == "8bit" else c.cpu(), x == 0, kind).double()
               for x, c in enumerate((pc.k_cache, pc.v_cache))]
    S.check_decode(out, None, q, pc, h, lens=[a + n for a in lens])
    assert status() == 0


def test_decode_negative_length_and_bad_table():
    """A negative length and bad entries read nothing out of place: zeros, or the rest of the row, and a flag."""
    K = kernel()
    pc = S.Paged("8bit", [40, 40, 40], 2, 64, 16, BF16, seed=6)
    q = torch.randn(3, 1, 2, 64, generator=torch.Generator().manual_seed(0)).bfloat16().to(DEV)
    bt = pc.bt.clone()
    bt[1, 1] = -3
    bt[2, 0] = 1 << 30
    status()
    out = api().flash_attn_with_kvcache(q, pc.k_cache, pc.v_cache, cache_seqlens=pc.L, page_table=bt, **pc.opts())
    assert status() == K.STATUS_TABLE
    good = api().flash_attn_with_kvcache(q, pc.k_cache, pc.v_cache, cache_seqlens=pc.L, page_table=pc.bt, **pc.opts())
    assert torch.equal(out[0], good[0]) and torch.isfinite(out).all()
    L = torch.tensor([40, -1, 400], dtype=torch.int32, device=DEV)
    out = api().flash_attn_with_kvcache(q[:2], pc.k_cache, pc.v_cache, cache_seqlens=L[:2], page_table=pc.bt[:2],
                                        **pc.opts())
    assert torch.equal(out[0], good[0]) and (out[1] == 0).all() and status() == 0
    api().flash_attn_with_kvcache(q, pc.k_cache, pc.v_cache, cache_seqlens=L, page_table=pc.bt, **pc.opts())
    assert status() & K.STATUS_LENS


def test_decode_large_batch():
    """More sequences than one launch takes."""
    B = 9000
    g = torch.Generator().manual_seed(0)
    codes = torch.randn(64, 1, 16, 32, generator=g)
    kc, vc = codes.to(S.F8).to(DEV), codes.flip(0).contiguous().to(S.F8).to(DEV)
    one = torch.ones(64, 1, device=DEV)
    bt = torch.randint(0, 64, (B, 2), generator=g).to(torch.int32)
    L = torch.randint(0, 33, (B,), generator=g).to(torch.int32)
    q = torch.randn(B, 1, 1, 32, generator=g).bfloat16()
    out = api().flash_attn_with_kvcache(q.to(DEV), kc, vc, cache_seqlens=L.to(DEV), page_table=bt.to(DEV),
                                        k_descale=one, v_descale=one)
    for i in list(range(0, B, 611)) + [8191, 8192, 8999]:
        one_row = api().flash_attn_with_kvcache(q[i:i + 1].to(DEV), kc, vc, cache_seqlens=L[i:i + 1].to(DEV),
                                                page_table=bt[i:i + 1].to(DEV), k_descale=one, v_descale=one)
        assert (out[i] - one_row[0]).abs().max() <= 2 ** -7 * one_row.abs().max() + 1e-6, i
        if L[i] == 0:
            assert (out[i] == 0).all()


def test_decode_strided_queries_and_host_indices():
    """q as a view of a fused projection, lengths and table on the host, an int length, cache_batch_idx."""
    pc = S.Paged("8bit", [50, 50], 2, 64, 16, BF16, seed=8)
    fused = torch.randn(2, 1, 3, 4, 64, generator=torch.Generator().manual_seed(0)).bfloat16().to(DEV)
    q = fused[:, :, 1]
    ref = api().flash_attn_with_kvcache(q.contiguous(), pc.k_cache, pc.v_cache, cache_seqlens=pc.L, page_table=pc.bt,
                                        **pc.opts())
    for L, bt in ((pc.L, pc.bt), (pc.L.cpu(), pc.bt.cpu()), (50, pc.bt)):
        out = api().flash_attn_with_kvcache(q, pc.k_cache, pc.v_cache, cache_seqlens=L, page_table=bt, **pc.opts())
        assert torch.equal(out, ref)
    out = api().flash_attn_with_kvcache(q, pc.k_cache, pc.v_cache, cache_seqlens=pc.L, block_table=pc.bt.flip(0),
                                        cache_batch_idx=torch.tensor([1, 0], device=DEV), **pc.opts())
    assert torch.equal(out, ref)
    # the ctypes path answers the same
    from cpu_attention import _kernel as K, _native
    fast, K._FAST = K.fastpath(), False
    try:
        got = _native.decode_split(0, q, pc.k_cache, pc.v_cache, None, None, pc.k_scale, pc.v_scale, pc.L, pc.bt, -1, 0,
                                   None)
    finally:
        K._FAST = fast
    assert torch.equal(got, ref)


def test_decode_graphs_and_streams():
    """Two captured steps (append and attend) replayed side by side on two streams, with fresh inputs: equal to eager
    calls; nothing is shared between them."""
    C = api()
    steps = []
    for x in range(2):
        pc = S.Paged("8bit", [700, 50, 1200, 16], 4, 128, 16, BF16, seed=10 + 2 * x, room=1)
        for c in (pc.k_cache, pc.v_cache):
            u = c.view(torch.uint8)
            u[(u & 0x7f) == 0x7f] = 0
        g = torch.Generator().manual_seed(x)
        q = torch.randn(4, 1, 16, 128, generator=g).bfloat16().to(DEV)
        k, v = (torch.randn(4, 1, 4, 128, generator=g).bfloat16().to(DEV) for _ in range(2))
        call = lambda pc=pc, q=q, k=k, v=v: C.flash_attn_with_kvcache(  # noqa: E731
            q, pc.k_cache, pc.v_cache, k=k, v=v, cache_seqlens=pc.L, page_table=pc.bt, **pc.opts())
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            out = call()
        steps.append((pc, q, k, v, call, s, graph, out))
    for r in range(3):
        g = torch.Generator().manual_seed(100 + r)
        for pc, q, k, v, call, s, graph, out in steps:
            for t in (q, k, v):
                t.copy_(torch.randn(t.shape, generator=g).bfloat16())
        torch.cuda.synchronize()
        for _ in range(5):
            for pc, q, k, v, call, s, graph, out in steps:
                with torch.cuda.stream(s):
                    graph.replay()
        torch.cuda.synchronize()
        for pc, q, k, v, call, s, graph, out in steps:
            assert torch.equal(out, call())


def test_decode_graphs_of_one_stream_on_two():
    """Two graphs captured on the same stream, replayed at once on two others: each has buffers of its own."""
    C = api()
    s = torch.cuda.Stream()
    runs = []
    for x in range(2):
        pc = S.Paged("8bit", [3000, 70, 900], 2, 64, 16, BF16, seed=20 + x)
        q = torch.randn(3, 1, 8, 64, generator=torch.Generator().manual_seed(x)).bfloat16().to(DEV)
        call = lambda pc=pc, q=q: C.flash_attn_with_kvcache(q, pc.k_cache, pc.v_cache, cache_seqlens=pc.L,  # noqa
                                                            page_table=pc.bt, window_size=(2000, 0), sink_tokens=5,
                                                            **pc.opts())
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            out = call()
        runs.append((graph, out, call, torch.cuda.Stream()))  # (the graph reads what `call` holds)
    torch.cuda.synchronize()
    for _ in range(20):
        for graph, _, _, stream in runs:
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for _, out, call, _ in runs:
        assert torch.equal(out, call())


def test_offsets_past_32_bits():
    """Blocks more than 2^32 bytes into 8-bit caches: written, read, copied and packed in place."""
    C = api()
    blocks, hk, page, d = 280000, 8, 16, 128  # 4.6e9 bytes a side
    kc, vc = (torch.zeros(blocks, hk, page, d, dtype=torch.uint8, device=DEV).view(S.F8) for _ in range(2))
    ks, vs = (torch.zeros(blocks, hk, device=DEV) for _ in range(2))
    g = torch.Generator().manual_seed(0)
    ids = [blocks - 1, 3, blocks - 7]
    table = torch.tensor([ids], dtype=torch.int32, device=DEV)
    L = torch.zeros(1, dtype=torch.int32, device=DEV)
    k, v = (torch.randn(1, 40, hk, d, generator=g).bfloat16().to(DEV) for _ in range(2))
    C.append_quantized(k, v, kc, vc, ks, vs, L, table)
    small = [t[ids].contiguous() for t in (kc.view(torch.uint8), vc.view(torch.uint8), ks, vs)]
    q = torch.randn(1, 1, 16, d, generator=g).bfloat16().to(DEV)
    want = C.flash_attn_with_kvcache(q, small[0].view(S.F8), small[1].view(S.F8), cache_seqlens=40,
                                     page_table=torch.tensor([[0, 1, 2]], dtype=torch.int32, device=DEV),
                                     k_descale=small[2], v_descale=small[3])
    ref, *_ = S.attention(q[0, 0, :2].double().cpu(), k[0, :, 0].double().cpu(), v[0, :, 0].double().cpu(),
                          torch.ones(2, 40, dtype=torch.bool), d ** -0.5)
    assert (want[0, 0, :2].double().cpu() - ref).abs().max() < 0.3  # the tokens, to 8 bits
    caches = [kc, vc, ks, vs]
    for step in range(3):
        got = C.flash_attn_with_kvcache(q, kc, vc, cache_seqlens=40, page_table=table, k_descale=ks, v_descale=vs)
        assert torch.equal(got, want), step
        if step == 0:
            C.copy_blocks(caches, torch.tensor([[blocks - 1, 100], [3, blocks - 2], [blocks - 7, blocks - 9]], device=DEV))
            table = torch.tensor([[100, blocks - 2, blocks - 9]], dtype=torch.int32, device=DEV)
        elif step == 1:
            table, used = C.compact_blocks(caches, table, torch.tensor([40], dtype=torch.int32, device=DEV), page)
            assert used.tolist() == [3] and sorted(table[0].tolist()) == [0, 1, 2]
    assert status() == 0


def test_strides_of_sizes_of_one():
    """One head, one token, one sequence: such a dim's stride may be anything."""
    C = api()
    g = torch.Generator().manual_seed(3)
    pc = S.Paged("8bit", [20], 1, 64, 16, BF16, seed=2, room=1)
    for c in (pc.k_cache, pc.v_cache):
        u = c.view(torch.uint8)
        u[(u & 0x7f) == 0x7f] = 0
    k, v = (torch.randn(1, 1, 1, 64, generator=g).bfloat16().to(DEV) for _ in range(2))
    q = torch.randn(1, 1, 1, 64, generator=g).bfloat16().to(DEV)
    want = C.flash_attn_with_kvcache(q, pc.k_cache, pc.v_cache, k=k, v=v, cache_seqlens=pc.L, page_table=pc.bt,
                                     **pc.opts())
    odd = lambda t: torch.as_strided(t, (1, 1, 1, 64), (3, 7, 5, 1))  # noqa: E731
    got = C.flash_attn_with_kvcache(odd(q), pc.k_cache, pc.v_cache, k=odd(k), v=odd(v), cache_seqlens=pc.L,
                                    page_table=pc.bt, **pc.opts())
    assert torch.equal(got, want)
    before = [bytes_of(c) for c in (pc.k_cache, pc.v_cache)]
    cu = torch.tensor([0, 1], dtype=torch.int32, device=DEV)
    for key, value in ((odd(k)[0], odd(v)[0]), (k[0], v[0])):
        C.append_quantized(key, value, pc.k_cache, pc.v_cache, pc.k_scale, pc.v_scale, pc.L, pc.bt, cu, 1)
        assert all(torch.equal(bytes_of(c), b) for c, b in zip((pc.k_cache, pc.v_cache), before))
    assert torch.equal(want, C.flash_attn_with_kvcache(q, pc.k_cache, pc.v_cache, cache_seqlens=pc.L + 1,
                                                       page_table=pc.bt, **pc.opts()))


def test_caches_at_an_odd_address_are_refused():
    C = api()
    raw = torch.zeros(4 * 16 * 64 + 16, dtype=torch.uint8, device=DEV)
    off = raw[4:4 + 4 * 16 * 64].view(4, 1, 16, 64).view(S.F8)
    one = torch.ones(4, 1, device=DEV)
    q = torch.zeros(1, 1, 1, 64, dtype=BF16, device=DEV)
    bt = torch.zeros(1, 1, dtype=torch.int32, device=DEV)
    with pytest.raises(ValueError, match="16 bytes"):
        C.flash_attn_with_kvcache(q, off, off, cache_seqlens=3, page_table=bt, k_descale=one, v_descale=one)
    with pytest.raises(ValueError, match="16 bytes"):
        C.append_quantized(q, q, off, off, one, one.clone(), torch.zeros(1, dtype=torch.int32, device=DEV), bt)


def test_empty_calls():
    """No sequences, no new tokens, tables of no pages."""
    C = api()
    kc, vc, ks, vs = empty_8bit(4, 2, 16, 64, 0)
    no = torch.zeros(0, dtype=torch.int32, device=DEV)
    q0 = torch.zeros(0, 1, 4, 64, dtype=BF16, device=DEV)
    out, lse = C.flash_attn_with_kvcache(q0, kc, vc, cache_seqlens=no, page_table=no.view(0, 3), k_descale=ks,
                                         v_descale=vs, return_softmax_lse=True)
    assert out.shape == q0.shape and lse.shape == (0, 4, 1)
    q = torch.ones(2, 1, 4, 64, dtype=BF16, device=DEV)
    two = torch.zeros(2, dtype=torch.int32, device=DEV)
    for table in (two.view(2, 1), no.view(2, 0)):
        new = torch.zeros(2, 0, 2, 64, dtype=BF16, device=DEV)
        out = C.flash_attn_with_kvcache(q, kc, vc, k=new, v=new, cache_seqlens=two, page_table=table, k_descale=ks,
                                        v_descale=vs)
        assert (out == 0).all()
        C.append_quantized(new, new, kc, vc, ks, vs, two, table)
    C.append_quantized(q0[:, 0, :2], q0[:, 0, :2], kc, vc, ks, vs, two, two.view(2, 1),
                       torch.zeros(3, dtype=torch.int32, device=DEV))
    pool = empty_8bit(0, 2, 16, 64, 0)
    out = C.flash_attn_with_kvcache(q, *pool[:2], cache_seqlens=two, page_table=two.view(2, 1), k_descale=pool[2],
                                    v_descale=pool[3])
    assert (out == 0).all() and (ks == 0).all() and status() == 0
    new, used = C.compact_blocks([kc], no.view(2, 0), two, 16)
    assert new.shape == (2, 0) and used.tolist() == [0]


# ------------------------------------------------------------------ prefill --
def check_prefill(out, lse, q, k, v, left, right, sinks, causal, scale=None):
    """One sequence: out [lq, h, d] against the definition. Weights enter the bf16 kernel's second product rounded to
    bf16 (2^-8), the fp32 kernel's not at all; up to 2^8 times the largest is the bf16 kernel's slack, which
    changes no relative error."""
    lq, h, d = q.shape
    lk, kv = k.shape[:2]
    scale = d ** -0.5 if scale is None else scale
    i, j = torch.arange(lq)[:, None] + lk - lq, torch.arange(lk)[None]
    r = 0 if causal else right
    seen = torch.ones(lq, lk, dtype=torch.bool)
    if left >= 0:
        seen &= (j >= i - left) | (j < sinks)
    if r >= 0:
        seen &= j <= i + r
    weight = 2.0 ** -8 if q.dtype == BF16 else 0.0
    for x in range(h):
        ref, z, spread, top = S.attention(q[:, x].double().cpu(), k[:, x * kv // h].double().cpu(),
                                          v[:, x * kv // h].double().cpu(), seen, scale)
        tol = S.bound(ref, spread, top, d, lk * 16, q.dtype, weight)
        err = (out[:, x].double().cpu() - ref).abs()
        assert (err <= tol).all(), (x, err.max().item(), (err / tol).max().item())
        if lse is not None:
            zz = lse[x].double().cpu()
            none = ~seen.any(-1)
            assert torch.equal(torch.isneginf(zz), none)
            assert ((zz - z)[~none].abs() <= 1e-4).all()


WINDOWS = [(0, 0, 0), (5, 0, 1), (64, 0, 4), (100, 30, 0), (127, -1, 130), (-1, 10, 3), (300, 0, 17), (40, 0, 1000),
           (0, 300, 5)]


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("left,right,sinks", WINDOWS)
@pytest.mark.parametrize("lq,lk,h,hk,d", [(1, 1, 1, 1, 64), (300, 300, 2, 1, 128), (77, 640, 2, 2, 64),
                                          (700, 513, 2, 2, 32), (1100, 1100, 1, 1, 64)])
def test_prefill_window(dtype, left, right, sinks, lq, lk, h, hk, d):
    g = torch.Generator().manual_seed(lq + left)
    q = torch.randn(2, lq, h, d, generator=g).to(dtype).to(DEV)
    k, v = (torch.randn(2, lk, hk, d, generator=g).to(dtype).to(DEV) for _ in range(2))
    for causal in (False, True):
        out, lse = api().flash_attn_func(q, k, v, causal=causal, window_size=(left, right), sink_tokens=sinks,
                                         return_attn_probs=True)
        for b in range(2):
            check_prefill(out[b], lse[b], q[b], k[b], v[b], left, right, sinks, causal)
        assert torch.equal(out, api().flash_attn_func(q, k, v, causal=causal, window_size=(left, right),
                                                      sink_tokens=sinks))
    assert status() == 0


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("left,right,sinks", [(16, 0, 4), (200, 0, 0), (60, 60, 140)])
def test_prefill_window_packed(dtype, left, right, sinks):
    """Packed sequences, one empty: each equals a dense call on it alone, bit for bit; a layout TMA cannot read too."""
    C = api()
    lens = [1, 300, 0, 77, 520]
    g = torch.Generator().manual_seed(left)
    t, h, hk, d = sum(lens), 4, 2, 64
    cu = torch.tensor([sum(lens[:i]) for i in range(6)], dtype=torch.int32, device=DEV)
    wide = torch.randn(t, h + 2 * hk, d + 4, generator=g).to(dtype).to(DEV)
    for q, k, v in ((wide[:, :h, :d].contiguous(), wide[:, h:h + hk, :d].contiguous(), wide[:, h + hk:, :d].contiguous()),
                    (wide[:, :h, 1:d + 1], wide[:, h:h + hk, 1:d + 1], wide[:, h + hk:, 1:d + 1])):
        for causal in (True, False):
            opts = dict(causal=causal, window_size=(left, right), sink_tokens=sinks, return_attn_probs=True)
            out, lse = C.flash_attn_varlen_func(q, k, v, cu, cu, 520, 520, **opts)
            for i, n in enumerate(lens):
                if n == 0:
                    continue
                a, z = int(cu[i]), int(cu[i + 1])
                check_prefill(out[a:z], lse[:, a:z], q[a:z], k[a:z], v[a:z], left, right, sinks, causal)
                dense, dl = C.flash_attn_func(q[a:z][None], k[a:z][None], v[a:z][None], **opts)
                assert torch.equal(out[a:z], dense[0]) and torch.equal(lse[:, a:z], dl[0])


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("causal,left,right,sinks", [(True, 40, 0, 4), (False, 130, 20, 0), (False, -1, 300, 1)])
def test_prefill_window_packed_rows_of_others(dtype, hd, causal, left, right, sinks):
    """What another sequence's rows, or padding behind the last one, hold (NaN, infinities) reaches no output."""
    C = api()
    lens, pad = [5, 130, 1, 300, 128, 77], 60
    g = torch.Generator().manual_seed(hd)
    t = sum(lens) + pad
    cu = torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device=DEV)
    q, k, v = (torch.randn(t, n, hd, generator=g).to(dtype).to(DEV) for n in (4, 2, 2))
    opts = dict(causal=causal, window_size=(left, right), sink_tokens=sinks, return_attn_probs=True)
    want, want_lse = C.flash_attn_varlen_func(q, k, v, cu, cu, 300, 300, **opts)
    for bad in (1, 3, 5):  # the even sequences and the padding; the padding alone
        kept = torch.zeros(t, dtype=torch.bool, device=DEV)
        for i, n in enumerate(lens):
            if i % 2 or bad == 5:
                kept[int(cu[i]):int(cu[i + 1])] = True
        kk, vv = k.clone(), v.clone()
        kk[~kept] = math.nan
        vv[~kept] = (math.nan, math.inf, -math.inf)[bad // 2]
        out, lse = C.flash_attn_varlen_func(q, kk, vv, cu, cu, 300, 300, **opts)
        assert torch.equal(out[kept], want[kept]) and torch.equal(lse[:, kept], want_lse[:, kept])


def test_prefill_window_that_hides_nothing():
    """A window as long as the sequences gives the result of no window (fp32: the same tiles, the same bits)."""
    g = torch.Generator().manual_seed(0)
    for dtype in (BF16, FP32):
        q, k, v = (torch.randn(1, 400, 2, 64, generator=g).to(dtype).to(DEV) for _ in range(3))
        plain = api().flash_attn_func(q, k, v, causal=True)
        wide = api().flash_attn_func(q, k, v, causal=True, window_size=(10 ** 12, 0), sink_tokens=3)
        assert torch.equal(plain, wide)
        assert torch.equal(plain, api().flash_attn_func(q, k, v, causal=True, sink_tokens=7))


# -------------------------------------------------------------- block moves --
def layer_caches(blocks, layers, g, page=16):
    out = []
    for _ in range(layers):
        out += [torch.randn(blocks, 2, page, 32, generator=g).bfloat16().to(DEV),
                torch.randn(blocks, 2, page, 64, generator=g).to(S.F8).to(DEV),
                torch.randn(blocks, 3, generator=g).to(DEV), torch.randint(0, 9, (blocks,), generator=g).to(DEV),
                torch.randint(0, 255, (blocks, 7), generator=g).to(torch.uint8).to(DEV)]
    return out


@pytest.mark.parametrize("layers", [1, 30])
def test_copy_blocks(layers):
    g = torch.Generator().manual_seed(layers)
    caches = layer_caches(40, layers, g)
    before = [bytes_of(c) for c in caches]
    pairs = torch.tensor([[3, 9], [3, 10], [-1, 4], [5, -7], [0, 39], [8, 8 + 12]], dtype=torch.int64)
    for where in (DEV, "cpu"):
        api().copy_blocks(caches, pairs.to(where))
        for c, was in zip(caches, before):
            now, want = bytes_of(c), was.clone()
            for a, b in pairs.tolist():
                if a >= 0 and b >= 0:
                    want[b] = was[a]
            assert torch.equal(now, want)
    status()
    api().copy_blocks(caches, torch.tensor([[1, 40], [1 << 40, 2], [6, 7]], device=DEV))
    assert status() == kernel().STATUS_SLOT
    assert torch.equal(bytes_of(caches[0])[7], before[0][6]) and torch.equal(bytes_of(caches[0])[2], before[0][2])
    api().copy_blocks(caches, torch.zeros(0, 2, dtype=torch.int64, device=DEV))
    api().copy_blocks([], torch.zeros(0, 2, dtype=torch.int64, device=DEV))
    api().copy_blocks(caches[0], torch.tensor([[0, 1]], device=DEV))
    assert torch.equal(bytes_of(caches[0])[1], before[0][0])


def plain_compact(table, lens, page, blocks, left, sinks):
    live = [[p * page < n and (left < 0 or (p + 1) * page > n - 1 - left or p * page < sinks) for p in range(len(row))]
            for row, n in zip(table, lens)]
    used = {b for row, on in zip(table, live) for b, x in zip(row, on) if x and 0 <= b < blocks}
    free = [b for b in range(len(used)) if b not in used]
    moves = dict(zip(sorted(b for b in used if b >= len(used)), free))
    new = [[moves.get(b, b) if x and 0 <= b < blocks else -1 for b, x in zip(row, on)]
           for row, on in zip(table, live)]
    return new, len(used), moves


@pytest.mark.parametrize("blocks,batch,width,left,sinks", [(50, 6, 5, -1, 0), (1000, 7, 40, 100, 4), (33, 1, 1, -1, 0),
                                                           (40000, 20, 1500, 300, 33), (64, 5, 9, 0, 0)])
def test_compact_blocks(blocks, batch, width, left, sinks):
    g = torch.Generator().manual_seed(blocks)
    page = 16
    caches = layer_caches(blocks, 1, g)
    before = [bytes_of(c) for c in caches]
    table = torch.randperm(blocks, generator=g)
    table = table[torch.randint(0, blocks, (batch, width), generator=g)] if batch * width > blocks // 2 else \
        table[:batch * width].reshape(batch, width)
    lens = torch.randint(0, width * page + 1, (batch,), generator=g)
    if batch > 2:
        table[1, :3] = table[0, :3]  # shared
    table, lens = table.to(torch.int32), lens.to(torch.int32)
    new, used = api().compact_blocks(caches, table.to(DEV), lens.to(DEV), page, window_size=(left, 0), sink_tokens=sinks)
    want, n, moves = plain_compact(table.tolist(), lens.tolist(), page, blocks, left, sinks)
    assert used.tolist() == [n] and new.tolist() == want
    for c, was in zip(caches, before):
        ref = was.clone()
        for a, b in moves.items():
            ref[b] = was[a]
        assert torch.equal(bytes_of(c), ref)
    # packed already: nothing moves
    again, used = api().compact_blocks(caches, new, lens.to(DEV), page, window_size=(left, 0), sink_tokens=sinks)
    assert torch.equal(again, new) and used.tolist() == [n]


def test_compact_flags_bad_entries():
    K = kernel()
    g = torch.Generator().manual_seed(0)
    caches = layer_caches(10, 1, g)
    table = torch.tensor([[9, 99], [-2, 8]], dtype=torch.int32, device=DEV)
    status()
    new, used = api().compact_blocks(caches, table, torch.tensor([20, 32], dtype=torch.int32, device=DEV), 16)
    assert status() == K.STATUS_TABLE
    assert new.tolist() == [[1, -1], [-1, 0]] and used.tolist() == [2]
    api().compact_blocks(caches, table[:1], torch.tensor([100], dtype=torch.int32, device=DEV), 16)
    assert status() & K.STATUS_LENS
    empty, used = api().compact_blocks(caches, table[:0], torch.zeros(0, dtype=torch.int32, device=DEV), 16)
    assert empty.shape == (0, 2) and used.tolist() == [0]


# ----------------------------------------------------------- a run together --
@pytest.mark.parametrize("kind", ["8bit", "bf16"])
def test_serving_run(kind):
    """Prompts enter the cache, sequences decode behind a window, one forks, the pool is packed, decoding goes on: the
    outputs are those of the same tokens attended in float64, whatever moved."""
    C = api()
    g = torch.Generator().manual_seed(5)
    h, hk, d, page, left, sinks = 8, 2, 64, 16, 40, 4
    lens = [70, 5, 33]
    width, blocks = 16, 80
    table = torch.full((4, width), -1, dtype=torch.int32)
    free = torch.randperm(blocks, generator=g).tolist()
    if kind == "8bit":
        kc, vc, ks, vs = empty_8bit(blocks, hk, page, d, 0)
        caches = [kc, vc, ks, vs]
        opts = dict(k_descale=ks, v_descale=vs)
    else:
        kc, vc = (torch.zeros(blocks, hk, page, d, dtype=BF16, device=DEV) for _ in range(2))
        caches, opts = [kc, vc], {}

    def grow(i, n):
        for p in range(-(-n // page)):
            if table[i, p] < 0 and (p * page < sinks or (p + 1) * page > n - 1 - left):
                table[i, p] = free.pop()

    hist = [[torch.randn(n, hk, d, generator=g).bfloat16() for _ in range(2)] for n in lens]
    for i, n in enumerate(lens):
        for p in range(-(-n // page)):
            table[i, p] = free.pop()
    cu = torch.tensor([0, 70, 75, 108], dtype=torch.int32, device=DEV)
    key, value = (torch.cat([x[s] for x in hist]).to(DEV) for s in range(2))
    if kind == "8bit":
        C.append_quantized(key, value, kc, vc, ks, vs, torch.zeros(3, dtype=torch.int32, device=DEV),
                           table[:3].to(DEV), cu, 70)
    else:
        pos = torch.cat([torch.arange(n) for n in lens])
        seq = torch.cat([torch.full((n,), i) for i, n in enumerate(lens)])
        C.reshape_and_cache(key, value, kc, vc, (table[seq, pos // page].long() * page + pos % page).to(DEV))
    lens = lens + [0]
    hist.append([torch.zeros(0, hk, d).bfloat16() for _ in range(2)])
    # what 8 bits lose: a value is off by at most 2^-4 of itself, or half a step of the smallest code's unit; three
    # scale growths at most (each rounds small codes again). Bounded here against the tokens themselves.
    for step in range(50):
        if step == 20:  # sequence 3 forks sequence 0: whole pages shared, the open one copied
            open_page = lens[0] // page
            table[3] = table[0]
            if lens[0] % page:
                fresh = free.pop()
                C.copy_blocks(caches, torch.tensor([[int(table[0, open_page]), fresh]], device=DEV))
                table[3, open_page] = fresh
            lens[3], hist[3] = lens[0], [x.clone() for x in hist[0]]
        if step == 35:  # free what the window has left, pack the rest
            L = torch.tensor(lens, dtype=torch.int32, device=DEV)
            new, used = C.compact_blocks(caches, table.to(DEV), L, page, window_size=(left, 0), sink_tokens=sinks)
            table = new.cpu()
            free = list(range(int(used), blocks))
            assert int(used) < 30
        rows = [0, 1, 2] if step < 20 else [0, 1, 2, 3]
        for i in rows:
            grow(i, lens[i] + 1)
        q = torch.randn(len(rows), 1, h, d, generator=g).bfloat16()
        k, v = (torch.randn(len(rows), 1, hk, d, generator=g).bfloat16() for _ in range(2))
        out = C.flash_attn_with_kvcache(q.to(DEV), kc, vc, k=k.to(DEV), v=v.to(DEV),
                                        cache_seqlens=torch.tensor([lens[i] for i in rows], dtype=torch.int32,
                                                                   device=DEV),
                                        page_table=table[rows].to(DEV), window_size=(left, 0), sink_tokens=sinks, **opts)
        for x, i in enumerate(rows):
            hist[i] = [torch.cat([hist[i][0], k[x]]), torch.cat([hist[i][1], v[x]])]
            lens[i] += 1
            if step % 7 and step not in (20, 35, 36):
                continue
            pos = torch.tensor(S.seen_decode(lens[i], left, sinks))
            for a in range(hk):
                kk, vv = (hist[i][s][pos, a].double() for s in range(2))
                qq = q[x, 0, a * 4:(a + 1) * 4].double()
                ref, _, spread, top = S.attention(qq, kk, vv, torch.ones(4, len(pos), dtype=torch.bool), d ** -0.5)
                # scores move by at most (2^-4 + growth) of sum |q||k|; each weight by the exponential of twice that;
                # values by 2^-4 of themselves plus two units of the smallest step of a block of N(0, 1) values
                eight = kind == "8bit"
                shift = top * 1.1 * 2 ** -4 if eight else torch.zeros_like(top)
                tol = S.bound(ref, spread, top, d, len(pos), BF16, 2.0 ** -11 if eight else 2.0 ** -16)
                tol = tol + (spread + 0.05) * (torch.expm1(2 * shift)[:, None] + (2 ** -4 if eight else 0)) + 1e-3
                err = (out[x, 0, a * 4:(a + 1) * 4].double().cpu() - ref).abs()
                assert (err <= tol).all(), (step, i, err.max().item())
    assert status() == 0


@pytest.mark.parametrize("kind", ["8bit", "bf16", "fp32"])
@pytest.mark.parametrize("left,sinks", [(63, 0), (30, 20), (-1, 0)])
def test_compact_keeps_what_is_seen_and_reserved(kind, left, sinks):
    """Lengths reserved ahead keep their pages; the window stays the one of the tokens that are there, so the next
    decode answers as if nothing had moved."""
    C = api()
    h, hk, d, page, ahead = 4, 2, 64, 16, 64
    dtype = FP32 if kind == "fp32" else BF16
    lens = [100, 3, 0, 256, 31, -1]
    pc = S.Paged(kind, lens, hk, d, page, dtype, seed=left + 71, room=ahead)
    pc.left, pc.sinks = left, sinks
    caches = [t for t in (pc.k_cache, pc.v_cache, pc.k_scale, pc.v_scale) if t is not None]
    reserved = [n + ahead for n in lens[:4]] + [2, ahead]  # (below the length: the length counts)
    q = torch.randn(len(lens), 1, h, d, generator=torch.Generator().manual_seed(1)).to(dtype).to(DEV)
    opts = dict(window_size=(left, 0), sink_tokens=sinks)
    want = C.flash_attn_with_kvcache(q, pc.k_cache, pc.v_cache, cache_seqlens=pc.L, page_table=pc.bt, **pc.opts(), **opts)
    S.check_decode(want, None, q, pc, h)
    old = pc.bt.tolist()
    keep = [[n >= 0 and p * page < max(n, r) and (left < 0 or (p + 1) * page > n - 1 - left or p * page < sinks)
             for p in range(len(row))] for row, n, r in zip(old, lens, reserved)]
    used_ids = {b for row, on in zip(old, keep) for b, x in zip(row, on) if x}
    free = [b for b in range(len(used_ids)) if b not in used_ids]
    moves = dict(zip(sorted(b for b in used_ids if b >= len(used_ids)), free))
    reserved = torch.tensor(reserved, dtype=torch.int32)
    for where in (DEV, "cpu"):  # the second call finds everything packed
        table, used = C.compact_blocks(caches, pc.bt, pc.L, page, reserved_seqlens=reserved.to(where), **opts)
        if where == DEV:
            assert table.tolist() == [[moves.get(b, b) if x else -1 for b, x in zip(row, on)]
                                      for row, on in zip(old, keep)]
            first = table
        else:
            assert torch.equal(table, first)
        assert used.tolist() == [len(used_ids)]
        pc.bt = table
        got = C.flash_attn_with_kvcache(q, pc.k_cache, pc.v_cache, cache_seqlens=pc.L, page_table=table, **pc.opts(),
                                        **opts)
        assert torch.equal(got, want)
    assert status() == 0
    # the ctypes path answers the same
    from cpu_attention import _kernel as K, _native
    fast, K._FAST = K.fastpath(), False
    try:
        again, n = _native.compact_blocks(0, caches, pc.bt, pc.L, page, left, sinks, reserved.to(DEV))
    finally:
        K._FAST = fast
    assert torch.equal(again, first) and n.tolist() == used.tolist()
    C.compact_blocks(caches, pc.bt, pc.L, page, reserved_seqlens=reserved.to(DEV) + 10000, **opts)
    assert status() & kernel().STATUS_LENS


def test_step_example_keeps_the_new_token():
    """The integration guide's decode step with a compaction behind it, with lengths that end at a page: the next step finds
    every token."""
    from test_serving_api import step_example
    C = api()
    lens, page, width = [16, 32, 5, 0, 47], 16, 4
    kc, vc, ks, vs = empty_8bit(40, 2, page, 64, 0)
    g = torch.Generator().manual_seed(8)
    table = torch.randperm(40, generator=g)[:5 * width].reshape(5, width).to(torch.int32).to(DEV)
    hist = [torch.randn(5, 48, 2, 64, generator=g).bfloat16().to(DEV) for _ in range(2)]
    names = dict(k_cache=kc, v_cache=vc, k_scale=ks, v_scale=vs, page=page, table=table)
    for i, n in enumerate(lens):  # the tokens before
        C.append_quantized(hist[0][i:i + 1, :n], hist[1][i:i + 1, :n], kc, vc, ks, vs,
                           torch.zeros(1, dtype=torch.int32, device=DEV), table[i:i + 1])
    before = [t.clone() for t in (kc.view(torch.uint8), vc.view(torch.uint8), ks, vs)]
    L = torch.tensor(lens, dtype=torch.int32, device=DEV)
    q = torch.randn(5, 1, 4, 64, generator=g).bfloat16().to(DEV)
    k, v = (torch.randn(5, 1, 2, 64, generator=g).bfloat16().to(DEV) for _ in range(2))
    exec(step_example(), names | dict(q=q, k=k, v=v, lens=L.clone()), names)
    again = C.flash_attn_with_kvcache(q, kc, vc, cache_seqlens=L + 1, page_table=names["table"], k_descale=ks,
                                      v_descale=vs, window_size=(4095, 0), sink_tokens=4)
    assert torch.equal(again, names["out"])
    want = C.flash_attn_with_kvcache(q, before[0].view(S.F8), before[1].view(S.F8), k=k, v=v, cache_seqlens=L,
                                     page_table=table, k_descale=before[2], v_descale=before[3])
    assert torch.equal(again, want) and status() == 0
    assert int(names["used"]) == sum(-(-(n + 1) // page) for n in lens)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("hd", [32, 64, 128])
@pytest.mark.parametrize("causal", [True, False])
def test_prefill_packed_rows_of_others(dtype, hd, causal):
    """Without a window too, what another sequence's rows, or padding behind the last one, hold (NaN, infinities)
    reaches no output; queries and keys of different lengths, one sequence without keys."""
    C = api()
    lq, lk, pad = [5, 130, 1, 300, 128, 77, 3], [9, 130, 257, 300, 128, 40, 0], 60
    g = torch.Generator().manual_seed(hd)
    cq, ck = (torch.tensor([sum(n[:i]) for i in range(len(n) + 1)], dtype=torch.int32, device=DEV) for n in (lq, lk))
    q = torch.randn(sum(lq), 4, hd, generator=g).to(dtype).to(DEV)
    k, v = (torch.randn(sum(lk) + pad, 2, hd, generator=g).to(dtype).to(DEV) for _ in range(2))
    call = lambda kk, vv: C.flash_attn_varlen_func(q, kk, vv, cq, ck, 300, 300, causal=causal,  # noqa: E731
                                                   return_attn_probs=True)
    want, want_lse = call(k, v)
    assert torch.isfinite(want).all()
    for bad in (math.nan, math.inf, -math.inf):
        for keep in (0, 1, 2):  # the sequences of an even index, of an odd one, all of them
            rows_q, rows_k = (torch.zeros(n, dtype=torch.bool, device=DEV) for n in (q.shape[0], k.shape[0]))
            for i in range(len(lq)):
                if keep == 2 or i % 2 == keep:
                    rows_q[int(cq[i]):int(cq[i + 1])] = True
                    rows_k[int(ck[i]):int(ck[i + 1])] = True
            kk, vv = k.clone(), v.clone()
            kk[~rows_k] = math.nan
            vv[~rows_k] = bad
            out, lse = call(kk, vv)
            assert torch.equal(out[rows_q], want[rows_q]) and torch.equal(lse[:, rows_q], want_lse[:, rows_q])
    assert status() == 0


@pytest.mark.parametrize("kind", ["8bit", "bf16", "fp32"])
@pytest.mark.parametrize("n,left,sinks", [(60, 20, 4), (100, 0, 0), (33, 15, 17), (200, 70, 40)])
def test_decode_appends_more_than_the_window(kind, n, left, sinks):
    """New tokens that are behind the window at once: stored where the table names their page, left out where the page
    is freed already (an entry outside the pool); the row is the same, and nothing is flagged."""
    C = api()
    lens, h, hk, d, page = [0, 15, 16, 100, 31], 4, 2, 64, 16
    dtype = FP32 if kind == "fp32" else BF16
    pc = S.Paged(kind, lens, hk, d, page, dtype, seed=n, room=n)
    for c in (pc.k_cache, pc.v_cache) if kind == "8bit" else ():
        u = c.view(torch.uint8)
        u[(u & 0x7f) == 0x7f] = 0
    g = torch.Generator().manual_seed(n)
    k, v = (torch.randn(len(lens), n, hk, d, generator=g).to(dtype).to(DEV) for _ in range(2))
    q = torch.randn(len(lens), 1, h, d, generator=g).to(dtype).to(DEV)
    opts = dict(window_size=(left, 0), sink_tokens=sinks)
    start = [t for t in (pc.k_cache, pc.v_cache, pc.k_scale, pc.v_scale) if t is not None]
    names = ["k_cache", "v_cache", "k_descale", "v_descale"][:len(start)]
    outs, ends = [], []
    table = pc.bt.clone()
    freed = torch.zeros(table.shape, dtype=torch.bool)
    for i, m in enumerate(lens):
        for p in range(table.shape[1]):
            freed[i, p] = p * page >= sinks and (p + 1) * page <= m + n - 1 - left
    for bad in (None, -1, 0x7fffffff):
        bt = table if bad is None else table.masked_fill(freed.to(DEV), bad)
        caches = dict(zip(names, [t.clone() for t in start]))
        outs.append(C.flash_attn_with_kvcache(q, k=k, v=v, cache_seqlens=pc.L, page_table=bt, **caches, **opts))
        assert status() == 0
        ends.append([bytes_of(t) for t in caches.values()])
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])
    # with every page named, all tokens are there: a longer window finds them
    stored = dict(zip(names, [t.clone() for t in start]))
    full = C.flash_attn_with_kvcache(q, k=k, v=v, cache_seqlens=pc.L, page_table=table, **stored,
                                     **({} if kind == "8bit" else dict(sink_tokens=0)))
    assert all(torch.equal(a, bytes_of(b)) for a, b in zip(ends[0], stored.values()))
    assert torch.isfinite(full).all()
    # what is left out: the freed pages keep what they held
    gone = table[freed.to(DEV)].long().cpu()
    for a, b, was in zip(ends[1], ends[2], start):
        assert torch.equal(a, b) and torch.equal(a[gone], bytes_of(was)[gone])
    kept = torch.ones(start[0].shape[0], dtype=torch.bool)
    kept[gone] = False
    assert all(torch.equal(a[kept], b[kept]) for a, b in zip(ends[0], ends[1]))
    # a bad entry of a page that is seen is flagged as ever
    first = (lens[3] + n - 1) // page
    table[3, first] = -1
    C.flash_attn_with_kvcache(q, k=k, v=v, cache_seqlens=pc.L, page_table=table,
                              **dict(zip(names, [t.clone() for t in start])), **opts)
    assert status() == kernel().STATUS_TABLE


# ------------------------------------------------ scales of a user's own -----
@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("own", [False, True])
@pytest.mark.parametrize("d,page,h,hk", [(32, 16, 4, 4), (64, 64, 6, 2), (128, 16, 8, 1), (128, 48, 20, 2)])
def test_decode_8bit_even_weights(dtype, own, d, page, h, hk):
    """Scores a few units apart, so that outputs are sums over many keys and joins carry weight; scales that are powers
    of two and ones that are not."""
    lens = LENS + [4100]
    pc = S.Paged("8bit", lens, hk, d, page, dtype, seed=d + page, own=own, even=True)
    assert own == bool((torch.frexp(pc.scale[0])[0] != 0.5).any())
    q = torch.randn(len(lens), 1, h, d, generator=torch.Generator().manual_seed(h)).to(dtype).to(DEV)
    out, lse = api().flash_attn_with_kvcache(q, pc.k_cache, pc.v_cache, cache_seqlens=pc.L, page_table=pc.bt,
                                             return_softmax_lse=True, **pc.opts())
    S.check_decode(out, lse, q, pc, h)
    assert status() == 0


def check_append_own(cache, scale, codes, scales, rows, lens, table, page):
    """One append where scales need not be powers of two: scales exactly, codes as near as the definition's roundings.
    A quotient x / s, or a ratio and its product with a code, is rounded to fp32 (half a step 2^-24 each) before it is
    rounded to a code: the code is within half a code's step, and 2^-23 of itself, of the exact quotient."""
    want = codes.clone(), scales.clone()
    exact = codes.clone()
    for i, n in enumerate(lens):
        r = rows[i]
        for p in range(n // page, -(-(n + r.shape[0]) // page)):
            a, z = max(n, p * page), min(n + r.shape[0], (p + 1) * page)
            b = table[i][p]
            for x in range(codes.shape[1]):
                old = 0.0 if a == p * page else scales[b, x].item()
                now = max(old, S.fit_scale(r[a - n:z - n, x]))
                want[1][b, x] = now
                if a != p * page and now != old:
                    exact[b, x] = codes[b, x] * old / now
                exact[b, x, a - p * page:z - p * page] = r[a - n:z - n, x] / now
    got = cache.cpu().double()
    _, e = torch.frexp(exact)
    half = torch.exp2((e - 5).clamp(min=-10).double())  # of the step at the exact value
    half = torch.where(exact.abs() > 448, math.inf, half)
    assert torch.equal(scale.cpu().double(), want[1])
    err = (got - exact).abs()
    assert (err <= half + exact.abs() * 2.0 ** -23).all(), (err - half).max().item()
    return got, want[1]


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("d,page", [(128, 16), (64, 32), (32, 48)])
@pytest.mark.parametrize("packed", [False, True])
def test_append_to_scales_of_a_users_own(dtype, d, page, packed):
    """Calibrated scales stay while they are large enough and codes are rounded to them; where they are too small the
    scale grows and the block's codes are rounded by a ratio that is no power of two; the row attended is the cache's."""
    g = torch.Generator().manual_seed(d + packed)
    heads, lens, width = 3, [5, page - 1, 2 * page - 3, page, 3], 4
    table = torch.randperm(5 * width + 2, generator=g)[:5 * width].reshape(5, width).to(torch.int32)
    blocks = 5 * width + 2
    caches = [S.round_e4m3(torch.randn(blocks, heads, page, d, generator=g, dtype=torch.float64) * 100) for _ in range(2)]
    scales = [torch.rand(blocks, heads, generator=g).mul(0.4).add(0.03).double() for _ in range(2)]
    scales[0][table[0][0]] = torch.tensor([0.37, 1e-3, 3e-38]).double()  # kept, grown, grown from next to nothing
    scales[1][table[1][0]] = torch.tensor([1e30, 0.0, 0.37]).double()
    scales = [s.float().double() for s in scales]
    kc, vc = (c.float().to(S.F8).to(DEV) for c in caches)
    ks, vs = (s.float().to(DEV) for s in scales)
    for n, size in ((1, 1.0), (3, 30.0), (page + 2, 3000.0)):
        k, v = (torch.randn(5, n, heads, d, generator=g).mul(size).to(dtype) for _ in range(2))
        more = {}
        args = (k.to(DEV), v.to(DEV))
        if packed:
            args = tuple(t.flatten(0, 1) for t in args)
            more = dict(cu_seqlens_new=torch.arange(0, 5 * n + 1, n, dtype=torch.int32, device=DEV), max_seqlen_new=n)
        api().append_quantized(*args, kc, vc, ks, vs, torch.tensor(lens, dtype=torch.int32, device=DEV), table.to(DEV),
                               **more)
        for x, (r, c, s) in enumerate(((k, kc, ks), (v, vc, vs))):
            caches[x], scales[x] = check_append_own(c, s, caches[x], scales[x], [t.double() for t in r], lens,
                                                    table.tolist(), page)
        lens = [a + n for a in lens]
    assert status() == 0
    q = torch.randn(5, 1, 6, d, generator=g).to(dtype).to(DEV)
    pc = S.Paged("8bit", lens, heads, d, page, dtype, own=True)
    pc.table, pc.rows, pc.scale = table.tolist(), caches, scales
    out, lse = api().flash_attn_with_kvcache(q, kc, vc, cache_seqlens=torch.tensor(lens, dtype=torch.int32, device=DEV),
                                             page_table=table.to(DEV), k_descale=ks, v_descale=vs, softmax_scale=1e-3,
                                             return_softmax_lse=True)
    S.check_decode(out, lse, q, pc, 6, scale=1e-3)


def test_append_packed_stated_maximum():
    """The stated longest sequence may be any number: too small a one is flagged (0, too), a huge one is no limit."""
    C, K = api(), kernel()
    g = torch.Generator().manual_seed(4)
    k, v = (torch.randn(20, 2, 64, generator=g).bfloat16().to(DEV) for _ in range(2))
    cu = torch.tensor([0, 5, 20], dtype=torch.int32, device=DEV)
    L = torch.zeros(2, dtype=torch.int32, device=DEV)
    table = torch.tensor([[2, 0], [1, 3]], dtype=torch.int32, device=DEV)
    want = empty_8bit(4, 2, 16, 64, 0)
    C.append_quantized(k, v, *want, L, table, cu)
    assert status() == 0 and (want[2] > 0).sum() == 4
    for most, flag in ((15, 0), (1 << 40, 0), (0, K.STATUS_LENS), (4, K.STATUS_LENS)):
        got = empty_8bit(4, 2, 16, 64, 0)
        C.append_quantized(k, v, *got, L, table, cu, most)
        assert status() == flag, most
        if not flag:
            assert all(torch.equal(bytes_of(a), bytes_of(b)) for a, b in zip(got, want))
        elif most == 0:
            assert all((bytes_of(a) == 0).all() for a in got)
    with pytest.raises(ValueError):
        C.append_quantized(k, v, *want, L, table, cu, -1)
    assert status() == 0


# --------------------------------------------------- workspaces and graphs -----
def small_decode(seed):
    """A decode whose items are split (its joins use the workspace), over float caches."""
    g = torch.Generator().manual_seed(seed)
    kc, vc = (torch.randn(80, 4, 16, 64, generator=g).bfloat16().to(DEV) for _ in range(2))
    bt = torch.randperm(80, generator=g).to(torch.int32).view(2, 40).to(DEV)
    L = torch.tensor([640, 333], dtype=torch.int32, device=DEV)
    q = torch.randn(2, 1, 4, 64, generator=g).bfloat16().to(DEV)
    return lambda: api().flash_attn_with_kvcache(q, kc, vc, cache_seqlens=L, page_table=bt)


def test_workspace_made_in_a_capture_is_zero_before_the_replay():
    """A stream's first call may be a captured one: what it leaves for the calls behind it does not wait for that
    graph's first replay. Graphs of one stream give the same in any order of replay."""
    K = kernel()
    stream = torch.cuda.Stream(priority=-1)  # (of a pool that nothing here has used)
    dev = torch.device("cuda", torch.cuda.current_device())
    first, second = small_decode(1), small_decode(2)
    want = first(), second()
    torch.cuda.synchronize()
    graphs = []
    for call in (first, second):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = call()
        graphs.append((graph, out))
        assert int(K.workspace(dev, stream.cuda_stream).count_nonzero()) == 0
    with torch.cuda.stream(stream):
        assert torch.equal(second(), want[1])
        for i in (1, 0, 1):
            graphs[i][0].replay()
            assert torch.equal(graphs[i][1], want[i])
        assert status() == 0


def test_outgrown_workspace_stays_for_graphs():
    """A graph holds its workspace's address; a larger call on the stream gets a new one and the old one stays."""
    K = kernel()
    stream = torch.cuda.Stream()
    dev = torch.device("cuda", torch.cuda.current_device())
    call = small_decode(3)
    with torch.cuda.stream(stream):
        want = call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = call()
    with torch.cuda.stream(stream):
        old = K.workspace(dev, stream.cuda_stream)
        address, size = old.data_ptr(), old.numel()
        del old
        assert K.workspace(dev, stream.cuda_stream, size + 1).data_ptr() != address
        others = [torch.full((size,), 0x5a, dtype=torch.uint8, device=DEV) for _ in range(8)]
        assert all(t.data_ptr() >= address + size or t.data_ptr() + size <= address for t in others)
        for _ in range(3):
            out.zero_()
            graph.replay()
            assert torch.equal(out, want)
        assert all(bool((t == 0x5a).all()) for t in others)
        assert torch.equal(call(), want)


@pytest.mark.parametrize("kind", ["8bit", "bf16", "fp32"])
def test_decode_append_skips_negative_lengths_without_a_flag(kind):
    """A sequence left out by a negative length takes no new tokens, however many there are for it."""
    dtype = FP32 if kind == "fp32" else BF16
    pc = S.Paged(kind, [3, -1, -1], 2, 64, 16, dtype, seed=2, room=10)
    for c in (pc.k_cache, pc.v_cache) if kind == "8bit" else ():
        u = c.view(torch.uint8)
        u[(u & 0x7f) == 0x7f] = 0
    before = [bytes_of(c) for c in (pc.k_cache, pc.v_cache)]
    q = torch.ones(3, 1, 4, 64, dtype=dtype, device=DEV)
    new = torch.ones(3, 40, 2, 64, dtype=dtype, device=DEV)
    status()
    out, lse = api().flash_attn_with_kvcache(q[1:], pc.k_cache, pc.v_cache, k=new[1:], v=new[1:], cache_seqlens=pc.L[1:],
                                             page_table=pc.bt[1:], sink_tokens=0, return_softmax_lse=True, **pc.opts())
    assert status() == 0
    assert (out == 0).all() and torch.isneginf(lse).all()
    assert all(torch.equal(bytes_of(c), b) for c, b in zip((pc.k_cache, pc.v_cache), before))


# ------------------------------------------------- captured, and from threads -----
def serving_step(seed):
    """Prompts into 8-bit caches, a fork, a packing, a windowed decode with new tokens, a windowed prefill: a call of all
    of them on fixed buffers, what fills the buffers, and what the call leaves."""
    C = api()
    hk, d, page, width, news = 2, 64, 16, 6, [30, 0, 47]
    lens, total = [3, 16, 20], 77
    g = torch.Generator().manual_seed(seed)
    start = [t.to(DEV) for t in (torch.randint(0, 120, (24, hk, page, d), generator=g, dtype=torch.uint8),
                                 torch.randint(0, 120, (24, hk, page, d), generator=g, dtype=torch.uint8),
                                 torch.rand(24, hk, generator=g), torch.rand(24, hk, generator=g))]
    caches = [t.clone() for t in start]
    kc, vc = (c.view(S.F8) for c in caches[:2])
    table = torch.randperm(24, generator=g)[:18].reshape(3, width).to(torch.int32)
    spare = sorted(set(range(24)) - set(table.flatten().tolist()))
    pairs = torch.tensor([[int(table[0, 0]), spare[0]], [int(table[2, 1]), spare[1]]], device=DEV)
    cu = torch.tensor([0, 30, 30, 77], dtype=torch.int32, device=DEV)
    L = torch.tensor(lens, dtype=torch.int32, device=DEV)
    table, after = table.to(DEV), L + torch.tensor(news, dtype=torch.int32, device=DEV)
    k, v, q1, k1, v1 = (torch.empty(*s, d, dtype=BF16, device=DEV) for s in ((total, hk), (total, hk), (3, 1, 4),
                                                                             (3, 1, hk), (3, 1, hk)))
    q = torch.empty(total, 4, d, dtype=BF16, device=DEV)

    def fill(r):
        g = torch.Generator().manual_seed(1000 * seed + r)
        for t in (k, v, q, q1, k1, v1):
            t.copy_(torch.randn(t.shape, generator=g).bfloat16())
        for t, was in zip(caches, start):
            t.copy_(was)

    def call():
        C.append_quantized(k, v, kc, vc, *caches[2:], L, table, cu, 47)
        C.copy_blocks([kc, vc, *caches[2:]], pairs)
        new, used = C.compact_blocks([kc, vc, *caches[2:]], table, after, page, (40, 0), 4, after + 1)
        out = C.flash_attn_with_kvcache(q1, kc, vc, k=k1, v=v1, cache_seqlens=after, page_table=new,
                                        k_descale=caches[2], v_descale=caches[3], window_size=(40, 0), sink_tokens=4)
        pre = C.flash_attn_varlen_func(q, k, v, cu, cu, 47, 47, causal=True, window_size=(20, 0), sink_tokens=2)
        return [out, pre, new, used]

    return fill, call, caches


def test_serving_calls_captured_and_from_threads():
    """The calls above captured on two streams and replayed side by side, and made by two threads at once on streams of
    their own, give what they give one after the other."""
    import threading
    K = kernel()
    steps = [serving_step(x) for x in (1, 2)]
    want = []
    for x, (fill, call, caches) in enumerate(steps):
        want.append([])
        for r in range(3):
            fill(r)
            want[x].append([t.clone() for t in call() + caches])
    assert status() == 0
    torch.cuda.synchronize()
    graphs = []
    for fill, call, caches in steps:
        fill(0)
        torch.cuda.synchronize()
        stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            outs = call()
        graphs.append((stream, graph, outs))
    for r in range(3):
        for fill, _, _ in steps:
            fill(r)
        torch.cuda.synchronize()
        for stream, graph, _ in graphs:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for (_, _, caches), (_, _, outs), w in zip(steps, graphs, want):
            assert all(torch.equal(a, b) for a, b in zip(outs + caches, w[r]))
    for stream, _, _ in graphs:
        with torch.cuda.stream(stream):
            assert status() == 0
    failed = []

    def work(x):
        fill, call, caches = steps[x]
        stream = torch.cuda.Stream()
        try:
            with torch.cuda.stream(stream):
                for r in range(30):
                    fill(r % 3)
                    got = call() + caches
                    if not all(torch.equal(a, b) for a, b in zip(got, want[x][r % 3])):
                        failed.append((x, r))
                if K.status(torch.device("cuda", torch.cuda.current_device())):
                    failed.append((x, "status"))
        except Exception as e:  # noqa: BLE001
            failed.append((x, repr(e)))

    threads = [threading.Thread(target=work, args=(x,)) for x in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("window", [(-1, -1), (5, 0), (-1, 9)])
def test_prefill_packed_offsets_past_the_tokens(dtype, window):
    """Offsets on the device that leave the packed tokens, or fall, are brought back and flagged: nothing is read or
    written out of place, and the sequences that they do not concern are as ever."""
    C, K = api(), kernel()
    g = torch.Generator().manual_seed(1)
    n = 330
    q, k, v = (torch.randn(n, h, 64, generator=g).to(dtype).to(DEV) for h in (4, 2, 2))
    cu = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    call = lambda cq, ck, causal: C.flash_attn_varlen_func(q, k, v, cq, ck, n, n, causal=causal,  # noqa: E731
                                                           window_size=window, return_attn_probs=True)
    for causal in (False, True):
        for bad, good in (((0, 200, 1 << 30), (0, 200, n)), ((-7, 200, n), (0, 200, n)), ((0, 200, 120), (0, 200, 200)),
                          ((0, 200, -(1 << 31)), (0, 200, 200)), ((0, 1 << 29, 1 << 30), (0, n, n))):
            want, want_lse = call(cu(*good), cu(*good), causal)
            assert status() == 0
            for cq, ck in ((bad, good), (good, bad), (bad, bad)):
                out, lse = call(cu(*cq), cu(*ck), causal)
                assert status() == K.STATUS_LENS
                rows = good[2]
                assert torch.equal(out[:rows], want[:rows]) and torch.equal(lse[:, :rows], want_lse[:, :rows])


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("window", [(-1, -1), (5, 0), (3, 9)])
def test_prefill_packed_without_any_key(dtype, window):
    """Packed sequences none of which has a key (the packed k and v are empty): zeros, and log-sum-exps of -inf."""
    q = torch.randn(9, 4, 64, generator=torch.Generator().manual_seed(0)).to(dtype).to(DEV)
    kv = torch.zeros(0, 2, 64, dtype=dtype, device=DEV)
    cq, ck = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in ([0, 2, 9], [0, 0, 0]))
    for causal in (False, True):
        out, lse = api().flash_attn_varlen_func(q, kv, kv, cq, ck, 7, 1, causal=causal, window_size=window, sink_tokens=2,
                                                return_attn_probs=True)
        assert out.shape == q.shape and (out == 0).all() and torch.isneginf(lse).all()
    assert status() == 0
