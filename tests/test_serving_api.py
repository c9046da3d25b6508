"""Refusals of the serving operators, decided on the host (CPU tensors here), and
the float64 implementations the GPU tests use."""

import ctypes

import pytest
import torch

import cpu_attention as C
import serving as S
from cpu_attention import _kernel as K

F8 = torch.float8_e4m3fn


def eight(page=16, d=64):
    kc = torch.zeros(4, 2, page, d).to(F8)
    one = torch.ones(4, 2)
    return torch.randn(2, 1, 4, d), kc, kc.clone(), torch.arange(4, dtype=torch.int32).view(2, 2), one, one.clone()


def test_names():
    for name in ("append_quantized", "copy_blocks", "compact_blocks"):
        assert callable(getattr(C, name))


def test_valid_calls_are_refused_on_cpu():
    q, kc, vc, bt, ks, vs = eight()
    with pytest.raises(ValueError, match="CUDA"):
        C.flash_attn_with_kvcache(q, kc, vc, cache_seqlens=4, page_table=bt, k_descale=ks, v_descale=vs)
    f = torch.zeros(4, 2, 16, 64)
    for left in (8, -1):
        with pytest.raises(ValueError, match="CUDA"):
            C.flash_attn_with_kvcache(q, f, f.clone(), cache_seqlens=4, page_table=bt, window_size=(left, 0),
                                      sink_tokens=0)
    k = torch.randn(2, 3, 2, 64)
    with pytest.raises(ValueError, match="CUDA"):
        C.append_quantized(k, k, kc, vc, ks, vs, torch.zeros(2, dtype=torch.int32), bt)
    with pytest.raises(ValueError, match="CUDA"):
        C.copy_blocks([f, f.clone()], torch.tensor([[0, 1]]))
    with pytest.raises(ValueError, match="CUDA"):
        C.compact_blocks([f], bt, torch.zeros(2, dtype=torch.int32), 16)
    x = torch.randn(1, 8, 2, 64)
    with pytest.raises(ValueError, match="CUDA"):
        C.flash_attn_func(x, x, x, window_size=(4, 0), sink_tokens=2)
    cu = torch.tensor([0, 8], dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        C.flash_attn_varlen_func(x[0], x[0], x[0], cu, cu, 8, 8, window_size=(4, 0))


@pytest.mark.parametrize("bad", ["no_scales", "scale_dtype", "scale_shape", "scale_strided", "mixed", "head_dim", "heads",
                                 "page", "capacity", "table", "kv_heads", "half", "two_queries"])
def test_eight_bit_decode_refusals(bad):
    q, kc, vc, bt, ks, vs = eight()
    lens, more = 4, {}
    if bad == "no_scales":
        ks = None
    elif bad == "scale_dtype":
        ks = ks.double()
    elif bad == "scale_shape":
        vs = vs[:, :1].contiguous()
    elif bad == "scale_strided":
        vs = torch.ones(2, 4).t()
    elif bad == "mixed":
        vc = vc.float()
    elif bad == "head_dim":
        q, kc, vc = q[..., :48], kc[..., :48].contiguous(), vc[..., :48].contiguous()
    elif bad == "heads":
        q = q[:, :, :3]
    elif bad == "page":
        kc, vc = kc[:, :, :8].contiguous(), vc[:, :, :8].contiguous()
    elif bad == "capacity":
        lens = 33
    elif bad == "table":
        bt = bt.long()
    elif bad == "kv_heads":
        more = dict(k=torch.randn(2, 1, 4, 64), v=torch.randn(2, 1, 4, 64))
    elif bad == "half":
        q = q.half()
    elif bad == "two_queries":
        with pytest.raises(NotImplementedError):
            C.flash_attn_with_kvcache(q.expand(2, 2, 4, 64), kc, vc, cache_seqlens=lens, page_table=bt, k_descale=ks,
                                      v_descale=vs)
        return
    with pytest.raises(ValueError):
        C.flash_attn_with_kvcache(q, kc, vc, cache_seqlens=lens, page_table=bt, k_descale=ks, v_descale=vs, **more)


@pytest.mark.parametrize("kwargs", [dict(q_descale=torch.ones(1)), dict(softcap=1.0), dict(window_size=(8, 0))])
def test_eight_bit_decode_unsupported_options(kwargs):
    q, kc, vc, bt, ks, vs = eight()
    with pytest.raises(NotImplementedError):
        C.flash_attn_with_kvcache(q, kc, vc, cache_seqlens=4, page_table=bt, k_descale=ks, v_descale=vs, **kwargs)


@pytest.mark.parametrize("window,sinks", [((-2, 0), 0), ((4, -5), 0), ((4, 0), -1), ((4,), 0), (4, 0), (("a", 0), 0),
                                          ((4, 0), "x")])
def test_bad_windows(window, sinks):
    q, kc, vc, bt, ks, vs = eight()
    f = torch.zeros(4, 2, 16, 64)
    x = torch.randn(1, 8, 2, 64)
    cu = torch.tensor([0, 8], dtype=torch.int32)
    with pytest.raises(ValueError):
        C.flash_attn_with_kvcache(q, f, f, cache_seqlens=4, page_table=bt, window_size=window, sink_tokens=sinks)
    with pytest.raises(ValueError):
        C.flash_attn_func(x, x, x, window_size=window, sink_tokens=sinks)
    with pytest.raises(ValueError):
        C.flash_attn_varlen_func(x[0], x[0], x[0], cu, cu, 8, 8, window_size=window, sink_tokens=sinks)
    with pytest.raises(ValueError):
        C.compact_blocks([f], bt, torch.zeros(2, dtype=torch.int32), 16, window_size=window, sink_tokens=sinks)


@pytest.mark.parametrize("bad", ["cache_dtype", "scale", "heads", "dtype", "lens", "table", "batch", "capacity", "dims",
                                 "cu_dtype", "cu_order", "cu_past_end", "cu_longest", "page", "strided_cache"])
def test_append_refusals(bad):
    _, kc, vc, bt, ks, vs = eight()
    k = torch.randn(2, 3, 2, 64)
    lens, cu, most = torch.zeros(2, dtype=torch.int32), None, None
    if bad == "cache_dtype":
        kc = kc.float()
    elif bad == "scale":
        ks = None
    elif bad == "heads":
        k = torch.randn(2, 3, 4, 64)
    elif bad == "dtype":
        k = k.half()
    elif bad == "lens":
        lens = lens.long()
    elif bad == "table":
        bt = bt[:1]
    elif bad == "batch":
        k = torch.randn(3, 3, 2, 64)
    elif bad == "capacity":
        lens = lens + 30
    elif bad == "dims":
        k = k[0]
    elif bad.startswith("cu_"):
        k, cu, most = torch.randn(6, 2, 64), torch.tensor([0, 2, 6], dtype=torch.int32), 4
        if bad == "cu_dtype":
            cu = cu.long()
        elif bad == "cu_order":
            cu[1] = 7
        elif bad == "cu_past_end":
            cu[2] = 7
        else:
            most = 3
    elif bad == "page":
        kc, vc = kc[:, :, :8].contiguous(), vc[:, :, :8].contiguous()
    elif bad == "strided_cache":
        kc = torch.zeros(4, 2, 64, 16).to(F8).transpose(2, 3)
    with pytest.raises(ValueError):
        C.append_quantized(k, k, kc, vc, ks, vs, lens, bt, cu, most)


@pytest.mark.parametrize("pairs", [torch.tensor([[0, 1]], dtype=torch.int32), torch.tensor([0, 1]),
                                   torch.tensor([[0, 4]]), torch.tensor([[0, 1], [2, 1]]),
                                   torch.tensor([[0, 1], [1, 2]]), torch.tensor([[2, 2]])])
def test_copy_refusals(pairs):
    with pytest.raises(ValueError):
        C.copy_blocks([torch.zeros(4, 3)], pairs)


def test_copy_and_compact_cache_refusals():
    pairs, bt, lens = torch.tensor([[0, 1]]), torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    for caches in ([torch.zeros(4, 3), torch.zeros(5, 3)], [torch.zeros(4, 6)[:, ::2]], [3], [torch.tensor(1.0)]):
        with pytest.raises(ValueError):
            C.copy_blocks(caches, pairs)
        with pytest.raises(ValueError):
            C.compact_blocks(caches, bt, lens, 16)
    ok = [torch.zeros(4, 3)]
    for args in ((ok, bt.long(), lens, 16), (ok, bt, lens.long(), 16), (ok, bt, lens, 8), (ok, bt, lens, 0),
                 (ok, bt[0], lens, 16), ([], bt, lens, 16)):
        with pytest.raises(ValueError):
            C.compact_blocks(*args)


def test_abi_declines_bad_arguments_without_a_device():
    lib = K.library()
    p, nan = ctypes.c_void_p(16), float("nan")

    def dec(q_stride=256, heads=4, kv=2, e=64, page=16, qt=1, ct=2, ks=p, kn=None, n=0, left=-1, sinks=0, width=2, b=2,
            ws=p, kc=p):
        return lib.ca_decode_split(p, q_stride, kc, p, ks, p, 4, kn, kn, 256, 128, n, p, p, width, p, None, b, heads, kv,
                                   e, page, qt, ct, left, sinks, nan, ws, 0, None, None)

    assert dec(qt=2) == K.EDTYPE and dec(qt=1, ct=0) == K.EDTYPE and dec(qt=0, ct=1) == K.EDTYPE
    assert dec(e=48) == K.EHEADDIM and dec(page=24) == K.EPAGE and dec(page=0) == K.EPAGE
    assert dec(heads=3) == K.ESHAPE and dec(kv=0) == K.ESHAPE and dec(left=-2) == K.ESHAPE
    assert dec(sinks=-1) == K.ESHAPE and dec(n=1) == K.ESHAPE and dec(kn=p) == K.ESHAPE
    assert dec(width=1 << 28) == K.ESHAPE and dec(ks=None) == K.ENULL and dec(ws=None) == K.ENULL
    assert dec(q_stride=100) == K.ELAYOUT and dec(kc=ctypes.c_void_p(8)) == K.ELAYOUT
    assert dec(b=0) == K.OK

    def app(key=p, ts=128, ss=384, n=3, cu=None, total=0, ks=p, h=2, e=64, page=16, dt=1, b=2, lens=p):
        return lib.ca_append_8bit(key, p, ss, ts, n, cu, total, p, p, ks, p, 4, lens, p, 2, b, h, e, page, dt, None, None)

    assert app(dt=2) == K.EDTYPE and app(e=16) == K.EHEADDIM and app(page=8) == K.EPAGE and app(h=0) == K.ESHAPE
    assert app(n=-1) == K.ESHAPE and app(key=None) == K.ENULL and app(ks=None) == K.ENULL and app(lens=None) == K.ENULL
    assert app(ts=100) == K.ELAYOUT and app(ss=300) == K.ELAYOUT and app(key=ctypes.c_void_p(17)) == K.ELAYOUT
    assert app(n=0) == K.OK and app(b=0) == K.OK and app(cu=p, total=0) == K.OK
    base, size = (ctypes.c_void_p * 1)(16), (ctypes.c_int64 * 1)(64)
    none, zero = (ctypes.c_void_p * 1)(None), (ctypes.c_int64 * 1)(0)
    assert lib.ca_copy_blocks(none, size, 1, 4, p, 1, None, None) == K.ENULL
    assert lib.ca_copy_blocks(base, zero, 1, 4, p, 1, None, None) == K.ESHAPE
    assert lib.ca_copy_blocks(base, size, 1, -1, p, 1, None, None) == K.ESHAPE
    assert lib.ca_copy_blocks(base, size, 1, 4, None, 1, None, None) == K.ENULL
    assert lib.ca_copy_blocks(base, size, 1, 4, p, 0, None, None) == K.OK
    need = lib.ca_compact_workspace_bytes(4)

    def pack(blocks=4, page=16, left=-1, sinks=0, used=p, wsb=need, lens=p):
        return lib.ca_compact_blocks(base, size, 1, blocks, p, lens, 1, 2, page, left, sinks, p, used, p, wsb, None, None)

    assert pack(page=8) == K.EPAGE and pack(left=-2) == K.ESHAPE and pack(sinks=-1) == K.ESHAPE
    assert pack(blocks=(1 << 20) + 1) == K.EUNSUPPORTED and pack(used=None) == K.ENULL and pack(lens=None) == K.ENULL
    assert pack(wsb=need - 1) == K.EWORKSPACE
    st = (ctypes.c_int64 * 3)(0, 0, 0)
    fl = lambda left, right, sinks: lib.ca_flash_window(p, p, p, p, None, 1, 4, 4, 2, 2, 64, st, st, st, None,  # noqa
                                                        None, 0, 0, 1.0, 1, left, right, sinks, 0, None, None)
    assert fl(-2, 0, 0) == K.ESHAPE and fl(0, -2, 0) == K.ESHAPE and fl(0, 0, -1) == K.ESHAPE


# ------------------------------------------- the float64 implementations -----
def test_round_e4m3_is_the_type():
    """Every code is a fixed point; between neighbours the nearer one wins, ties to the even code."""
    codes = torch.arange(256, dtype=torch.uint8).view(F8).double()
    codes = codes[torch.isfinite(codes)].unique()
    assert torch.equal(S.round_e4m3(codes), codes)
    x = torch.linspace(-448, 448, 20011, dtype=torch.float64)
    x = torch.cat([x, x / 400, x / 40000, (codes[1:] + codes[:-1]) / 2])
    assert torch.equal(S.round_e4m3(x), x.float().to(F8).double())


def test_fit_scale():
    for top in (1.0, 448.0, 448.5, 1.75, 1.7500001, 3.4e38, 1e-40, 0.0, 2.0 ** -118):
        s = S.fit_scale(torch.tensor([top, -top / 2, float("inf")], dtype=torch.float64))
        assert s >= 2.0 ** -126 and top <= 448 * s and (s == 2.0 ** -126 or 448 * s / 2 < top)


def test_layouts_round_trip():
    from oracle import paged
    x = torch.randn(2, 3, 16, 32)
    for dt in (torch.float32, torch.bfloat16):
        for k_side in (True, False):
            assert torch.equal(S.unpack(S.pack(x.to(dt), k_side, "f"), k_side, "f"), x.to(dt))
    packed = S.pack(x.bfloat16(), True, "f")[1, 2].flatten()
    perm = torch.from_numpy(paged.k_perm(16, 32, True))
    assert torch.equal(packed[perm], x.bfloat16()[1, 2])


def test_compact_reserved_lengths_refusals():
    caches, bt, lens = [torch.zeros(4, 3)], torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    for reserved in (lens.long(), torch.zeros(2, dtype=torch.int32), lens.view(1, 1), 5, [5]):
        with pytest.raises(ValueError, match="reserved_seqlens"):
            C.compact_blocks(caches, bt, lens, 16, reserved_seqlens=reserved)
    with pytest.raises(ValueError, match="CUDA"):
        C.compact_blocks(caches, bt, lens, 16, reserved_seqlens=lens)


def step_example():
    """The decode step with compaction that the integration guide shows, as code."""
    import os
    import re

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    blocks = re.findall(r"```python\n(.*?)```", open(os.path.join(root, "INTEGRATION.md")).read(), re.S)
    (code,) = [b for b in blocks if "compact_blocks" in b]
    return code


def test_step_example_packs_with_the_new_token_counted(monkeypatch):
    """The decode leaves its lengths as they were; the compaction behind it has to count the token it appended."""
    lens, seen = torch.tensor([16, 5], dtype=torch.int32), {}

    def attend(*args, cache_seqlens, **kwargs):
        seen["attend"] = cache_seqlens.clone()
        return args[0]

    def pack(caches, table, cache_seqlens, page, **kwargs):
        seen["pack"] = cache_seqlens.clone()
        return table, torch.zeros(1, dtype=torch.int32)

    monkeypatch.setattr(C, "flash_attn_with_kvcache", attend)
    monkeypatch.setattr(C, "compact_blocks", pack)
    names = dict.fromkeys("q k v k_cache v_cache k_scale v_scale table".split())
    exec(step_example(), dict(names, lens=lens, page=16))
    assert seen["attend"].tolist() == [16, 5] and seen["pack"].tolist() == [17, 6]


def test_refused_window_names_the_way():
    """A window alone is the reference's refusal; its message says how to have one."""
    q, kc, vc, bt, ks, vs = eight()
    f = torch.zeros(4, 2, 16, 64)
    for caches in ((f, f.clone(), {}), (kc, vc, dict(k_descale=ks, v_descale=vs))):
        with pytest.raises(NotImplementedError, match="sink_tokens=0"):
            C.flash_attn_with_kvcache(q, *caches[:2], cache_seqlens=4, page_table=bt, window_size=(8, 0), **caches[2])


def test_negative_lengths_pass_the_capacity_check():
    """Sequences left out by a negative length have no tokens to place: the call goes on to the device check."""
    q, kc, vc, bt, ks, vs = eight()
    k, out = torch.randn(2, 40, 2, 64), torch.tensor([-1, -3], dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        C.flash_attn_with_kvcache(q, kc, vc, k=k, v=k, cache_seqlens=out, page_table=bt, k_descale=ks, v_descale=vs)
    with pytest.raises(ValueError, match="CUDA"):
        C.append_quantized(k, k, kc, vc, ks, vs, out, bt)
    out[0] = 0
    with pytest.raises(ValueError, match="capacity"):
        C.flash_attn_with_kvcache(q, kc, vc, k=k, v=k, cache_seqlens=out, page_table=bt, k_descale=ks, v_descale=vs)
    with pytest.raises(ValueError, match="capacity"):
        C.append_quantized(k, k, kc, vc, ks, vs, out, bt)
