"""The paged KV cache: writing tokens (``reshape_and_cache``, and
``append_quantized`` for caches held in 8 bits) and moving blocks
(``copy_blocks``, ``compact_blocks``).

The cache layout belongs to this library (head-major pages with K stored
transposed inside each page, the reference's x86 layout), so tokens reach it
only through this function (vLLM's signature, the reference's
`cpu_attention/cache.py`) or through ``flash_attn_with_kvcache(k=..., v=...)``.
"""

import torch

from . import _kernel as K
from . import _native


def reshape_and_cache(key, value, k_cache, v_cache, slot_mapping) -> None:
    """Writes the K/V rows of ``num_tokens`` tokens into their cache slots.

    ``key`` and ``value`` are ``[num_tokens, nheads_k, headdim]`` with heads and
    dims packed; the token stride is free (a chunk of a fused projection needs
    no copy). The caches are ``[num_blocks, nheads_k, page_block_size,
    headdim]``. ``slot_mapping`` (int64 ``[num_tokens]``) gives each token's
    slot, ``block * page_block_size + position``; a negative slot leaves the
    token out (padding). The write is bit-exact: the cache holds the given
    values in its own layout.
    """
    if _native.store(0, key, value, k_cache, v_cache, slot_mapping) is not None:
        return
    key, value, slot_mapping = _explain_store(key, value, k_cache, v_cache, slot_mapping)
    if _native.store(0, key, value, k_cache, v_cache, slot_mapping) is None:
        raise RuntimeError("cpu_attention: the kernel declined arguments that passed validation")


def _explain_store(key, value, k_cache, v_cache, slots):
    """Called when the store entry declined: raise the reference's error for a
    bad argument, else return key/value with packed rows and the slots
    contiguous on the cache's device."""
    key, value, slots = (x.as_subclass(torch.Tensor) if isinstance(x, torch.Tensor)
                         and type(x) not in (torch.Tensor, torch.nn.Parameter) else x for x in (key, value, slots))
    if key.dim() != 3 or value.shape != key.shape:
        raise ValueError("cpu_attention: key/value must both be [num_tokens, nheads, headdim]")
    if k_cache.dim() != 4 or v_cache.shape != k_cache.shape:
        raise ValueError("cpu_attention: k_cache/v_cache must be "
                         "[num_blocks, nheads, page_block_size, headdim] and match")
    tokens, heads, hd = key.shape
    blocks, cache_heads, page, cache_hd = k_cache.shape
    if (heads, hd) != (cache_heads, cache_hd):
        raise ValueError("cpu_attention: key/value heads or head_dim do not match the cache")
    if not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        raise ValueError("cpu_attention: the paged caches must be contiguous")
    if key.dtype not in K.DTYPES or any(t.dtype != key.dtype for t in (value, k_cache, v_cache)):
        raise ValueError("cpu_attention: key/value and the caches must share a dtype (fp32 or bf16)")
    if hd not in K.HEAD_DIMS or page % 16:
        raise ValueError("cpu_attention: head_dim must be 32/64/128 and the page a multiple of 16")
    if slots.dtype != torch.int64 or tuple(slots.shape) != (tokens,):
        raise ValueError("cpu_attention: slot_mapping must be int64 [num_tokens]")
    if tokens and int(slots.max()) >= blocks * page:
        raise ValueError("cpu_attention: slot_mapping points past the end of the cache")
    dev = k_cache.device
    if dev.type != "cuda" or any(t.device != dev for t in (key, value, v_cache)):
        raise ValueError("cpu_attention: key/value and the caches must be CUDA tensors on one device "
                         f"(the cache is on {dev})")
    if key.stride(-1) != 1 or key.stride(-2) != hd or value.stride() != key.stride():
        key, value = key.contiguous(), value.contiguous()
    slots = slots.contiguous()
    return key, value, slots if slots.device == dev else slots.to(dev, non_blocking=True)


def check_eight_bit(k_cache, v_cache, k_descale, v_descale):
    """Raise unless these are caches held in 8 bits with their scales."""
    if any(t is None or t.dtype != K.EIGHT_BIT for t in (k_cache, v_cache)):
        raise ValueError("cpu_attention: caches held in 8 bits must both be torch.float8_e4m3fn")
    if k_cache.dim() != 4 or v_cache.shape != k_cache.shape:
        raise ValueError("cpu_attention: k_cache/v_cache must be "
                         "[num_blocks, nheads, page_block_size, headdim] and match")
    for name, t in (("k_descale", k_descale), ("v_descale", v_descale)):
        if (not isinstance(t, torch.Tensor) or t.dtype != torch.float32 or tuple(t.shape) != tuple(k_cache.shape[:2])
                or not t.is_contiguous()):
            raise ValueError(f"cpu_attention: caches held in 8 bits need {name}: float32 [num_blocks, nheads], "
                             "contiguous")


def check_packed_caches(k_cache, v_cache):
    """Raise unless the kernels can read the caches' 16-byte vectors."""
    if not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        raise ValueError("cpu_attention: the paged caches must be contiguous")
    if any(t.numel() and t.data_ptr() % 16 for t in (k_cache, v_cache)):
        raise ValueError("cpu_attention: the paged caches must start at a multiple of 16 bytes")


def packed_rows(*ts):
    """Copies of the tensors with the strides of a fresh tensor (a size of 1 may
    have any stride in one that is contiguous), all or none."""
    def plain(t):
        want, n = [], 1
        for size in reversed(t.shape):
            want.append(n)
            n *= max(size, 1)
        return t.stride() == tuple(reversed(want))
    return ts if all(map(plain, ts)) else tuple(t.clone(memory_format=torch.contiguous_format).view(-1).view(t.shape)
                                                for t in ts)


def append_quantized(key, value, k_cache, v_cache, k_descale, v_descale, cache_seqlens, page_table,
                     cu_seqlens_new=None, max_seqlen_new=None) -> None:
    """Appends tokens to paged caches held in 8 bits.

    The caches are ``torch.float8_e4m3fn`` ``[num_blocks, nheads_k,
    page_block_size, headdim]`` (K is not transposed), the scales float32
    ``[num_blocks, nheads_k]``; a value is its code times the scale of its block
    and head. ``key`` and ``value`` (fp32 or bf16) are ``[batch, n, nheads_k,
    headdim]``, or ``[total, nheads_k, headdim]`` packed with
    ``cu_seqlens_new`` (int32 ``[batch + 1]``, no sequence longer than
    ``max_seqlen_new``). Sequence i's tokens go to positions
    ``cache_seqlens[i]`` (int32 ``[batch]``, the lengths before) onwards, through
    ``page_table`` (int32 ``[batch, max_blocks]``); a negative length leaves the
    sequence out.

    A block's scale is a power of two that fits its largest value into e4m3
    (448). It only grows while the block fills -- then the codes in it are
    rounded to the new scale, which loses nothing but what falls below the
    smallest code -- and starts afresh when a token is written at the block's
    position 0. A scale of the caller's own stays as long as it is large enough;
    where one that is no power of two has to grow, codes move by up to half of
    their step. An infinity is stored as the largest code, NaN as NaN. A partly
    filled block that sequences share has to be copied (``copy_blocks``) before
    one of them appends to it.
    """
    args = (key, value, k_cache, v_cache, k_descale, v_descale, cache_seqlens, page_table, cu_seqlens_new)
    most = 0
    if cu_seqlens_new is not None:
        most = key.shape[0] if max_seqlen_new is None else min(int(max_seqlen_new), key.shape[0])
    if _native.append_8bit(0, *args, most) is not None:
        return
    args = _explain_append(*args, most)
    if _native.append_8bit(0, *args, most) is None:
        raise RuntimeError("cpu_attention: the kernel declined arguments that passed validation")


def _plain(*ts):
    return tuple(x.as_subclass(torch.Tensor) if isinstance(x, torch.Tensor)
                 and type(x) not in (torch.Tensor, torch.nn.Parameter) else x for x in ts)


def _explain_append(key, value, k_cache, v_cache, k_scale, v_scale, lens, table, cu, most):
    """Called when the append declined: raise for a bad argument, else return
    the tensors in the forms the kernel reads, on the caches' device."""
    key, value, k_cache, v_cache, k_scale, v_scale, lens, table, cu = _plain(key, value, k_cache, v_cache, k_scale,
                                                                             v_scale, lens, table, cu)
    if key.dim() != (4 if cu is None else 3) or value.shape != key.shape:
        raise ValueError("cpu_attention: key/value must both be [batch, seqlen_new, nheads, headdim], or "
                         "[total, nheads, headdim] with cu_seqlens_new")
    check_eight_bit(k_cache, v_cache, k_scale, v_scale)
    blocks, heads, page, hd = k_cache.shape
    if tuple(key.shape[-2:]) != (heads, hd):
        raise ValueError("cpu_attention: key/value heads or head_dim do not match the cache")
    if key.dtype not in K.DTYPES or value.dtype != key.dtype:
        raise ValueError("cpu_attention: key/value must share a dtype (fp32 or bf16)")
    check_packed_caches(k_cache, v_cache)
    if hd not in K.HEAD_DIMS or page % 16 or page < 1 or heads < 1:
        raise ValueError("cpu_attention: head_dim must be 32/64/128 and the page a multiple of 16")
    if lens.dtype != torch.int32 or lens.dim() != 1:
        raise ValueError("cpu_attention: cache_seqlens must be an int32 [batch] tensor")
    batch = lens.shape[0]
    if table.dtype != torch.int32 or table.dim() != 2 or table.shape[0] != batch:
        raise ValueError("cpu_attention: page_table must be int32 [batch, max_blocks]")
    if cu is None:
        if key.shape[0] != batch:
            raise ValueError("cpu_attention: key/value and cache_seqlens disagree on the batch")
        new = key.shape[1]
        longest = int(lens.max()) if batch and new else -1  # (negative: every sequence is left out)
        if longest >= 0 and longest + new > table.shape[1] * page:
            raise ValueError("cpu_attention: cache_seqlens exceed the page table's capacity")
    else:
        if not isinstance(cu, torch.Tensor) or cu.dtype != torch.int32 or tuple(cu.shape) != (batch + 1,):
            raise ValueError("cpu_attention: cu_seqlens_new must be int32 [batch + 1]")
        if most < 0:
            raise ValueError("cpu_attention: max_seqlen_new must not be negative")
        if cu.device.type == "cpu":
            n = cu[1:] - cu[:-1]
            if int(cu[0]) != 0 or bool((n < 0).any()) or int(cu[-1]) > key.shape[0] or \
                    (batch and int(n.max()) > most):
                raise ValueError("cpu_attention: cu_seqlens_new must rise from 0 to at most the token count, "
                                 "no sequence longer than max_seqlen_new")
    dev = k_cache.device
    if dev.type != "cuda" or any(t.device != dev for t in (key, value, v_cache, k_scale, v_scale)):
        raise ValueError("cpu_attention: key/value, the caches and their scales must be CUDA tensors on one device "
                         f"(the cache is on {dev})")
    key, value = packed_rows(key, value)
    lens, table, cu = (x if x is None else x.contiguous().to(dev) for x in (lens, table, cu))
    return key, value, k_cache, v_cache, k_scale, v_scale, lens, table, cu


def _block_list(caches):
    caches = [caches] if isinstance(caches, torch.Tensor) else list(caches)
    caches = list(_plain(*caches))
    for t in caches:
        if not isinstance(t, torch.Tensor) or t.dim() < 1 or t.shape[0] != caches[0].shape[0]:
            raise ValueError("cpu_attention: the caches must be tensors [num_blocks, ...] of one num_blocks")
        if not t.is_contiguous():
            raise ValueError("cpu_attention: the paged caches must be contiguous")
    return caches


def copy_blocks(caches, block_mapping) -> None:
    """Copies blocks within caches: block ``block_mapping[i, 0]`` becomes block
    ``block_mapping[i, 1]`` in every tensor of ``caches`` (a tensor, or a
    sequence of contiguous tensors ``[num_blocks, ...]`` -- the K and V caches
    of all layers, and the scales of caches held in 8 bits), in one launch for
    up to 128 tensors. ``block_mapping`` is int64 ``[n, 2]``; a pair with a
    negative id is left out. A block may be the source of several pairs (a fork)
    but the destination of one, and no destination may be a source: on the host
    that is checked, on the device it is the caller's to keep.
    """
    if isinstance(caches, torch.Tensor):
        caches = [caches]
    if not len(caches):
        return
    if isinstance(block_mapping, torch.Tensor) and block_mapping.is_cuda and \
            _native.copy_blocks(0, caches, block_mapping) is not None:
        return
    caches = _block_list(caches)
    (pairs,) = _plain(block_mapping)
    if not isinstance(pairs, torch.Tensor) or pairs.dtype != torch.int64 or pairs.dim() != 2 or pairs.shape[1] != 2:
        raise ValueError("cpu_attention: block_mapping must be int64 [n, 2]")
    if pairs.device.type == "cpu":
        kept = pairs[(pairs >= 0).all(1)]
        if kept.numel() and int(kept.max()) >= caches[0].shape[0]:
            raise ValueError("cpu_attention: block_mapping points past the end of the cache")
        src, dst = set(kept[:, 0].tolist()), kept[:, 1].tolist()
        if len(set(dst)) != len(dst) or src & set(dst):
            raise ValueError("cpu_attention: block_mapping writes a block twice, or one that it also reads")
    dev = caches[0].device
    if dev.type != "cuda" or any(t.device != dev for t in caches):
        raise ValueError(f"cpu_attention: the caches must be CUDA tensors on one device (the first is on {dev})")
    if _native.copy_blocks(0, caches, pairs.contiguous().to(dev)) is None:
        raise RuntimeError("cpu_attention: the kernel declined arguments that passed validation")


def compact_blocks(caches, page_table, cache_seqlens, page_block_size, window_size=(-1, -1), sink_tokens=0,
                   reserved_seqlens=None):
    """Moves the blocks in use to the front of the pool.

    In use are the blocks behind ``page_table`` (int32 ``[batch, max_blocks]``)
    whose page holds one of its sequence's ``cache_seqlens`` tokens and, with a
    window (``window_size``, ``sink_tokens`` as in ``flash_attn_with_kvcache``),
    is not wholly between the first tokens and the window: those pages are
    freed. ``cache_seqlens`` counts every token in the cache; tokens that a
    decode has just appended are not in the lengths it was given. To keep pages
    for tokens to come, give the lengths they will reach as ``reserved_seqlens``
    (int32 ``[batch]``; below ``cache_seqlens`` it changes nothing): the window
    is measured from ``cache_seqlens`` all the same, so nothing that is still
    seen is freed. A negative ``cache_seqlens`` leaves a sequence out. With n
    blocks in use, each one with an id of n or more moves, in ascending order,
    to the free ids below n, in every tensor of ``caches`` (contiguous
    ``[num_blocks, ...]``); blocks that sequences share move once and stay
    shared.

    Returns ``(new_table, used)``: the renumbered page table, -1 in every entry
    that is not in use, and n as int32 ``[1]`` on the device (no host
    synchronisation); ids from n on are free. ``page_table`` stays as it was.
    At most 2**20 blocks.
    """
    from .flash_attn_interface import _window

    left, _, sinks = _window(window_size, sink_tokens)
    caches = _block_list(caches)
    table, lens = _plain(page_table, cache_seqlens)
    page = int(page_block_size)
    if not caches:
        raise ValueError("cpu_attention: compact_blocks needs the caches")
    if page < 16 or page % 16:
        raise ValueError("cpu_attention: page_block_size must be a multiple of 16")
    if caches[0].shape[0] > 1 << 20:
        raise ValueError("cpu_attention: compact_blocks takes at most 2**20 blocks")
    if table.dtype != torch.int32 or table.dim() != 2:
        raise ValueError("cpu_attention: page_table must be int32 [batch, max_blocks]")
    if lens.dtype != torch.int32 or tuple(lens.shape) != (table.shape[0],):
        raise ValueError("cpu_attention: cache_seqlens must be an int32 [batch] tensor")
    if reserved_seqlens is not None:
        (reserved_seqlens,) = _plain(reserved_seqlens)
        if not isinstance(reserved_seqlens, torch.Tensor) or reserved_seqlens.dtype != torch.int32 \
                or tuple(reserved_seqlens.shape) != (table.shape[0],):
            raise ValueError("cpu_attention: reserved_seqlens must be an int32 [batch] tensor")
    dev = caches[0].device
    if dev.type != "cuda" or any(t.device != dev for t in caches):
        raise ValueError(f"cpu_attention: the caches must be CUDA tensors on one device (the first is on {dev})")
    table, lens, reserved = (x if x is None else x.contiguous().to(dev) for x in (table, lens, reserved_seqlens))
    got = _native.compact_blocks(0, caches, table, lens, page, left, sinks, reserved)
    if got is None:
        raise RuntimeError("cpu_attention: the kernel declined arguments that passed validation")
    return got
