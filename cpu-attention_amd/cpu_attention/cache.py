# Derived from ducviet00/cpu-attention (cpu_attention/cache.py), Apache License
# 2.0; modified for the MI355X build (see NOTICE at the repository root).  Kept
# from the original because the drop-in contract needs them: the function name
# and signature, the order of the argument checks, the exception types and the
# error messages.

"""``reshape_and_cache``: writing tokens into the paged KV cache; its 8-bit form
(``reshape_and_cache_fp8``) and copies of pages (``copy_blocks``).

The cache is in the original library's own layout -- per (block, head) a page of
``page_block_size`` tokens, K stored transposed inside the page -- so only this
library writes it: here, or through ``flash_attn_with_kvcache(k=..., v=...)``.
"""

import torch

from . import _kernel as K


def reshape_and_cache(key, value, k_cache, v_cache, slot_mapping) -> None:
    """Stores token ``i`` of ``key``/``value`` in cache slot ``slot_mapping[i]``.

    ``key`` and ``value`` are ``[num_tokens, nheads, headdim]`` with heads and head
    dims packed and any token stride (so the K and V slices of a fused projection
    are read in place); the caches are ``[num_blocks, nheads, page_block_size,
    headdim]``.  A slot ``s`` (int64) names block ``s // page_block_size``, position
    ``s % page_block_size``; a negative slot leaves its token out (padding), vLLM's
    convention.  The copy is queued on torch's current stream.
    """
    store = K.module().store
    if store(K.runtime(), key, value, k_cache, v_cache, slot_mapping) is None:
        key, value, slot_mapping = _check(key, value, k_cache, v_cache, slot_mapping)
        if store(K.runtime(), key, value, k_cache, v_cache, slot_mapping) is None:
            raise RuntimeError("cpu_attention: the kernel declined arguments that passed validation")


def _check(key, value, k_cache, v_cache, slots):
    """Called once the kernel module declined a store: raises the error that names
    the broken rule (the original library's checks in its order, then this
    build's device and alignment rules), or returns key, value and the slots in
    layouts the store kernel reads in place."""
    if key.dim() != 3 or value.shape != key.shape:
        raise ValueError("cpu_attention: key/value must both be [num_tokens, nheads, headdim]")
    if k_cache.dim() != 4 or v_cache.shape != k_cache.shape:
        raise ValueError("cpu_attention: k_cache/v_cache must be "
                         "[num_blocks, nheads, page_block_size, headdim] and match")
    if key.shape[1:] != (k_cache.shape[1], k_cache.shape[3]):
        raise ValueError("cpu_attention: key/value heads or head_dim do not match the cache")
    if not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        raise ValueError("cpu_attention: the paged caches must be contiguous")
    if key.dtype not in K.DTYPES or not key.dtype == value.dtype == k_cache.dtype == v_cache.dtype:
        raise ValueError("cpu_attention: key/value and the caches must share a dtype (fp32 or bf16)")
    if key.shape[2] not in K.HEAD_DIMS or k_cache.shape[2] % 16:
        raise ValueError("cpu_attention: head_dim must be 32/64/128 and the page a multiple of 16")
    if slots.dtype != torch.int64 or slots.shape != (key.shape[0],):
        raise ValueError("cpu_attention: slot_mapping must be int64 [num_tokens]")
    capacity = k_cache.shape[0] * k_cache.shape[2]
    if key.shape[0] and int(slots.max()) >= capacity:
        raise ValueError("cpu_attention: slot_mapping points past the end of the cache")
    dev = k_cache.device
    if not (k_cache.is_cuda and v_cache.device == dev and key.device == dev and value.device == dev):
        raise ValueError("cpu_attention: the MI355X build takes tensors on one ROCm GPU")
    if not (K.aligned(k_cache) and K.aligned(v_cache)):
        raise ValueError("cpu_attention: the paged caches must start 16-byte aligned")
    plain = (torch.Tensor, torch.nn.Parameter)
    key, value, slots = (x if type(x) in plain else x.as_subclass(torch.Tensor) for x in (key, value, slots))
    # one shared layout with packed heads, then 16-byte alignment
    if key.stride(-1) != 1 or key.stride(-2) != key.shape[2] or value.stride() != key.stride():
        key, value = key.contiguous(), value.contiguous()
    step = key.stride(0) if key.shape[0] > 1 else 0
    if not (K.aligned(key, (step,)) and K.aligned(value, (step,))):
        key, value = (x.clone(memory_format=torch.contiguous_format) for x in (key, value))
    return key, value, slots.contiguous()


SCALES = ("cpu_attention: k_scale and v_scale must be two fp32 [num_blocks, nheads] tensors, contiguous, "
          "on the caches' device")


def reshape_and_cache_fp8(key, value, k_cache, v_cache, k_scale, v_scale, slot_mapping) -> None:
    """``reshape_and_cache`` into an 8-bit cache, with one scale per page and head.

    The caches are ``torch.float8_e4m3fn`` ``[num_blocks, nheads, page_block_size,
    headdim]``, ``k_scale`` and ``v_scale`` fp32 ``[num_blocks, nheads]`` (zeros for a
    fresh cache); a code stands for code * scale.  ``key``, ``value`` (bf16 or fp32) and
    ``slot_mapping`` are ``reshape_and_cache``'s.

    Scales are powers of two, 2**-100 or more, just large enough for the largest finite
    magnitude that they cover to stay within e4m3's 448, so dividing by them is exact
    and a value is rounded once, to nearest even.  Pages are filled from position 0 on:

    - a call that writes position 0 of a page starts the page anew.  Its scale is taken
      from the call's tokens alone, and what the page held before is gone;
    - any other call adds to the page.  Its scale grows where the new tokens need it,
      and the codes that the page holds are then rescaled (exactly, unless a code
      becomes subnormal: the error stays below 2**-18 of the page's largest value).

    Infinities and NaNs are stored as NaN and take no part in a scale.  A slot named
    twice takes its last token.  Nothing depends on the order of the other slots.
    """
    store = K.module().store_fp8
    if store(K.runtime(), key, value, k_cache, v_cache, k_scale, v_scale, slot_mapping) is None:
        key, value, k_scale, v_scale, slots = _check_fp8(key, value, k_cache, v_cache, k_scale, v_scale, slot_mapping)
        if store(K.runtime(), key, value, k_cache, v_cache, k_scale, v_scale, slots) is None:
            raise RuntimeError("cpu_attention: the kernel declined arguments that passed validation")


def check_fp8_cache(k_cache, v_cache, k_scale, v_scale):
    """Raises the error that names what is wrong with an 8-bit cache's types or scales."""
    if k_cache.dtype != K.FP8 or v_cache.dtype != K.FP8:
        raise ValueError("cpu_attention: the 8-bit caches must be torch.float8_e4m3fn")
    for x in (k_scale, v_scale):
        if not isinstance(x, torch.Tensor) or x.dtype != torch.float32 or x.shape != k_cache.shape[:2] \
                or not x.is_contiguous() or x.device != k_cache.device:
            raise ValueError(SCALES)
    if k_scale.numel() and (k_scale.data_ptr() == v_scale.data_ptr() or k_cache.data_ptr() == v_cache.data_ptr()):
        raise ValueError("cpu_attention: K and V need caches and scales of their own")


def _check_fp8(key, value, k_cache, v_cache, k_scale, v_scale, slots):
    """Called once the kernel module declined an 8-bit store: ``_check``'s rules and the
    8-bit cache's."""
    if key.dim() != 3 or value.shape != key.shape:
        raise ValueError("cpu_attention: key/value must both be [num_tokens, nheads, headdim]")
    if k_cache.dim() != 4 or v_cache.shape != k_cache.shape:
        raise ValueError("cpu_attention: k_cache/v_cache must be "
                         "[num_blocks, nheads, page_block_size, headdim] and match")
    if key.shape[1:] != (k_cache.shape[1], k_cache.shape[3]):
        raise ValueError("cpu_attention: key/value heads or head_dim do not match the cache")
    if not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        raise ValueError("cpu_attention: the paged caches must be contiguous")
    check_fp8_cache(k_cache, v_cache, k_scale, v_scale)
    if key.dtype not in K.DTYPES or key.dtype != value.dtype:
        raise ValueError("cpu_attention: key/value must share a dtype (fp32 or bf16)")
    if key.shape[2] not in K.HEAD_DIMS or k_cache.shape[2] == 0 or k_cache.shape[2] % 16:
        raise ValueError("cpu_attention: head_dim must be 32/64/128 and the page a multiple of 16")
    if slots.dtype != torch.int64 or slots.shape != (key.shape[0],):
        raise ValueError("cpu_attention: slot_mapping must be int64 [num_tokens]")
    capacity = k_cache.shape[0] * k_cache.shape[2]
    if key.shape[0] and int(slots.max()) >= capacity:
        raise ValueError("cpu_attention: slot_mapping points past the end of the cache")
    dev = k_cache.device
    if not (k_cache.is_cuda and v_cache.device == dev and key.device == dev and value.device == dev):
        raise ValueError("cpu_attention: the MI355X build takes tensors on one ROCm GPU")
    if not (K.aligned(k_cache) and K.aligned(v_cache)):
        raise ValueError("cpu_attention: the paged caches must start 16-byte aligned")
    plain = (torch.Tensor, torch.nn.Parameter)
    key, value, k_scale, v_scale, slots = (x if type(x) in plain else x.as_subclass(torch.Tensor)
                                           for x in (key, value, k_scale, v_scale, slots))
    # one shared layout with packed heads, then 16-byte alignment
    if key.stride(-1) != 1 or key.stride(-2) != key.shape[2] or value.stride() != key.stride() \
            or (key.shape[0] > 1 and key.stride(0) < key.shape[1] * key.shape[2]):
        key, value = key.contiguous(), value.contiguous()
    step = key.stride(0) if key.shape[0] > 1 else 0
    if not (K.aligned(key, (step,)) and K.aligned(value, (step,))):
        key, value = (x.clone(memory_format=torch.contiguous_format) for x in (key, value))
    return key, value, k_scale, v_scale, slots.contiguous()


def copy_blocks(key_caches, value_caches, block_mapping, key_scales=None, value_scales=None) -> None:
    """Copies pages within the caches of several layers: page ``block_mapping[i][0]`` to
    page ``block_mapping[i][1]`` of every cache, for every pair ``i``.

    ``key_caches`` and ``value_caches`` are lists of as many caches of one shape and type
    (fp32, bf16 or float8_e4m3fn), ``block_mapping`` int64 ``[num_pairs, 2]``;
    ``key_scales`` and ``value_scales`` are an 8-bit cache's scales, layer by layer, and
    go with their pages.  It serves a forked sequence, whose last page cannot be shared
    once both append to it, and compacting a cache whose sequences have ended (the
    caller's page tables then name the new pages).

    A pair with a negative page is padding, a page copied to itself stays.  All pages
    are copied as if at once: destinations must be distinct, and no pair's destination
    another pair's source.  With host checks on that is checked (ValueError, nothing
    copied); with them off, such pages end up with unspecified contents, and pages past
    the caches are left out.  The copies are queued on torch's current stream.
    """
    copy, rt = K.module().copy_blocks, K.runtime()
    if K.host_checks() or copy(rt, key_caches, value_caches, key_scales, value_scales, block_mapping) is None:
        lists = _check_copy(key_caches, value_caches, block_mapping, key_scales, value_scales)
        if copy(rt, *lists) is None:
            raise RuntimeError("cpu_attention: the kernel declined arguments that passed validation")


def _check_copy(key_caches, value_caches, mapping, key_scales, value_scales):
    """Raises the error that names what is wrong with a call, or returns its arguments as
    the kernel module takes them: lists of plain tensors, and a contiguous mapping, read
    with host checks on."""
    keys, values = [_plain(x) for x in key_caches], [_plain(x) for x in value_caches]
    caches = keys + values
    if len(keys) != len(values):
        raise ValueError("cpu_attention: as many key caches as value caches")
    if (key_scales is None) != (value_scales is None):
        raise ValueError("cpu_attention: pass key_scales and value_scales, or neither")
    for x in caches:
        if x.dim() != 4 or x.shape != caches[0].shape or x.dtype != caches[0].dtype or not x.is_contiguous():
            raise ValueError("cpu_attention: the caches must be [num_blocks, nheads, page_block_size, headdim], "
                             "contiguous, of one shape and dtype")
    if caches and (caches[0].dtype not in (*K.DTYPES, K.FP8) or caches[0].shape[3] not in K.HEAD_DIMS
                   or caches[0].shape[2] == 0 or caches[0].shape[2] % 16):
        raise ValueError("cpu_attention: the caches must be fp32, bf16 or float8_e4m3fn, "
                         "head_dim 32/64/128 and the page a multiple of 16")
    if caches and caches[0].dtype == K.FP8 and key_scales is None:
        raise ValueError("cpu_attention: 8-bit caches are copied with key_scales and value_scales")
    scales = []
    if key_scales is not None:
        key_scales, value_scales = ([_plain(x) for x in xs] for xs in (key_scales, value_scales))
        scales = key_scales + value_scales
        if caches and caches[0].dtype != K.FP8 or not len(key_scales) == len(value_scales) == len(keys):
            raise ValueError("cpu_attention: key_scales and value_scales go with 8-bit caches, one per cache")
        for k, v, ks, vs in zip(keys, values, key_scales, value_scales):
            check_fp8_cache(k, v, ks, vs)
    if not isinstance(mapping, torch.Tensor) or mapping.dtype != torch.int64 or mapping.dim() != 2 or mapping.shape[1] != 2:
        raise ValueError("cpu_attention: block_mapping must be int64 [num_pairs, 2]")
    mapping = _plain(mapping).contiguous()
    if caches:
        dev = caches[0].device
        if not caches[0].is_cuda or any(x.device != dev for x in caches + scales):
            raise ValueError("cpu_attention: the MI355X build takes tensors on one ROCm GPU")
        if any(x.data_ptr() % 16 for x in caches):
            raise ValueError("cpu_attention: the paged caches must start 16-byte aligned")
        if mapping.device.type != "cpu" and mapping.device != dev:
            raise ValueError("cpu_attention: block_mapping must be on the caches' device or the CPU")
        if K.host_checks():
            check_mapping(mapping.cpu(), caches[0].shape[0])
    return keys, values, key_scales, value_scales, mapping


def _plain(x):
    """Tensor subclasses become plain tensors; anything else passes through."""
    return x.as_subclass(torch.Tensor) if isinstance(x, torch.Tensor) and type(x) is not torch.Tensor else x


def check_mapping(mapping, num_blocks):
    """Raises unless the pairs of ``mapping`` (a CPU tensor) can be copied at once: pages
    within the cache, distinct destinations, none of them another pair's source."""
    used = mapping[(mapping >= 0).all(1)]
    if used.numel() and int(used.max()) >= num_blocks:
        raise ValueError("cpu_attention: block_mapping points past the end of the cache")
    src, dst = used[used[:, 0] != used[:, 1]].unbind(1)
    to = dst.sort().values
    if bool((to[1:] == to[:-1]).any()):
        raise ValueError("cpu_attention: block_mapping names a destination twice")
    if bool(torch.isin(src, to).any()):
        raise ValueError("cpu_attention: block_mapping copies a page that it also overwrites")
