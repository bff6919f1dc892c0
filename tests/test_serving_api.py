"""Refusals of the window, 8-bit-cache and page-copy entries, their C structures and what
the library declines (CPU only).  The device rule comes last, so a call on CPU tensors that
meets another error shows that rule fired, and a well-formed one meets the device rule."""

import ctypes
import math
import os
import subprocess

import pytest
import torch

import cpu_attention as C
from cpu_attention import _kernel as K

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
F8 = torch.float8_e4m3fn


def dense():
    q = torch.randn(2, 8, 4, 64)
    return q, q.clone(), q.clone()


def paged(fp8):
    q = torch.randn(2, 1, 4, 64)
    kc = torch.zeros(4, 4, 16, 64, dtype=F8 if fp8 else torch.float32)
    scales = [torch.ones(4, 4), torch.ones(4, 4)] if fp8 else []
    table = torch.arange(4, dtype=torch.int32).view(2, 2)
    return q, kc, torch.zeros_like(kc), scales, table


@pytest.mark.parametrize("kw,msg", [
    (dict(window_size=(3,)), "two ints"), (dict(window_size=5), "two ints"), (dict(window_size=(1.5, 0)), "two ints"),
    (dict(window_size=(-2, 0)), "-1"), (dict(window_size=(0, -3)), "-1"), (dict(sink_tokens=-1), "0 or more"),
    (dict(sink_tokens=1.0), "an int"), (dict(softmax_scale=0.0), "positive"), (dict(softmax_scale=-1.0), "positive"),
    (dict(softmax_scale=math.inf), "positive"), (dict(softmax_scale=math.nan), "positive"),
    (dict(window_size=(1 << 63, 0)), "-1"),
])
@pytest.mark.parametrize("op", ["window", "step", "step8"])
def test_bad_options(op, kw, msg):
    with pytest.raises(ValueError, match=msg):
        if op == "window":
            C.flash_attn_window_func(*dense(), **kw)
        else:
            q, kc, vc, scales, table = paged(op == "step8")
            fn = C.flash_attn_with_kvcache_fp8 if scales else C.flash_attn_window_with_kvcache
            fn(q, kc, vc, *scales, cache_seqlens=4, page_table=table, **kw)


@pytest.mark.parametrize("bad,msg,error", [
    ("dtype", "share a dtype", ValueError), ("head_dim", "head_dim must be", ValueError), ("heads", "matching q", ValueError),
    ("batch", "matching q", ValueError), ("rank", "must be \\[batch", ValueError), ("empty", "matching q", ValueError),
    ("grouped", "MHA only", NotImplementedError), ("none", "ROCm GPU", ValueError),
])
def test_window_bad_arguments(bad, msg, error):
    q, k, v = dense()
    if bad == "dtype":
        q, k, v = q.half(), k.half(), v.half()
    elif bad == "head_dim":
        q, k, v = q[..., :48], k[..., :48], v[..., :48]
    elif bad == "heads":
        q = q[:, :, :3]
    elif bad == "batch":
        k, v = k[:1], v[:1]
    elif bad == "rank":
        q = q[0]
    elif bad == "empty":
        k, v = k[:, :0], v[:, :0]
    elif bad == "grouped":
        k, v = k[:, :, :2], v[:, :, :2]
    with pytest.raises(error, match=msg):
        C.flash_attn_window_func(q, k, v, window_size=(3, 0), sink_tokens=1)


@pytest.mark.parametrize("bad,msg,error", [
    ("dtype", "", ValueError), ("head_dim", "head_dim must be", ValueError), ("page", "multiple of 16", ValueError),
    ("heads", "disagree on heads", ValueError), ("grouped", "MHA only", NotImplementedError),
    ("no_table", "pass `page_table`", ValueError), ("both_tables", "not both", ValueError),
    ("no_seqlens", "is required", ValueError), ("lens_dtype", "cache_seqlens must be", ValueError),
    ("table_dtype", "page_table must be", ValueError), ("capacity", "exceed the page table", ValueError),
    ("append_capacity", "exceed the page table", ValueError), ("many_capacity", "exceed the page table", ValueError),
    ("kv_shape", "k/v must both be", ValueError), ("k_alone", "k/v must both be", ValueError),
    ("kv_dtype", "k/v must both be", ValueError), ("kv_lengths", "k/v must both be", ValueError),
    ("q_dim", "q must be", ValueError), ("rows", "one query token", NotImplementedError),
    ("cache_shape", "must be", ValueError), ("noncontig", "must be contiguous", ValueError), ("none", "ROCm GPU", ValueError),
    ("scale_dtype", "k_scale and v_scale", ValueError), ("scale_shape", "k_scale and v_scale", ValueError),
    ("scale_strides", "k_scale and v_scale", ValueError), ("scale_none", "k_scale and v_scale", ValueError),
    ("scale_same", "of their own", ValueError),
])
@pytest.mark.parametrize("fp8", [False, True], ids=["fp32", "fp8"])
def test_kvcache_bad_arguments(fp8, bad, msg, error):
    q, kc, vc, scales, table = paged(fp8)
    lens, extra = 4, {}
    if bad.startswith("scale") and not fp8:
        return
    if bad == "dtype":
        kc, vc = kc.to(torch.float16), vc.to(torch.float16)
        msg = "float8_e4m3fn" if fp8 else "share a dtype"
    elif bad == "head_dim":
        q, kc, vc = q[..., :48], kc[..., :48].contiguous(), vc[..., :48].contiguous()
    elif bad == "page":
        kc, vc = kc[:, :, :8].contiguous(), vc[:, :, :8].contiguous()
    elif bad == "heads":
        q = q[:, :, :3]
    elif bad == "grouped":
        kc, vc = kc[:, :2].contiguous(), vc[:, :2].contiguous()
    elif bad == "no_table":
        table = None
    elif bad == "both_tables":
        extra = dict(block_table=table)
    elif bad == "no_seqlens":
        lens = None
    elif bad == "lens_dtype":
        lens = torch.full((2,), 4, dtype=torch.int64)
    elif bad == "table_dtype":
        table = table.long()
    elif bad == "capacity":
        lens = 33  # 2 pages of 16
    elif bad == "append_capacity":
        lens, extra = 32, dict(k=torch.randn(2, 1, 4, 64), v=torch.randn(2, 1, 4, 64))
    elif bad == "many_capacity":
        lens, extra = 20, dict(k=torch.randn(2, 13, 4, 64), v=torch.randn(2, 13, 4, 64))
    elif bad == "kv_shape":
        extra = dict(k=torch.randn(2, 1, 4, 64), v=torch.randn(2, 1, 4, 32))
    elif bad == "k_alone":
        extra = dict(k=torch.randn(2, 1, 4, 64))
    elif bad == "kv_dtype":
        extra = dict(k=torch.randn(2, 1, 4, 64).half(), v=torch.randn(2, 1, 4, 64).half())
    elif bad == "kv_lengths":
        extra = dict(k=torch.randn(2, 3, 4, 64), v=torch.randn(2, 2, 4, 64))
    elif bad == "q_dim":
        q = q[:, 0]
    elif bad == "rows":
        q = q.expand(2, 3, 4, 64)
    elif bad == "cache_shape":
        vc = vc[:3]
    elif bad == "noncontig":
        kc = kc.transpose(2, 3).contiguous().transpose(2, 3)
    elif bad == "scale_dtype":
        scales[0] = scales[0].double()
    elif bad == "scale_shape":
        scales[1] = scales[1][:3]
    elif bad == "scale_strides":
        scales[0] = scales[0].t()
    elif bad == "scale_none":
        scales[1] = None
    elif bad == "scale_same":
        scales[1] = scales[0]
    fn = C.flash_attn_with_kvcache_fp8 if fp8 else C.flash_attn_window_with_kvcache
    with pytest.raises(error, match=msg):
        fn(q, kc, vc, *scales, cache_seqlens=lens, page_table=table, window_size=(3, 0), **extra)


@pytest.mark.parametrize("bad,msg", [
    ("dtype", "share a dtype"), ("cache_dtype", "float8_e4m3fn"), ("heads", "do not match the cache"),
    ("slots_dtype", "int64"), ("slots_len", "int64"), ("past_end", "past the end"), ("rank", "key/value must both be"),
    ("page", "multiple of 16"), ("scales", "k_scale and v_scale"), ("same", "of their own"), ("noncontig", "contiguous"),
    ("none", "ROCm GPU"),
])
def test_reshape_and_cache_fp8_bad_arguments(bad, msg):
    k = torch.randn(5, 2, 64)
    kc, vc = torch.zeros(2, 2, 16, 64, dtype=F8), torch.zeros(2, 2, 16, 64, dtype=F8)
    scales, slots = [torch.zeros(2, 2), torch.zeros(2, 2)], torch.arange(5)
    v = k
    if bad == "dtype":
        v = k.bfloat16()
    elif bad == "cache_dtype":
        kc = kc.float()
        vc = vc.float()
    elif bad == "heads":
        k = v = torch.randn(5, 3, 64)
    elif bad == "slots_dtype":
        slots = slots.int()
    elif bad == "slots_len":
        slots = slots[:4]
    elif bad == "past_end":
        slots = slots + 30
    elif bad == "rank":
        k = v = k[None]
    elif bad == "page":
        kc, vc = kc[:, :, :8].contiguous(), vc[:, :, :8].contiguous()
    elif bad == "scales":
        scales[0] = torch.zeros(2)
    elif bad == "same":
        vc = kc
    elif bad == "noncontig":
        kc = kc.transpose(2, 3).contiguous().transpose(2, 3)
    with pytest.raises(ValueError, match=msg):
        C.reshape_and_cache_fp8(k, v, kc, vc, *scales, slots)


@pytest.mark.parametrize("bad,msg", [
    ("lists", "as many"), ("shapes", "one shape"), ("dtypes", "one shape"), ("type", "must be fp32"), ("dim", "must be fp32"),
    ("mapping_dtype", "block_mapping must be"), ("mapping_shape", "block_mapping must be"), ("one_scale", "or neither"),
    ("no_scales", "copied with"), ("needless_scales", "go with 8-bit"), ("few_scales", "go with 8-bit"),
    ("scale_shape", "k_scale and v_scale"), ("none", "ROCm GPU"),
])
def test_copy_blocks_bad_arguments(bad, msg):
    kc, vc = ([torch.zeros(4, 2, 16, 64) for _ in range(2)] for _ in range(2))
    mapping, kw = torch.tensor([[0, 1]]), {}
    f8 = [[torch.zeros(4, 2, 16, 64, dtype=F8) for _ in range(2)] for _ in range(2)]
    s8 = [[torch.zeros(4, 2) for _ in range(2)] for _ in range(2)]
    if bad == "lists":
        vc = vc[:1]
    elif bad == "shapes":
        vc[1] = vc[1][:3]
    elif bad == "dtypes":
        vc[1] = vc[1].bfloat16()
    elif bad == "type":
        kc, vc = ([x.half() for x in xs] for xs in (kc, vc))
    elif bad == "dim":
        kc, vc = ([x[..., :48].contiguous() for x in xs] for xs in (kc, vc))
    elif bad == "mapping_dtype":
        mapping = mapping.int()
    elif bad == "mapping_shape":
        mapping = mapping[0]
    elif bad == "one_scale":
        kw = dict(key_scales=s8[0])
    elif bad == "no_scales":
        kc, vc = f8
    elif bad == "needless_scales":
        kw = dict(key_scales=s8[0], value_scales=s8[1])
    elif bad == "few_scales":
        (kc, vc), kw = f8, dict(key_scales=s8[0][:1], value_scales=s8[1])
    elif bad == "scale_shape":
        (kc, vc), kw = f8, dict(key_scales=s8[0], value_scales=[torch.zeros(4, 2), torch.zeros(2, 4)])
    with pytest.raises(ValueError, match=msg):
        C.copy_blocks(kc, vc, mapping, **kw)


def test_copy_blocks_pairs_are_checked_before_anything():
    from cpu_attention.cache import check_mapping

    check_mapping(torch.tensor([[0, 1], [0, 2], [3, 3], [-1, 4], [5, -9]]), 6)
    check_mapping(torch.tensor([[3, 3], [3, 4]]), 5)  # staying is no overwriting
    check_mapping(torch.zeros(0, 2, dtype=torch.int64), 0)
    for pairs, msg in (([[0, 1], [2, 1]], "twice"), ([[0, 1], [1, 2]], "overwrites"), ([[0, 6]], "past the end"),
                       ([[6, 0]], "past the end")):
        with pytest.raises(ValueError, match=msg):
            check_mapping(torch.tensor(pairs), 6)


@pytest.mark.parametrize("binding", ["default", "ctypes"])
def test_module_entries_decline_with_none(binding):
    mod, rt = (K.module() if binding == "default" else K.ctypes_module()), K.runtime()
    q, k, v = dense()
    assert mod.flash_window(rt, q, k, v, None, True, 3, 0, 1) is None
    assert mod.flash_window(rt, q, k, v, None, 1, 3, 0, 1) is None
    lens = torch.full((2,), 4, dtype=torch.int32)
    for fp8 in (False, True):
        q, kc, vc, scales, table = paged(fp8)
        s = scales or [None, None]
        assert mod.decode_window(rt, q, kc, vc, *s, None, None, lens, table, None, 3, 1, 1) is None
        assert mod.decode_window(rt, q.half(), kc, vc, *s, None, None, lens, table, None, 3, 1, 1) is None
        assert mod.decode_window(rt, q, kc, vc, *s, None, None, lens, table, None, 3, 1, 0) is None
    x = torch.randn(3, 4, 64)
    assert mod.store_fp8(rt, x, x, kc, vc, *scales, torch.arange(3)) is None
    assert mod.copy_blocks(rt, [kc], [vc], *[[x] for x in scales], torch.tensor([[0, 1]])) is None
    if isinstance(mod, K.NativeModule):
        for entry in (mod.flash_window, mod.decode_window, mod.store_fp8, mod.copy_blocks):
            with pytest.raises(TypeError):
                entry(None)


_LAYOUT_C = r"""
#include <stddef.h>
#include <stdio.h>
#include "cpu_attention_hip.h"
#define F(T, f) printf("%s.%s %zu %zu\n", #T, #f, offsetof(T, f), sizeof(((T*)0)->f));
#define S(T) printf("%s %zu\n", #T, sizeof(T));
int main(void) { LINES return 0; }
"""


def test_ctypes_structures_match_the_header(tmp_path):
    structs = {"ca_flash_window_args": K.FlashWindowArgs, "ca_decode_window_args": K.DecodeWindowArgs,
               "ca_store_fp8_args": K.StoreFp8Args, "ca_copy_blocks_args": K.CopyBlocksArgs}
    lines = " ".join([f"S({c})" for c in structs] + [f"F({c}, {n})" for c, py in structs.items() for n, _ in py._fields_])
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text(_LAYOUT_C.replace("LINES", lines))
    subprocess.run(["gcc", "-std=c11", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split("\n")
    for line in filter(None, out):
        name, *numbers = line.split()
        if len(numbers) == 1:
            assert ctypes.sizeof(structs[name]) == int(numbers[0]), line
        else:
            cname, field = name.split(".")
            desc = getattr(structs[cname], field)
            assert (desc.offset, desc.size) == tuple(map(int, numbers)), line


def test_library_declines_malformed_calls_without_a_gpu():
    lib = K.load_library()

    def rc(entry, args):
        return getattr(lib, entry)(ctypes.byref(args), None)

    for entry in ("ca_flash_window", "ca_decode_window", "ca_store_fp8", "ca_copy_blocks"):
        assert getattr(lib, entry)(None, None) == K.CA_DECLINED
    f = K.FlashWindowArgs(left=3, right=0, sinks=0)
    f.flash.batch, f.flash.seq_q, f.flash.seq_k, f.flash.num_heads, f.flash.head_dim = 1, 40, 40, 2, 64
    f.flash.dtype, f.flash.scale = 1, 1.0
    assert rc("ca_flash_window", f) == K.CA_DECLINED  # null pointers
    f.flash.batch = 0
    assert rc("ca_flash_window", f) == K.CA_OK
    for field, value in (("scale", 0.0), ("scale", -1.0), ("head_dim", 48), ("seq_k", 0), ("seq_q", 1 << 30), ("dtype", 2)):
        old = getattr(f.flash, field)
        setattr(f.flash, field, value)
        assert rc("ca_flash_window", f) == K.CA_DECLINED, field
        setattr(f.flash, field, old)
    f.sinks = -1
    assert rc("ca_flash_window", f) == K.CA_DECLINED
    d = K.DecodeWindowArgs(left=3, sinks=0)
    a = d.decode
    a.num_seqs, a.num_heads, a.head_dim, a.page_size, a.dtype, a.scale, a.page_table_width = 2, 2, 64, 16, 1, 1.0, 4
    assert rc("ca_decode_window", d) == K.CA_DECLINED  # null pointers
    a.num_seqs = 0
    assert rc("ca_decode_window", d) == K.CA_OK
    d.k_scale = 16
    assert rc("ca_decode_window", d) == K.CA_DECLINED  # one scale
    d.k_scale, a.slots = None, 16
    assert rc("ca_decode_window", d) == K.CA_DECLINED  # slots
    a.slots, a.scale = None, math.nan
    assert rc("ca_decode_window", d) == K.CA_DECLINED
    s = K.StoreFp8Args()
    t = s.store
    t.num_tokens, t.num_heads, t.head_dim, t.page_size, t.num_blocks = 4, 2, 64, 16, 3
    assert rc("ca_store_fp8", s) == K.CA_DECLINED  # null pointers
    t.num_tokens = 0
    assert rc("ca_store_fp8", s) == K.CA_OK
    t.page_size = 24
    assert rc("ca_store_fp8", s) == K.CA_DECLINED
    c = K.CopyBlocksArgs(num_caches=1, block_bytes=64, num_pairs=1, num_blocks=2)
    assert rc("ca_copy_blocks", c) == K.CA_DECLINED  # null pointers
    c.num_pairs = 0
    assert rc("ca_copy_blocks", c) == K.CA_OK
    c.block_bytes = 24
    assert rc("ca_copy_blocks", c) == K.CA_DECLINED
    c.block_bytes, c.num_scales, c.row_bytes = 64, 1, 6
    assert rc("ca_copy_blocks", c) == K.CA_DECLINED


def test_workspace_queries():
    lib = K.load_library()
    # a row of the call's window never outgrows one block of 8 tiles of 64 keys: no partials,
    # whatever the page table holds
    assert lib.ca_decode_window_workspace_bytes(4, 8, 128, 16, 100000, 400, 4) == 0
    assert lib.ca_decode_window_workspace_bytes(4, 8, 128, 16, 100000, 2047, 4) > 0
    assert lib.ca_decode_window_workspace_bytes(4, 8, 128, 16, 100000, -1, 4) \
        == lib.ca_decode_window_workspace_bytes(4, 8, 128, 16, 100000, 10 ** 9, 0)
    assert lib.ca_decode_window_workspace_bytes(4, 8, 128, 16, -1, 3, 0) == -1
    assert lib.ca_store_fp8_workspace_bytes(1, 10 ** 6, 16) == 0
    assert lib.ca_store_fp8_workspace_bytes(5000, 100, 16) >= 4 * (100 * 16 + 100)
    assert lib.ca_store_fp8_workspace_bytes(-1, 100, 16) == -1
    # a window that leaves nothing out asks for what ca_flash does
    assert lib.ca_flash_window_workspace_bytes(1, 4, 8192, 8, 64, 1, 1, -1, -1, 0) \
        == lib.ca_flash_workspace_bytes(1, 4, 8192, 8, 64, 1) > 0
    assert lib.ca_flash_window_workspace_bytes(1, 512, 8192, 8, 64, 1, 1, 100, 0, 0) == 0
    # splits are at most the 64 that the combine merges
    for dtype in (0, 1):
        assert lib.ca_flash_window_workspace_bytes(1, 1, 1 << 20, 1, 64, dtype, 1, 1 << 19, 0, 0) == 64 * 66 * 4


def test_no_heads():
    q = torch.zeros(1, 4, 0, 64)
    with pytest.raises(ValueError, match="at least one head"):
        C.flash_attn_window_func(q, q, q, window_size=(2, 0))
    with pytest.raises(ValueError, match="at least one head"):
        C.flash_attn_window_func(torch.zeros(1, 4, 2, 64), q, q, window_size=(2, 0))


def test_window_positions_stay_within_31_bits():
    """An empty batch, so that only the sizes are looked at."""
    lib = K.load_library()
    f = K.FlashWindowArgs(left=3, right=-1, sinks=0)
    f.flash.seq_q, f.flash.num_heads, f.flash.head_dim, f.flash.dtype, f.flash.scale = 40, 2, 64, 1, 1.0
    for seq_k, want in (((1 << 30) - 1024, K.CA_OK), ((1 << 30) - 1023, K.CA_DECLINED), ((1 << 30) - 1, K.CA_DECLINED)):
        f.flash.seq_k = seq_k
        assert lib.ca_flash_window(ctypes.byref(f), None) == want
    d = K.DecodeWindowArgs(left=3, sinks=0, longest=12)
    d.decode.num_heads, d.decode.head_dim, d.decode.page_size, d.decode.scale = 2, 64, 16, 1.0
    assert lib.ca_decode_window(ctypes.byref(d), None) == K.CA_DECLINED
    d.longest = 16
    assert lib.ca_decode_window(ctypes.byref(d), None) == K.CA_OK
