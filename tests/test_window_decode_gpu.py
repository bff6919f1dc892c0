"""flash_attn_window_with_kvcache and flash_attn_with_kvcache_fp8 against the float64
oracle, within bounds derived from the arithmetic.  Everything that a row does not see is
NaN (cache positions, pages, scales) or out of range (page-table entries)."""

import ctypes

import numpy as np
import pytest
import torch

import cpu_attention as C
from cpu_attention import _kernel as K
from helpers import values
from oracle import serving as R
from serving_helpers import NAME, Paged, capture, close, same_bytes

pytestmark = pytest.mark.gpu
BF16, FP32 = torch.bfloat16, torch.float32
KINDS = [(BF16, False), (FP32, False), (BF16, True), (FP32, True)]
IDS = ["bf16", "fp32", "bf16-fp8", "fp32-fp8"]


def call(p, fp8, q=None, lens=None, table=None, **kw):
    q = p.q if q is None else q
    lens = p.lens_t if lens is None else lens
    table = p.table if table is None else table
    if fp8:
        return C.flash_attn_with_kvcache_fp8(q, p.kc, p.vc, p.kscale, p.vscale, cache_seqlens=lens, page_table=table, **kw)
    return C.flash_attn_window_with_kvcache(q, p.kc, p.vc, cache_seqlens=lens, page_table=table, **kw)


def reference(p, left, sinks, scale=None):
    return R.decode(values(p.q)[:, 0], p.ks, p.vs, scale or p.dim ** -0.5, left, sinks)


def hide(p, left, sinks, fp8):
    """Page-table entries of pages that hold no visible key become out of range, and
    positions of the other pages that are not seen NaN."""
    table = p.table.cpu()
    kc = p.kc.cpu().view(torch.uint8)
    vc = p.vc.cpu().view(torch.uint8)
    es = p.kc.element_size()
    per = 4 // es
    k = kc.view(p.blocks, p.heads, p.dim // per, p.page, 4)
    v = vc.view(p.blocks, p.heads, p.page, p.dim * es)
    nan = {1: [0x7f] * 4, 2: [0xc0, 0x7f] * 2, 4: [0, 0, 0xc0, 0x7f]}[es]
    for i, n in enumerate(p.lens):
        seen = R.sees([n - 1], max(n, 1), left, -1, sinks)[0]
        for b in range(-(-n // p.page)):
            part = seen[b * p.page:(b + 1) * p.page]
            blk = int(table[i, b])
            if not part.any():
                table[i, b] = -7
                continue
            for t in np.nonzero(~part)[0]:
                k[blk, :, :, t] = torch.tensor(nan, dtype=torch.uint8)
                v[blk, :, t] = torch.tensor(nan, dtype=torch.uint8).repeat(p.dim * es // 4)
    p.kc.copy_(kc.view(p.kc.dtype).view_as(p.kc))
    p.vc.copy_(vc.view(p.vc.dtype).view_as(p.vc))
    p.table.copy_(table)


# (lengths, heads, dim, page, left, sinks)
SHAPES = [
    ([1], 1, 64, 16, -1, 0),
    ([0, 1, 2, 15, 16, 17], 3, 32, 16, 0, 0),
    ([0, 1, 30, 100], 2, 128, 16, 7, 3),
    ([5, 63, 64, 65, 200], 5, 64, 32, 31, 1),
    ([500, 40, 511, 513], 4, 128, 48, 100, 17),
    ([300, 1000], 3, 32, 64, 299, 64),
    ([2000, 3, 700], 2, 64, 16, 600, 4),     # more than one block of keys
    ([3000, 2500], 2, 128, 16, 2047, 33),
    ([5000], 1, 128, 32, -1, 0),
    ([1500, 1, 0, 800], 2, 32, 16, -1, 9),
    ([700, 90], 7, 64, 1040, 50, 2),
    ([4000, 4100], 2, 64, 16, 4050, 5),
]


@pytest.mark.parametrize("dtype,fp8", KINDS, ids=IDS)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "-".join(map(str, s)).replace(" ", ""))
def test_against_float64(cuda, shape, dtype, fp8):
    lens, h, d, page, left, sinks = shape
    p = Paged(lens, h, d, page, dtype, sum(lens) + d, cuda, fp8=fp8)
    ref = reference(p, left, sinks)
    hide(p, left, sinks, fp8)
    out = call(p, fp8, window_size=(left, 0), sink_tokens=sinks)
    assert out.shape == p.q.shape and out.dtype == dtype
    close(out, ref, dtype)


# (lengths, heads, dim, page, left, sinks, new tokens): one token is stored by the decode
# itself up to 1024 rows and, in an 8-bit cache, pages of 64; by a kernel before it above,
# and for more tokens
APPENDS = [
    ([0, 15, 16, 40, 700, 33], 3, 64, 16, 50, 2, 1),
    ([0, 15, 16, 40, 700, 33], 3, 64, 16, 50, 2, 5),
    ([0, 15, 16, 40, 700, 33], 3, 64, 16, 50, 2, 37),
    ([0, 1, 31, 32, 33, 64, 65, 500], 2, 128, 32, 3, 0, 1),
    ([47, 48, 49, 95, 96, 10, 0, 300], 2, 32, 48, 0, 0, 1),
    ([63, 64, 100, 127, 128, 1000], 2, 64, 64, 20, 70, 1),    # sinks in the last page, or past it
    ([10, 44, 45, 46, 63], 2, 64, 64, 0, 40, 1),
    ([79, 80, 81, 200, 5], 2, 64, 80, 30, 3, 1),              # pages over 64
    ([2050, 2047, 1023, 511, 512, 513], 1, 64, 16, -1, 0, 1),  # at the ends of blocks of tiles
    ([2050, 575, 576, 577], 2, 128, 64, 559, 16, 1),
    ([3 + i % 70 for i in range(350)], 3, 32, 16, 25, 1, 1),   # 1050 rows
]


@pytest.mark.parametrize("dtype,fp8", KINDS, ids=IDS)
@pytest.mark.parametrize("shape", APPENDS, ids=lambda s: f"{len(s[0])}x{s[0][0]}-" + "-".join(map(str, s[1:])))
def test_append_of_one_and_of_many(cuda, shape, dtype, fp8):
    """New tokens are seen by the query; the cache holds them afterwards, bit for bit, and
    nothing else changes (8-bit: by the store's rule)."""
    lens, h, d, page, left, sinks, n = shape
    for size in (1.0, 300.0) if n == 1 and len(lens) < 100 else (1.0,):  # 300: every 8-bit page is rescaled
        p = Paged(lens, h, d, page, dtype, n, cuda, fp8=fp8, spare=n)
        g = torch.Generator().manual_seed(n)
        fused = (torch.randn(len(lens), n, 2, h, d, generator=g) * size).to(dtype).to(cuda)
        k, v = fused[:, :, 0], fused[:, :, 1]
        slots = [int(p.table[i, (s + j) // page]) * page + (s + j) % page for i, s in enumerate(lens) for j in range(n)]
        kr, vr = values(k).reshape(-1, h, d), values(v).reshape(-1, h, d)
        if fp8:
            want = R.Cache8(p.rows[0].copy(), p.rows[1].copy(), p.kscale.cpu().numpy(), p.vscale.cpu().numpy())
            for s in (want.scales[0], want.scales[1]):
                s[np.isnan(s)] = 0.0
            want.store(kr, vr, slots)

            def seq(i, w):
                pages = p.table[i, :-(-(lens[i] + n) // page)]
                return np.concatenate([want.values(w)[int(b)].transpose(1, 0, 2) for b in pages])[:lens[i] + n]

            p.ks, p.vs = ([seq(i, w) for i in range(len(lens))] for w in (0, 1))
        else:
            k0, v0 = p.rows_of()
            p.ks = [np.concatenate([x, kr[i * n:(i + 1) * n]]) for i, x in enumerate(p.ks)]
            p.vs = [np.concatenate([x, vr[i * n:(i + 1) * n]]) for i, x in enumerate(p.vs)]
        out = call(p, fp8, k=k, v=v, window_size=(left, -1), sink_tokens=sinks)
        k1, v1 = p.rows_of()
        if fp8:
            for got, ref in ((k1, want.codes[0]), (v1, want.codes[1])):
                assert np.array_equal(R.e4m3_decode(got.numpy()), R.e4m3_decode(ref), equal_nan=True)
            for got, w in ((p.kscale, want.scales[0]), (p.vscale, want.scales[1])):
                got = got.cpu().numpy()
                assert np.array_equal(got[~np.isnan(got)], w[~np.isnan(got)])
        else:
            es = k.element_size()
            for now, was, x in ((k1, k0, k), (v1, v0, v)):
                rows = x.reshape(-1, h, d).cpu().contiguous().view(torch.uint8)
                for s, row in zip(slots, rows):
                    was[s // page, :, s % page] = row.view(h, d * es)
                assert torch.equal(now, was)
        close(out, R.decode(values(p.q)[:, 0], p.ks, p.vs, d ** -0.5, left, sinks), dtype)


@pytest.mark.parametrize("dtype,fp8", KINDS, ids=IDS)
def test_an_open_window_is_the_whole_sequence(cuda, dtype, fp8):
    p = Paged([70, 900, 1], 2, 64, 16, dtype, 3, cuda, fp8=fp8)
    a = call(p, fp8, window_size=(-1, -1), sink_tokens=4)
    b = call(p, fp8, window_size=(10 ** 6, 0), sink_tokens=4)
    assert same_bytes(a, b)
    close(a, reference(p, -1, 0), dtype)
    if not fp8:
        close(C.flash_attn_with_kvcache(p.q, p.kc, p.vc, cache_seqlens=p.lens_t, page_table=p.table),
              reference(p, -1, 0), dtype)


@pytest.mark.parametrize("dtype,fp8", KINDS, ids=IDS)
def test_what_is_seen_may_be_nan(cuda, dtype, fp8):
    """A NaN that a row sees comes out, also where a whole tile or the query holds nothing
    else; other rows stay finite."""
    p = Paged([200, 200], 2, 64, 16, dtype, 4, cuda, fp8=fp8)
    p.q[0, 0, 1] = float("nan")
    out = call(p, fp8, window_size=(20, 0), sink_tokens=1)
    assert bool(out[0, 0, 1].isnan().all()) and bool(out[0, 0, 0].isfinite().all()) and bool(out[1].isfinite().all())
    if fp8:
        p.kscale[int(p.table[1, 12])] = float("nan")  # keys 192 ..
        out = call(p, fp8, window_size=(20, 0))
        assert bool(out[1].isnan().all()) and bool(out[0, 0, 0].isfinite().all())


@pytest.mark.parametrize("dtype,fp8", KINDS, ids=IDS)
def test_bad_pages_and_lengths_are_not_read(cuda, dtype, fp8):
    """With host checks off: page-table entries that name no block leave their keys out, a
    length past the table is cut, a negative one gives zeros and stores nothing."""
    old = K.set_host_checks(False)
    try:
        p = Paged([100, 64], 2, 64, 16, dtype, 6, cuda, fp8=fp8)
        table = p.table[:, :6].clone()
        table[0, 5] = p.blocks + 3  # keys 80 .. 95 of sequence 0
        table[0, 4] = -1            # keys 64 .. 79
        lens = torch.tensor([96, 10 ** 6], dtype=torch.int32, device=cuda)
        out = call(p, fp8, lens=lens, table=table[:, :6], window_size=(60, 0), sink_tokens=2)
        # sequence 0 stands at 95 and sees 0, 1, 35 .. 95 without 64 .. 95
        keep = [0, 1, *range(35, 64)]
        ref = R.decode(values(p.q)[:1, 0], [p.ks[0][keep]], [p.vs[0][keep]], 64 ** -0.5, -1, 0)
        close(out[:1], ref, dtype)
        lens = torch.tensor([-5, -1], dtype=torch.int32, device=cuda)
        before = p.kc.clone()
        k = torch.ones(2, 1, 2, 64, dtype=dtype, device=cuda)
        assert bool((call(p, fp8, lens=lens, k=k, v=k, window_size=(3, 0)) == 0).all())
        assert same_bytes(before, p.kc)
    finally:
        K.set_host_checks(old)


@pytest.mark.parametrize("dtype,fp8", KINDS, ids=IDS)
def test_strided_q_new_batch_index_and_cpu_indices(cuda, dtype, fp8):
    p = Paged([90, 33, 60], 3, 32, 16, dtype, 8, cuda, fp8=fp8)
    ref = reference(p, 20, 2)
    want = call(p, fp8, window_size=(20, 0), sink_tokens=2)
    close(want, ref, dtype)
    wide = torch.zeros(3, 1, 2, 3, 32, dtype=dtype, device=cuda)
    wide[:, :, 1] = p.q
    assert same_bytes(call(p, fp8, q=wide[:, :, 1], window_size=(20, 0), sink_tokens=2), want)
    odd = torch.zeros(3, 1, 3, 33, dtype=dtype, device=cuda)
    odd[..., :32] = p.q
    assert same_bytes(call(p, fp8, q=odd[..., :32], window_size=(20, 0), sink_tokens=2), want)
    assert same_bytes(call(p, fp8, lens=p.lens_t.cpu(), table=p.table.cpu(), window_size=(20, 0), sink_tokens=2), want)
    idx = torch.tensor([2, 0, 0], device=cuda)
    out = call(p, fp8, q=p.q[idx], lens=p.lens_t[idx], cache_batch_idx=idx, window_size=(20, 0), sink_tokens=2)
    assert same_bytes(out, want[idx])


@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "fp8"])
def test_offsets_past_32_bits(cuda, fp8):
    """Pages at the end of caches of more than 2^32 elements."""
    heads, dim, page = 16, 128, 64
    blocks = (1 << 32) // (heads * dim * page) + 40
    dtype = BF16
    p = Paged([130, 75], heads, dim, page, dtype, 2, cuda, fp8=fp8, spare=1)
    kc = torch.empty(blocks, heads, page, dim, dtype=p.kc.dtype, device=cuda)
    vc = torch.empty_like(kc)
    kc[-p.blocks:].view(torch.uint8).copy_(p.kc.view(torch.uint8))
    vc[-p.blocks:].view(torch.uint8).copy_(p.vc.view(torch.uint8))
    table = p.table.clone()
    table[table < p.blocks] += blocks - p.blocks
    k, v = torch.randn(2, 2, 1, heads, dim, device=cuda).to(dtype)
    want = call(p, fp8, k=k, v=v, window_size=(99, 0), sink_tokens=3)
    big = Paged.__new__(Paged)
    big.q, big.lens_t, big.table, big.kc, big.vc = p.q, p.lens_t, table, kc, vc
    if fp8:
        q = Paged([130, 75], heads, dim, page, dtype, 2, cuda, fp8=fp8, spare=1)
        big.kscale, big.vscale = (torch.zeros(blocks, heads, device=cuda) for _ in range(2))
        big.kscale[-p.blocks:], big.vscale[-p.blocks:] = q.kscale, q.vscale
    got = call(big, fp8, k=k, v=v, window_size=(99, 0), sink_tokens=3)
    assert same_bytes(got, want)
    assert same_bytes(kc[-p.blocks:], p.kc) and same_bytes(vc[-p.blocks:], p.vc)


@pytest.mark.parametrize("dtype,fp8", KINDS, ids=IDS)
@pytest.mark.parametrize("left", [40, 2500])
def test_captured_and_two_at_once(cuda, dtype, fp8, left):
    old = K.set_host_checks(False)
    try:
        p = Paged([100, 3000, 16], 2, 64, 16, dtype, 12, cuda, fp8=fp8, spare=4)
        k, v = (torch.zeros(3, 1, 2, 64, dtype=dtype, device=cuda) for _ in range(2))
        lens = p.lens_t.clone()

        def step():
            return call(p, fp8, lens=lens, k=k, v=v, window_size=(left, 0), sink_tokens=4)

        first = [x.clone() for x in (p.kc, p.vc)] + ([p.kscale.clone(), p.vscale.clone()] if fp8 else [])
        state = [p.kc, p.vc] + ([p.kscale, p.vscale] if fp8 else [])
        graph, out = capture(step)
        for i in range(3):
            g = torch.Generator().manual_seed(i)
            p.q.copy_(torch.randn(p.q.shape, generator=g))
            k.copy_(torch.randn(k.shape, generator=g) * 10 ** i)
            v.copy_(torch.randn(v.shape, generator=g))
            lens.copy_(p.lens_t + i)
            for x, y in zip(state, first):
                x.copy_(y)
            want = step().clone()
            after = [x.clone() for x in state]
            for x, y in zip(state, first):
                x.copy_(y)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert same_bytes(out, want) and all(same_bytes(x, y) for x, y in zip(state, after))
        a, b = (torch.cuda.Stream() for _ in range(2))
        torch.cuda.synchronize()
        got = []
        for s in (a, b):
            with torch.cuda.stream(s):
                got.append(call(p, fp8, window_size=(left, 0), sink_tokens=4))
        torch.cuda.synchronize()
        assert same_bytes(*got) and same_bytes(got[0], call(p, fp8, window_size=(left, 0), sink_tokens=4))
    finally:
        K.set_host_checks(old)


@pytest.mark.parametrize("dtype,fp8", KINDS, ids=IDS)
def test_bindings_agree(cuda, dtype, fp8):
    p = Paged([100, 700, 16], 2, 64, 16, dtype, 13, cuda, fp8=fp8)
    scales = (p.kscale, p.vscale) if fp8 else (None, None)
    args = (K.runtime(), p.q, p.kc, p.vc, *scales, None, None, p.lens_t, p.table, None, 50, 4, 1)
    assert same_bytes(K.module().decode_window(*args), K.ctypes_module().decode_window(*args))
    bad = (K.runtime(), p.q, p.kc, p.vc, *scales, None, None, p.lens_t.long(), p.table, None, 50, 4, 1)
    assert K.module().decode_window(*bad) is None and K.ctypes_module().decode_window(*bad) is None


def test_empty_batch_and_empty_cache(cuda):
    for fp8 in (False, True):
        p = Paged([4], 2, 64, 16, BF16, 1, cuda, fp8=fp8)
        assert call(p, fp8, q=p.q[:0], lens=p.lens_t[:0], table=p.table[:0], window_size=(3, 0)).shape == (0, 1, 2, 64)
        zero = torch.zeros(1, dtype=torch.int32, device=cuda)
        assert bool((call(p, fp8, lens=zero, table=p.table[:, :0], window_size=(3, 0)) == 0).all())


@pytest.mark.parametrize("dtype,fp8", KINDS, ids=IDS)
@pytest.mark.parametrize("seqs,heads,n", [(3, 2, 0), (3, 2, 1), (1, 1, 1), (100, 2, 1), (3, 2, 5), (70, 16, 1)])
def test_a_length_past_the_table_stores_nothing(cuda, dtype, fp8, seqs, heads, n):
    """With host checks on, whichever sequence's length it is, whether the decode stores the
    token itself or a kernel before it does."""
    p = Paged([(20 + 7 * i) % 60 for i in range(seqs)], heads, 32, 16, dtype, 14, cuda, fp8=fp8, spare=8)
    room = p.table.shape[1] * 16
    kv = {}
    if n:
        k, v = torch.randn(2, seqs, n, heads, 32, device=cuda).to(dtype) * 100
        kv = {"k": k, "v": v}
    state = [p.kc, p.vc] + ([p.kscale, p.vscale] if fp8 else [])
    before = [x.clone() for x in state]
    for i in sorted({0, seqs // 2, seqs - 1}):
        lens = p.lens_t.clone()
        lens[i] = room + 1 - n
        for where in (lens, lens.cpu()):
            with pytest.raises(ValueError, match="exceed the page table's capacity"):
                call(p, fp8, lens=where, window_size=(30, 0), sink_tokens=2, **kv)
        torch.cuda.synchronize()
        assert all(same_bytes(x, y) for x, y in zip(state, before))
    out = call(p, fp8, window_size=(30, 0), sink_tokens=2)
    close(out, reference(p, 30, 2), dtype)
    with torch.cuda.stream(torch.cuda.Stream()):
        torch.cuda.current_stream().wait_stream(torch.cuda.default_stream())
        assert same_bytes(call(p, fp8, window_size=(30, 0), sink_tokens=2), out)


@pytest.mark.parametrize("fp8", [False, True], ids=["bf16", "fp8"])
def test_longest_at_the_c_entry(cuda, fp8):
    p = Paged([100, 300, 16], 2, 64, 16, BF16, 15, cuda, fp8=fp8, spare=4)
    lib = K.load_library()
    out = torch.empty_like(p.q)
    slot = torch.full((2,), -1, dtype=torch.int64).pin_memory()
    a = K.DecodeWindowArgs()
    d = a.decode
    d.q, d.q_stride, d.out, d.lens = p.q.data_ptr(), p.q.stride(0), out.data_ptr(), p.lens_t.data_ptr()
    d.k_cache, d.v_cache = p.kc.data_ptr(), p.vc.data_ptr()
    d.page_table, d.page_table_width = p.table.data_ptr(), p.table.shape[1]
    d.scale, d.num_seqs, d.num_heads, d.head_dim = 64 ** -0.5, 3, 2, 64
    d.page_size, d.num_blocks, d.dtype = 16, p.blocks, K.DTYPES[BF16]
    a.left, a.sinks = 200, 4
    if fp8:
        a.k_scale, a.v_scale = p.kscale.data_ptr(), p.vscale.data_ptr()
    need = lib.ca_decode_window_workspace_bytes(3, 2, 64, 16, d.page_table_width, a.left, a.sinks)
    ws = torch.empty(max(need, 16), dtype=torch.uint8, device=cuda)
    d.workspace, d.workspace_bytes = ws.data_ptr(), need
    run = lambda: lib.ca_decode_window(ctypes.byref(a), torch.cuda.current_stream().cuda_stream)
    want = call(p, fp8, window_size=(200, 0), sink_tokens=4)
    for lens, longest in ((p.lens, 300), ([-4, -1, -9], 0)):
        p.lens_t.copy_(torch.tensor(lens, dtype=torch.int32))
        slot.fill_(-1)
        a.longest = slot.data_ptr()
        assert run() == K.CA_OK
        torch.cuda.synchronize()
        assert slot.tolist() == [longest, -1]
        assert same_bytes(out, want) or longest == 0 and bool((out == 0).all())
    a.longest = slot.data_ptr() + 4
    assert run() == K.CA_DECLINED
    p.lens_t.copy_(torch.tensor(p.lens, dtype=torch.int32))
    a.longest = slot.data_ptr()
    k = torch.zeros(3, 2, 2, 64, dtype=BF16, device=cuda)
    d.k_new = d.v_new = k.data_ptr()
    d.kv_stride, d.new_tokens = k.stride(1), 2
    assert run() == K.CA_DECLINED  # two new tokens each: stored ahead of the decode
    d.k_new = d.v_new = None
    d.kv_stride = d.new_tokens = 0
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        declined = run()
        a.longest = None
        captured = run()
    assert (declined, captured) == (K.CA_DECLINED, K.CA_OK)
    for _ in range(2):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert same_bytes(out, want)


@pytest.mark.parametrize("dtype,fp8", KINDS, ids=IDS)
@pytest.mark.parametrize("seqs,heads,left", [(3, 2, 1000), (3, 2, 1300), (3, 2, 1700), (3, 2, 2560), (8, 8, 1700), (8, 8, 2200),
                                             (32, 16, 900), (34, 16, 900)])
def test_rows_of_several_blocks(cuda, dtype, fp8, seqs, heads, left):
    """2 to 6 blocks of 512 keys a row, rows of one block among them: merged by the row's last
    block or by a second kernel, whatever the workspace holds, replayed in a graph too."""
    g = torch.Generator().manual_seed(16)
    lens = [int(x) for x in torch.randint(1, 2600, (seqs,), generator=g)]
    lens[0], lens[-1] = 2599, 7
    p = Paged(lens, heads, 32, 64, dtype, 17, cuda, fp8=fp8)
    lib = K.load_library()
    out = torch.empty_like(p.q)
    a = K.DecodeWindowArgs()
    d = a.decode
    d.q, d.q_stride, d.out, d.lens = p.q.data_ptr(), p.q.stride(0), out.data_ptr(), p.lens_t.data_ptr()
    d.k_cache, d.v_cache = p.kc.data_ptr(), p.vc.data_ptr()
    d.page_table, d.page_table_width = p.table.data_ptr(), p.table.shape[1]
    d.scale, d.num_seqs, d.num_heads, d.head_dim = 32 ** -0.5, seqs, heads, 32
    d.page_size, d.num_blocks, d.dtype = 64, p.blocks, K.DTYPES[dtype]
    a.left, a.sinks = left, 3
    if fp8:
        a.k_scale, a.v_scale = p.kscale.data_ptr(), p.vscale.data_ptr()
    need = lib.ca_decode_window_workspace_bytes(seqs, heads, 32, 64, d.page_table_width, left, 3)
    assert need > 0
    ws = torch.zeros(need, dtype=torch.uint8, device=cuda)
    d.workspace, d.workspace_bytes = ws.data_ptr(), need

    def run():
        assert lib.ca_decode_window(ctypes.byref(a), torch.cuda.current_stream().cuda_stream) == K.CA_OK

    run()
    first = out.clone()
    some = sorted({0, seqs // 2, seqs - 1})
    close(first[some], R.decode(values(p.q)[some, 0], [p.ks[i] for i in some], [p.vs[i] for i in some], 32 ** -0.5, left, 3),
          dtype)
    for i in range(12):
        if i % 3 == 0:
            ws.fill_(0 if i % 2 else 255)
        elif i % 3 == 1:
            ws.random_(0, 256)
        out.zero_()
        run()
        assert same_bytes(out, first)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for i in range(4):
        out.zero_()
        if i == 2:
            ws.random_(0, 256)
        graph.replay()
        torch.cuda.synchronize()
        assert same_bytes(out, first)
        run()
        assert same_bytes(out, first)
