"""copy_blocks, byte for byte: types, many layers, padding, pages of a size that fills no
whole piece, captured, and an 8-bit cache's scales."""

import numpy as np
import pytest
import torch

import cpu_attention as C
from cpu_attention import _kernel as K
from oracle import serving as R
from serving_helpers import capture, same_bytes

pytestmark = pytest.mark.gpu
F8 = torch.float8_e4m3fn


def caches(layers, blocks, heads, page, dim, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    es = torch.empty(0, dtype=dtype).element_size()
    made = [torch.randint(0, 256, (blocks, heads, page, dim * es), generator=g, device="cuda", dtype=torch.uint8).view(dtype)
            for _ in range(2 * layers)]
    scales = [torch.rand(blocks, heads, generator=g, device="cuda") for _ in range(2 * layers)]
    return made[:layers], made[layers:], scales[:layers], scales[layers:]


def copied(x, pairs):
    return torch.from_numpy(R.copy_pages(x.contiguous().view(torch.uint8).cpu().numpy(), pairs))


def pairs_of(blocks, n, seed):
    rng = np.random.default_rng(seed)
    order = rng.permutation(blocks)
    src, dst = order[:n], order[n:2 * n]
    src = rng.choice(src, n)  # a page may be copied to several
    pairs = np.stack([src, dst], 1)
    pairs[rng.random(n) < 0.15, rng.integers(0, 2)] = -1  # padding
    return pairs


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, F8], ids=["bf16", "fp32", "fp8"])
@pytest.mark.parametrize("shape", [(1, 2, 1, 16, 32, 1), (3, 40, 3, 16, 64, 17), (2, 30, 5, 48, 128, 15),
                                   (70, 9, 1, 16, 32, 4), (1, 600, 4, 32, 128, 300), (2, 8, 32, 64, 128, 3)],
                         ids=lambda s: "-".join(map(str, s)))
def test_copies(cuda, shape, dtype):
    layers, blocks, heads, page, dim, n = shape
    kc, vc, ks, vs = caches(layers, blocks, heads, page, dim, dtype)
    pairs = pairs_of(blocks, n, n)
    lists = [kc, vc] + ([ks, vs] if dtype == F8 else [])
    want = [[copied(x, pairs) for x in xs] for xs in lists]
    mapping = torch.from_numpy(pairs).cuda()
    kw = dict(key_scales=ks, value_scales=vs) if dtype == F8 else {}
    C.copy_blocks(kc, vc, mapping, **kw)
    for xs, ws in zip(lists, want):
        for x, w in zip(xs, ws):
            assert torch.equal(x.contiguous().view(torch.uint8).cpu().view(-1), w.view(-1))
    before = [x.clone() for x in kc]
    C.copy_blocks(kc, vc, mapping[:0], **kw)
    C.copy_blocks(kc, vc, torch.tensor([[1, 1], [0, 0]]), **kw)  # to themselves
    assert all(same_bytes(x, y) for x, y in zip(before, kc))


@pytest.mark.parametrize("where", ["cpu", "cuda"])
def test_what_cannot_be_copied_at_once_is_refused(cuda, where):
    kc, vc, _, _ = caches(1, 8, 2, 16, 32, torch.bfloat16)
    before = kc[0].clone()
    for pairs, msg in (([[0, 1], [2, 1]], "twice"), ([[0, 1], [1, 2]], "overwrites"), ([[0, 1], [1, 0]], "overwrites"),
                       ([[0, 8]], "past the end"), ([[9, 1]], "past the end"), ([[3, 4], [3, 4]], "twice")):
        with pytest.raises(ValueError, match=msg):
            C.copy_blocks(kc, vc, torch.tensor(pairs, device=where))
    assert same_bytes(before, kc[0])
    C.copy_blocks(kc, vc, torch.tensor([[0, 1], [0, 2], [5, -1], [-1, 0]], device=where))  # one source, two copies
    assert same_bytes(kc[0][1], before[0]) and same_bytes(kc[0][2], before[0]) and same_bytes(kc[0][0], before[0])


def test_past_the_cache_without_checks(cuda):
    old = K.set_host_checks(False)
    try:
        kc, vc, _, _ = caches(1, 8, 2, 16, 32, torch.bfloat16)
        before = kc[0].clone()
        C.copy_blocks(kc, vc, torch.tensor([[0, 8], [1 << 40, 2], [3, 1 << 40], [1, 4]], device=cuda))
        before[4] = before[1]
        assert same_bytes(before, kc[0])
    finally:
        K.set_host_checks(old)


def test_offsets_past_32_bits(cuda):
    heads, page, dim = 16, 64, 128
    blocks = (1 << 32) // (heads * page * dim) + 9
    kc, vc = (torch.zeros(blocks, heads, page, dim, dtype=F8, device=cuda) for _ in range(2))
    ks, vs = (torch.zeros(blocks, heads, device=cuda) for _ in range(2))
    kc[-1].view(torch.uint8).fill_(7)
    vc[-2].view(torch.uint8).fill_(9)
    ks[-1] = 3.0
    C.copy_blocks([kc], [vc], torch.tensor([[blocks - 1, 0], [blocks - 2, blocks - 5]]), key_scales=[ks], value_scales=[vs])
    assert bool((kc[0].view(torch.uint8) == 7).all()) and bool((vc[-5].view(torch.uint8) == 9).all())
    assert bool((ks[0] == 3.0).all())


def test_captured(cuda):
    old = K.set_host_checks(False)
    try:
        kc, vc, ks, vs = caches(2, 50, 3, 16, 64, F8)
        mapping = torch.full((20, 2), -1, dtype=torch.int64, device=cuda)
        graph, _ = capture(lambda: C.copy_blocks(kc, vc, mapping, key_scales=ks, value_scales=vs))
        for i in range(3):
            pairs = pairs_of(50, 20, i)
            mapping.copy_(torch.from_numpy(pairs))
            want = [copied(x, pairs) for x in (*kc, *vc, *ks, *vs)]
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            for x, w in zip((*kc, *vc, *ks, *vs), want):
                assert torch.equal(x.contiguous().view(torch.uint8).cpu().view(-1), w.view(-1))
    finally:
        K.set_host_checks(old)


def test_bindings_agree(cuda):
    mapping = torch.tensor([[0, 3], [1, 4]], device=cuda)
    a, b = caches(2, 8, 2, 16, 64, F8), caches(2, 8, 2, 16, 64, F8)
    assert K.module().copy_blocks(K.runtime(), *a, mapping) is True
    assert K.ctypes_module().copy_blocks(K.runtime(), *b, mapping) is True
    assert all(same_bytes(x, y) for xs, ys in zip(a, b) for x, y in zip(xs, ys))
    for mod in (K.module(), K.ctypes_module()):
        assert mod.copy_blocks(K.runtime(), *a, mapping.int()) is None
        assert mod.copy_blocks(K.runtime(), a[0], a[1], None, None, mapping) is None  # 8-bit, no scales
        assert mod.copy_blocks(K.runtime(), a[0], a[1][:1], a[2], a[3], mapping) is None
        assert mod.copy_blocks(K.runtime(), a[0], a[1], a[2], a[2], mapping) is None  # K's scales for V
        assert mod.copy_blocks(K.runtime(), [], [], None, None, mapping) is True
