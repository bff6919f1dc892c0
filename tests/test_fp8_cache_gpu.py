"""reshape_and_cache_fp8 against the rule in numpy, bit for bit (codes, scales, and what
stays as it was): every route, page size, type and order of slots."""

import numpy as np
import pytest
import torch

import cpu_attention as C
from cpu_attention import _kernel as K
from helpers import values
from oracle import serving as R
from serving_helpers import NAME, capture, same_bytes

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float32]
F8 = torch.float8_e4m3fn


class Pair:
    """A cache on the GPU and its oracle, with the same (random, valid) contents."""

    def __init__(self, blocks, heads, page, dim, seed=0, fresh=False):
        rng = np.random.default_rng(seed)
        shape = (blocks, heads, page, dim)
        codes = [rng.integers(0, 256, shape).astype(np.uint8) for _ in range(2)]
        scales = [np.zeros(shape[:2], np.float32) if fresh else 2.0 ** rng.integers(-12, 4, shape[:2]).astype(np.float32)
                  for _ in range(2)]
        self.ref = R.Cache8(codes[0].copy(), codes[1].copy(), scales[0].copy(), scales[1].copy())
        self.kc = torch.from_numpy(R.k_words(codes[0])).view(F8).cuda()
        self.vc = torch.from_numpy(codes[1]).view(F8).cuda()
        self.ks, self.vs = (torch.from_numpy(s.copy()).cuda() for s in scales)

    @property
    def gpu(self):
        return self.kc, self.vc, self.ks, self.vs

    def store(self, key, value, slots):
        C.reshape_and_cache_fp8(key, value, *self.gpu, torch.as_tensor(slots).cuda())
        self.ref.store(values(key), values(value), np.asarray(slots))

    def same(self):
        k = R.k_rows(self.kc.cpu().view(torch.uint8).numpy())
        v = self.vc.cpu().view(torch.uint8).numpy()
        for got, want in ((k, self.ref.codes[0]), (v, self.ref.codes[1])):
            a, b = R.e4m3_decode(got), R.e4m3_decode(want)
            assert np.array_equal(np.isnan(a), np.isnan(b)) and np.array_equal(got[~np.isnan(a)], want[~np.isnan(a)])
        assert np.array_equal(self.ks.cpu().numpy(), self.ref.scales[0].astype(np.float32))
        assert np.array_equal(self.vs.cpu().numpy(), self.ref.scales[1].astype(np.float32))


def tokens(n, heads, dim, dtype, seed, size=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(2, n, heads, dim, generator=g) * torch.exp(torch.randn(2, n, heads, 1, generator=g)) * size
    return x[0].to(dtype).cuda(), x[1].to(dtype).cuda()


def test_conversion_of_every_code_and_every_tie(cuda):
    """One page whose scale is 1 (an element of 448): its codes are e4m3's own rounding."""
    vals = R.e4m3_values()[:127]
    ties = np.concatenate([vals, (vals[1:] + vals[:-1]) / 2, np.nextafter(np.float32((vals[1:] + vals[:-1]) / 2), 1e9)])
    x = np.concatenate([ties, -ties]).astype(np.float32)
    x = np.resize(x, (16 * 2, 2, 32))
    x[:, :, 0] = 448.0
    key = torch.from_numpy(x).cuda()
    p = Pair(2, 2, 16, 32, fresh=True)
    p.store(key, key.flip(0).contiguous(), np.arange(32))
    p.same()
    assert bool((p.ks == 1.0).all())
    back = p.vc.float() * p.vs[..., None, None]
    want = key.flip(0).view(2, 16, 2, 32).transpose(1, 2).to(F8).float()
    assert torch.equal(back, want)


# (heads, dim, page, tokens): scan route up to 512 tokens and pages of up to 1024, lists above
SHAPES = [(1, 32, 16, 1), (3, 64, 16, 5), (5, 128, 16, 40), (2, 32, 48, 100), (4, 64, 64, 300), (2, 128, 256, 700),
          (3, 32, 1024, 500), (2, 64, 1040, 500), (1, 128, 1040, 1300), (3, 64, 16, 512), (3, 64, 16, 513),
          (6, 128, 32, 2000), (1, 32, 16, 5000)]


@pytest.mark.parametrize("dtype", DTYPES, ids=NAME.get)
@pytest.mark.parametrize("order", ["rising", "random"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "-".join(map(str, s)))
def test_store(cuda, shape, order, dtype):
    heads, dim, page, n = shape
    blocks = -(-n // page) + 3
    rng = np.random.default_rng(n + dim)
    p = Pair(blocks, heads, page, dim, seed=n)
    slots = rng.permutation(blocks * page)[:n] if order == "random" else np.arange(n) + 7
    slots = np.where(rng.random(n) < 0.1, -1 - rng.integers(0, 5, n), slots)
    key, value = tokens(n, heads, dim, dtype, n)
    p.store(key, value, slots)
    p.same()


@pytest.mark.parametrize("dtype", DTYPES, ids=NAME.get)
@pytest.mark.parametrize("n", [300, 1500])
def test_slots_named_more_than_once_take_the_last_token(cuda, dtype, n):
    rng = np.random.default_rng(n)
    p = Pair(6, 3, 32, 64, seed=1)
    key, value = tokens(n, 3, 64, dtype, 2)
    p.store(key, value, rng.integers(0, 6 * 32, n))
    p.same()
    # the scale goes by the tokens that stay
    key[0], value[0] = 1e6, 1e6
    p.store(key[:2], value[:2], np.array([5, 5]))
    p.same()


@pytest.mark.parametrize("dtype", DTYPES, ids=NAME.get)
@pytest.mark.parametrize("page", [16, 48])
def test_token_by_token_growth(cuda, dtype, page):
    """Pages filled one token a call, each larger or smaller than the ones before, then
    started anew."""
    p = Pair(3, 2, page, 32, fresh=True)
    for t in range(page + 5):
        key, value = tokens(2, 2, 32, dtype, t, size=2.0 ** (t % 7 - 2 + (t > 9) * 6))
        p.store(key, value, np.array([t, 2 * page + t % page]))
        p.same()


@pytest.mark.parametrize("dtype", DTYPES, ids=NAME.get)
def test_extreme_values(cuda, dtype):
    """Zeros, the type's smallest and largest, infinities and NaNs, in pages begun and not."""
    big = torch.finfo(dtype).max
    rows = [0.0, -0.0, 1e-45, torch.finfo(dtype).tiny, 2.0 ** -100, 448.0 * 2.0 ** -100, 1.0, big, -big, float("inf"),
            -float("inf"), float("nan")]
    for begin in (0, 1):
        for fresh in (True, False):
            p = Pair(len(rows), 2, 16, 32, seed=3, fresh=fresh)
            key = torch.zeros(len(rows), 2, 32, device=cuda)
            key[:, :, 5] = torch.tensor(rows, device=cuda)[:, None]
            key[:, 1, 9] = 0.5
            p.store(key.to(dtype), key.to(dtype).flip(1).contiguous(), np.arange(len(rows)) * 16 + begin)
            p.same()


@pytest.mark.parametrize("n", [40, 1200])
def test_padding_of_any_content_changes_nothing(cuda, n):
    p = Pair(90, 2, 16, 64, seed=4)
    before = [x.clone() for x in p.gpu]
    key = torch.full((n, 2, 64), float("nan"), device=cuda)
    p.store(key, key.clone(), np.full(n, -1))
    assert all(same_bytes(a, b) for a, b in zip(before, p.gpu))
    C.reshape_and_cache_fp8(key[:0], key[:0], *p.gpu, torch.zeros(0, dtype=torch.int64, device=cuda))
    slots = np.where(np.arange(n) % 3, -1, np.arange(n))
    key[torch.from_numpy(slots >= 0).cuda()] = 2.0
    p.store(key, key.clone(), slots)
    p.same()
    old = K.set_host_checks(False)
    try:
        before = [x.clone() for x in p.gpu]
        far = torch.full((n,), 90 * 16, dtype=torch.int64, device=cuda)
        far[1::2] = 1 << 60
        C.reshape_and_cache_fp8(key, key.clone(), *p.gpu, far)  # past the cache: not stored
        assert all(same_bytes(a, b) for a, b in zip(before, p.gpu))
    finally:
        K.set_host_checks(old)


@pytest.mark.parametrize("dtype", DTYPES, ids=NAME.get)
def test_views(cuda, dtype):
    """K and V of a fused projection, a token broadcast, unaligned rows, CPU slots."""
    g = torch.Generator().manual_seed(1)
    p = Pair(4, 3, 16, 64, seed=5)
    fused = torch.randn(30, 3, 3, 64, generator=g).to(dtype).cuda()
    p.store(fused[:, 1], fused[:, 2], np.arange(30)[::-1].copy() + 3)
    p.same()
    one = torch.randn(1, 3, 64, generator=g).to(dtype).cuda()
    p.store(one.expand(9, -1, -1), one.expand(9, -1, -1), np.arange(9) + 20)
    p.same()
    odd = torch.randn(2, 9, 3, 65, generator=g).to(dtype).cuda()[..., 1:]
    p.store(odd[0], odd[1], np.arange(9) + 33)
    p.same()
    C.reshape_and_cache_fp8(fused[:5, 0], fused[:5, 1], *p.gpu, torch.arange(5))
    p.ref.store(values(fused[:5, 0]), values(fused[:5, 1]), np.arange(5))
    p.same()


@pytest.mark.parametrize("n", [50, 1100])
def test_captured_and_repeated(cuda, n):
    """Replays of a captured store, each against an eager one from the same contents."""
    old = K.set_host_checks(False)
    try:
        p = Pair(n // 16 + 4, 2, 16, 64, seed=6)
        first = [x.clone() for x in p.gpu]
        key, value = tokens(n, 2, 64, torch.bfloat16, 0)
        slots = torch.zeros(n, dtype=torch.int64, device=cuda)

        def store():
            C.reshape_and_cache_fp8(key, value, *p.gpu, slots)

        graph, _ = capture(store)
        for i in range(3):
            k, v = tokens(n, 2, 64, torch.bfloat16, i + 1)
            key.copy_(k)
            value.copy_(v)
            slots.copy_(torch.randperm((n // 16 + 4) * 16, generator=torch.Generator().manual_seed(i))[:n])
            for x, y in zip(p.gpu, first):
                x.copy_(y)
            store()
            want = [x.clone() for x in p.gpu]
            for x, y in zip(p.gpu, first):
                x.copy_(y)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert all(same_bytes(x, y) for x, y in zip(p.gpu, want))
    finally:
        K.set_host_checks(old)


def test_bindings_agree(cuda):
    for n in (20, 1100):
        a, b = Pair(90, 2, 16, 64, seed=7), Pair(90, 2, 16, 64, seed=7)
        key, value = tokens(n, 2, 64, torch.bfloat16, 3)
        slots = torch.randperm(90 * 16, generator=torch.Generator().manual_seed(0))[:n].cuda()
        assert K.module().store_fp8(K.runtime(), key, value, *a.gpu, slots) is True
        assert K.ctypes_module().store_fp8(K.runtime(), key, value, *b.gpu, slots) is True
        assert all(same_bytes(x, y) for x, y in zip(a.gpu, b.gpu))


def test_no_heads_and_no_pages(cuda):
    for heads, blocks in ((0, 4), (2, 0)):
        kc, vc = (torch.zeros(blocks, heads, 16, 64, device=cuda).to(torch.float8_e4m3fn) for _ in range(2))
        ks, vs = (torch.zeros(blocks, heads, device=cuda) for _ in range(2))
        key = torch.ones(3, heads, 64, device=cuda)
        C.reshape_and_cache_fp8(key, key, kc, vc, ks, vs, torch.full((3,), -1, device=cuda))
        assert K.ctypes_module().store_fp8(K.runtime(), key, key, kc, vc, ks, vs, torch.full((3,), -1, device=cuda)) is True
