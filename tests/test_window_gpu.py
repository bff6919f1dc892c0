"""flash_attn_window_func against the float64 oracle, within bounds derived from the
arithmetic (oracle/serving.py, Rows.bound): sizes on both sides of every route, sides and
sinks that cut tiles, rows that see nothing, values that must not be seen."""

import numpy as np
import pytest
import torch

import cpu_attention as C
from cpu_attention import _kernel as K
from helpers import values
from oracle import serving as R
from serving_helpers import NAME, capture, close, same_bytes

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float32]
BF16, FP32 = DTYPES


def inputs(N, L, S, H, E, dtype, seed=0, device="cuda", size=1.0):
    g = torch.Generator().manual_seed(seed)
    return tuple((torch.randn(N, n, H, E, generator=g) * s).to(dtype).to(device)
                 for n, s in ((L, size), (S, 1.0), (S, 1.0)))


def check(q, k, v, left, right, sinks, causal, scale=None):
    out = C.flash_attn_window_func(q, k, v, window_size=(left, right), sink_tokens=sinks, softmax_scale=scale,
                                   causal=causal)
    assert out.shape == q.shape and out.dtype == q.dtype and out.is_contiguous()
    ref = R.window(values(q), values(k), values(v), scale or q.shape[-1] ** -0.5, left, right, sinks, causal)
    close(out, ref, q.dtype, rounds_p=q.dtype == BF16)
    return out


# (N, L, S, H, E, left, right, sinks, causal); bf16 routes by items = N H ceil(L / 128) and the
# tiles a block can have: up to 256 keys one wave per 32 rows, then key groups past 8 tiles up to
# 256 items, splits from 16 tiles up to 64 items and from 40 up to 170, one group otherwise.
# fp32: split operands from 64 (E = 128), 80 (64) or 160 (32) 128-row blocks; 32-bit MFMAs in
# 128-row blocks from 256 (E = 128: 192) of them, 32-row ones from 256, else 16-row ones, split
# from 4 tiles of 128 keys where they leave half of the CUs idle.
SHAPES = [
    (1, 1, 1, 1, 64, 0, 0, 0, True),
    (1, 1, 77, 2, 32, 3, 0, 2, True),
    (2, 5, 5, 3, 128, 2, 1, 0, False),
    (1, 64, 64, 2, 64, 0, 0, 1, True),
    (1, 100, 100, 2, 32, 31, 0, 4, True),
    (2, 129, 129, 3, 64, 40, 0, 0, True),
    (1, 300, 300, 2, 128, 64, 0, 5, True),
    (1, 333, 700, 3, 64, 100, 7, 70, False),
    (1, 700, 333, 3, 64, 100, 0, 4, True),      # the first rows see no key
    (1, 400, 90, 2, 128, 50, 20, 3, False),     # rows before the first key, rows that see it late
    (1, 600, 600, 2, 32, 200, 300, 0, False),
    (1, 257, 1500, 2, 128, -1, 40, 0, False),   # open to the left
    (1, 257, 1500, 2, 64, 300, -1, 9, False),   # open to the right
    (1, 700, 700, 4, 64, 600, 0, 4, True),      # two key groups
    (1, 1000, 1000, 3, 128, 800, 0, 64, True),
    (1, 40, 3000, 2, 64, 2500, 0, 4, True),     # splits
    (2, 130, 2500, 3, 128, 2100, 3, 65, False),
    (1, 4, 4000, 8, 32, 3000, 0, 1, True),
    (1, 8, 40000, 1, 64, 39000, 0, 4, True),    # as many as the combine merges
    (1, 1, 20000, 2, 128, 19000, 0, 1, True),
    (1, 700, 6000, 12, 64, 4500, 0, 4, True),   # 72 and 108 items
    (1, 600, 6000, 22, 32, 4500, 100, 0, False),
    (3, 700, 700, 50, 32, 90, 0, 4, True),      # more items than 256
    (2, 500, 500, 40, 64, 450, 0, 130, True),
    (1, 1100, 1100, 33, 128, 129, 0, 16, True),
    (5, 130, 130, 40, 128, 30, 0, 2, True),
]


@pytest.mark.parametrize("dtype", DTYPES, ids=NAME.get)
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: "-".join(map(str, s)))
def test_against_float64(cuda, shape, dtype):
    N, L, S, H, E, left, right, sinks, causal = shape
    check(*inputs(N, L, S, H, E, dtype, seed=L + S), left, right, sinks, causal)


def test_random_sizes(cuda):
    rng = np.random.default_rng(7)
    for i in range(60):
        S = int(np.exp(rng.uniform(0, np.log(900))))
        L = S if rng.random() < 0.6 else int(rng.integers(1, 400))
        causal = bool(rng.random() < 0.7)
        case = (int(rng.integers(1, 3)), L, S, int(rng.integers(1, 6)), int(rng.choice([32, 64, 128])),
                int(rng.integers(0, S + 2)), int(rng.integers(0, 100)), int(rng.choice([0, 1, 4, 63, 64, 65, 200])), causal)
        N, L, S, H, E, left, right, sinks, causal = case
        print(i, case, flush=True)
        check(*inputs(N, L, S, H, E, DTYPES[i % 2], seed=i), left, right, sinks, causal)


@pytest.mark.parametrize("dtype", DTYPES, ids=NAME.get)
def test_views_are_read_in_place(cuda, dtype):
    """Slices of a fused projection, a broadcast batch, and heads before tokens."""
    g = torch.Generator().manual_seed(3)
    fused = torch.randn(2, 150, 3, 4, 64, generator=g).to(dtype).cuda()
    check(fused[:, :, 0], fused[:, :, 1], fused[:, :, 2], 40, 0, 4, True)
    q, k, v = inputs(1, 150, 150, 4, 64, dtype)
    check(q.expand(3, -1, -1, -1), k.expand(3, -1, -1, -1), v.expand(3, -1, -1, -1), 40, 0, 4, True)
    t = torch.randn(3, 2, 4, 150, 64, generator=g).to(dtype).cuda().transpose(2, 3)
    check(t[0], t[1], t[2], 40, 0, 4, True)
    odd = torch.randn(3, 2, 150, 4, 65, generator=g).to(dtype).cuda()[..., :64]  # copied: rows not 16-byte aligned
    check(odd[0], odd[1], odd[2], 40, 0, 4, True)


@pytest.mark.parametrize("dtype", DTYPES, ids=NAME.get)
def test_open_windows_are_flash_attn_func(cuda, dtype):
    q, k, v = inputs(2, 200, 300, 3, 64, dtype)
    for window, causal in (((-1, -1), False), ((-1, -1), True), ((299, 0), False), ((-1, 0), False), ((400, 199), False)):
        got = C.flash_attn_window_func(q, k, v, window_size=window, sink_tokens=4, causal=causal)
        want = C.flash_attn_func(q, k, v, causal=causal or window[1] == 0)
        assert same_bytes(got, want)


@pytest.mark.parametrize("dtype", DTYPES, ids=NAME.get)
@pytest.mark.parametrize("shape", [(1, 300, 300, 2, 64, 50, 0, 4), (1, 700, 700, 2, 128, 600, 0, 4),
                                   (1, 40, 3000, 2, 64, 2500, 0, 4), (4, 300, 300, 40, 32, 100, 0, 70)],
                         ids=lambda s: "-".join(map(str, s)))
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_unseen_values_stay_out(cuda, dtype, shape, bad):
    """Keys that only some rows see hold NaN or an infinity in K, in V, or in both: the rows
    that do not see them are as without, and the others as the formula has it."""
    N, L, S, H, E, left, right, sinks = shape
    q, k, v = inputs(N, L, S, H, E, dtype, seed=5)
    edge = max(sinks, S - L // 2 - 1 - left)  # the middle row's first key (no sink)
    at = [edge, edge + 1, S - 3]
    for x in ((v,), (k,), (k, v)):
        kk, vv = k.clone(), v.clone()
        for j in at:
            if x[0] is k:
                kk[0, j, 0, 3] = bad
            if x[-1] is v:
                vv[0, j, 0, 5] = bad
        out = C.flash_attn_window_func(q, kk, vv, window_size=(left, right), sink_tokens=sinks)
        ref = R.window(values(q), values(kk), values(vv), E ** -0.5, left, right, sinks, False)
        clean = R.window(values(q), values(k), values(v), E ** -0.5, left, right, sinks, False)
        seen = R.sees(np.arange(L) + S - L, S, left, right, sinks)[:, at].any(1)
        got = values(out)
        assert (~seen).sum() > 0 and seen.sum() > 0
        touched = np.zeros(got.shape, bool)
        touched[0, seen, 0] = True
        err = np.abs(got - clean.out)
        assert np.all(np.isfinite(got[~touched])) and np.all(err[~touched] <= clean.bound(NAME[dtype], True)[~touched])
        # rows that see it: not finite where the formula is not
        assert np.array_equal(np.isnan(got[touched]), np.isnan(ref.out[touched]))


@pytest.mark.parametrize("dtype", DTYPES, ids=NAME.get)
def test_nan_queries_stay_in_their_rows(cuda, dtype):
    for N, L, S, H, E, left in ((1, 200, 100, 2, 64, 60), (1, 700, 700, 2, 128, 600), (1, 40, 3000, 2, 64, 2500)):
        q, k, v = inputs(N, L, S, H, E, dtype, seed=13)
        q[0, 3::7, 1, 2] = float("nan")
        check(q, k, v, left, 0, 4, True)


@pytest.mark.parametrize("dtype", DTYPES, ids=NAME.get)
def test_inputs_of_nothing_but_nans(cuda, dtype):
    """NaN wherever a row sees a key, soon; zeros elsewhere."""
    for N, L, S, H, E, left in ((1, 200, 100, 2, 64, 60), (1, 3000, 3000, 4, 128, 2000), (1, 40, 9000, 2, 64, 8000)):
        q, k, v = (torch.full_like(x, float("nan")) for x in inputs(N, L, S, H, E, dtype))
        out = C.flash_attn_window_func(q, k, v, window_size=(left, 0), sink_tokens=4)
        some = torch.arange(L, device=cuda) + S - L >= 0
        assert bool(out[:, some].isnan().all()) and bool((out[:, ~some] == 0).all())


@pytest.mark.parametrize("dtype", DTYPES, ids=NAME.get)
@pytest.mark.parametrize("level", [-600.0, -90.0, 90.0, 600.0])
def test_sinks_far_from_the_window(cuda, dtype, level):
    """Sink logits far above or below the window's: the running max has to follow."""
    for N, L, S, H, E, left in ((1, 500, 500, 2, 64, 60), (1, 700, 700, 2, 128, 600), (1, 40, 3000, 2, 64, 2500)):
        q, k, v = inputs(N, L, S, H, E, dtype, seed=9)
        q[..., 0] = 8.0
        k[..., 0] = 0.0
        k[:, :4, :, 0] = level / (8.0 * E ** -0.5)
        check(q, k, v, left, 0, 4, True)


@pytest.mark.parametrize("dtype", DTYPES, ids=NAME.get)
def test_lowest_values_and_large_logits(cuda, dtype):
    """Logits of about +-1e4 and values near the type's largest."""
    q, k, v = inputs(1, 200, 200, 2, 64, dtype, seed=11, size=500.0)
    out = C.flash_attn_window_func(q, k, v * 1e37, window_size=(50, 0), sink_tokens=2, causal=True)
    # Rows are close to one-hot: compared with the oracle on the inputs' own exponents,
    # the logits' rounding (E + 8 roundings of their size) in the bound.
    ref = R.window(values(q), values(k), values(v * 1e37), 64 ** -0.5, 50, 0, 2, True)
    close(out, ref, dtype, rounds_p=dtype == BF16)


@pytest.mark.parametrize("dtype", DTYPES, ids=NAME.get)
def test_empty_batch_and_scale(cuda, dtype):
    q, k, v = inputs(0, 5, 5, 2, 64, dtype)
    assert C.flash_attn_window_func(q, k, v, window_size=(1, 0)).shape == q.shape
    check(*inputs(1, 50, 50, 2, 64, dtype), 9, 0, 1, True, scale=0.7)


@pytest.mark.parametrize("dtype", DTYPES, ids=NAME.get)
@pytest.mark.parametrize("shape", [(1, 300, 300, 3, 64, 50), (1, 40, 3000, 2, 64, 2500)])
def test_captured_and_on_another_stream(cuda, dtype, shape):
    N, L, S, H, E, left = shape
    q, k, v = inputs(N, L, S, H, E, dtype)

    def call():
        return C.flash_attn_window_func(q, k, v, window_size=(left, 0), sink_tokens=4)

    graph, out = capture(call)
    for seed in (1, 2, 3):
        for x, y in zip((q, k, v), inputs(N, L, S, H, E, dtype, seed=seed)):
            x.copy_(y)
        want = call()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert same_bytes(out, want)
        inputs(1, 500, 500, 4, 128, dtype)  # other work between the replays
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for s in streams:  # two calls at once
        with torch.cuda.stream(s):
            got.append(call())
    torch.cuda.synchronize()
    assert all(same_bytes(x, want) for x in got)


@pytest.mark.parametrize("dtype", DTYPES, ids=NAME.get)
def test_bindings_agree(cuda, dtype):
    q, k, v = inputs(1, 200, 300, 3, 64, dtype)
    rt, mod = K.runtime(), K.ctypes_module()
    for left, right, sinks, causal in ((40, 0, 4, True), (250, 3, 1, False), (-1, -1, 0, False)):
        a = K.module().flash_window(rt, q, k, v, None, causal, left, right, sinks)
        b = mod.flash_window(rt, q, k, v, None, causal, left, right, sinks)
        assert same_bytes(a, b)
    assert K.module().flash_window(rt, q, k[:, :, :2], v, None, True, 4, 0, 0) is None
    assert mod.flash_window(rt, q, k[:, :, :2], v, None, True, 4, 0, 0) is None


# fp32 calls on split operands: two key groups and one at each head dim, rows of two blocks.
SPLIT = [(2, 130, 500, 24, 64), (5, 130, 500, 32, 64), (2, 130, 500, 16, 128), (5, 130, 500, 32, 128),
         (3, 130, 500, 32, 32), (9, 130, 500, 32, 32), (1, 1030, 1030, 10, 64), (1, 1100, 1100, 8, 128)]


def _spoil(kind, q, k, v):
    if kind == "sinks":            # keys with logits far above the others, values near none
        k[:, :4] *= 6
        v[:, :4] *= 2.0 ** -6
    elif kind == "growing keys":   # past what the first tile's scale holds
        k[:, 250:] *= 300
        q *= 2.0 ** -8
    elif kind == "wide column":
        v[..., 5] *= 1e4
    elif kind == "zero columns":
        v[..., 3:17] = 0
    elif kind == "late column":    # zeros in the first tiles only
        v[:, :300, :, 7] = 0
    elif kind == "zeros":
        q[:, ::3] = 0
        k[:, 40:90] = 0
        v[:, 200:260] = 0
    elif kind == "tiny":
        q *= 1e-18
        k *= 1e-18
        v *= 1e-30
    elif kind == "peaked":
        q *= 30
    elif kind == "uneven":
        g = torch.Generator().manual_seed(3)
        k *= torch.randn(k.shape, generator=g).mul(1.5).exp().to(k.device)
        v *= torch.randn(v.shape, generator=g).mul(2).exp().to(v.device)
    elif kind == "late nan":       # seen by the last rows only
        v[0, -1, 1, 2] = float("nan")
        k[0, -2, 0, 1] = float("inf")


def _check_split(q, k, v, left, parts):
    """A call on split operands: they hold values near their tile's largest; blocks where that
    costs a row too much are done in 32-bit MFMAs.  Beside fp32's own errors there are the
    quanta of values whose low half is subnormal: q', k', v', p' (scaled) are each off by at
    most 2^-25.
      V's: in a dim, 2^-25 sum p'.  The kernel keeps a block only if top^2 >= 2^10 sum p' (top:
        the row's largest |O'|), and p' <= 2^14, so sum p' <= sqrt(n 2^14) top / 2^5: at most
        2^-23 sqrt(n) top over n keys.
      P's: 2^-25 sum |v'| <= 2^-25 sqrt(n) sqrt(sum v'^2), and top^2 >= sum v'^2 / 2^6: at most
        2^-22 sqrt(n) top, n the keys staged (the rows' and up to 191 around them).
      the logits': c 2^-25 E (2^11 + |k'|), and c max(2^11, |k'|) <= max(1, X / 2) / 2 for a
        logit of X log2 units: at most E 2^-25 max(1, X / 2), X / 2 times it within fp32's own
        logit term, once it in numerator and denominator each: E 2^-24.
    top is at most the largest sum p |v| of a dim, in each of the `parts` (key groups or
    splits) that share the keys: sqrt(parts n) over all."""
    N, L, H, E = q.shape
    out = C.flash_attn_window_func(q, k, v, window_size=(left, 0), sink_tokens=4, causal=True)
    ref = R.window(values(q), values(k), values(v), E ** -0.5, left, 0, 4, True)
    n = left + 5 + 191
    top = np.where(np.isfinite(ref.size), ref.size, 0).max(-1, keepdims=True)
    bound = ref.bound("fp32", False) + E * 2.0 ** -24 * ref.size + (2.0 ** -23 + 2.0 ** -22) * (parts * n) ** 0.5 * top
    got, nan = values(out), np.isnan(ref.out)
    assert np.array_equal(np.isnan(got), nan)
    fine = np.isfinite(ref.out)
    assert np.array_equal(got[~fine & ~nan], ref.out[~fine & ~nan])
    assert np.all(np.abs(got - ref.out)[fine] <= bound[fine]), np.max((np.abs(got - ref.out) / bound)[fine])


KINDS = ["normal", "sinks", "growing keys", "wide column", "zero columns", "late column", "zeros", "tiny", "peaked", "uneven",
         "late nan"]


@pytest.mark.parametrize("shape", SPLIT, ids=lambda s: "-".join(map(str, s)))
@pytest.mark.parametrize("kind", KINDS)
def test_fp32_values_of_every_size(cuda, shape, kind):
    N, L, S, H, E = shape
    q, k, v = inputs(N, L, S, H, E, torch.float32, seed=E + H)
    _spoil(kind, q, k, v)
    _check_split(q, k, v, 270, 2)


# Few blocks over long windows share their tiles out: 7, 11 and 11 splits.
@pytest.mark.parametrize("shape", [(1, 256, 2000, 8, 64, 1900), (1, 130, 3001, 6, 128, 2800), (2, 100, 3001, 10, 32, 2800)],
                         ids=lambda s: "-".join(map(str, s)))
@pytest.mark.parametrize("kind", KINDS)
def test_fp32_splits_of_every_size(cuda, shape, kind):
    N, L, S, H, E, left = shape
    q, k, v = inputs(N, L, S, H, E, torch.float32, seed=E + H)
    _spoil(kind, q, k, v)
    _check_split(q, k, v, left, 11)


def test_fp32_split_operands_captured(cuda):
    """Replays of a call whose blocks stay on the split operands in one and are redone in the
    next, a workspace of any contents."""
    N, L, S, H, E = SPLIT[0]
    q, k, v = inputs(N, L, S, H, E, torch.float32)

    def call():
        return C.flash_attn_window_func(q, k, v, window_size=(270, 0), sink_tokens=4, causal=True)

    graph, out = capture(call)
    for i, kind in enumerate(("normal", "wide column", "normal", "late nan", "normal")):
        for x, y in zip((q, k, v), inputs(N, L, S, H, E, torch.float32, seed=i)):
            x.copy_(y)
        _spoil(kind, q, k, v)
        want = call()
        graph.replay()
        torch.cuda.synchronize()
        assert same_bytes(out, want)


@pytest.mark.parametrize("dtype", DTYPES, ids=NAME.get)
@pytest.mark.parametrize("shape", [(1, 1100, 1100, 60, 128, 800, 0, 4), (1, 1100, 1300, 57, 128, 1200, 3, 0),
                                   (1, 2100, 2100, 16, 128, 1700, 0, 4), (1, 1990, 1990, 17, 128, 1500, 0, 70),
                                   (8, 260, 260, 50, 64, 220, 0, 4), (7, 390, 400, 40, 32, 300, 20, 1)],
                         ids=lambda s: "-".join(map(str, s)))
def test_windows_of_most_keys(cuda, dtype, shape):
    """Blocks in pairs, an odd one among them, of one and of two key groups."""
    N, L, S, H, E, left, right, sinks = shape
    check(*inputs(N, L, S, H, E, dtype, seed=L), left, right, sinks, False)


def test_windows_of_most_keys_redo_rows(cuda):
    for N, L, H, E, left in ((1, 1100, 60, 128, 800), (8, 260, 50, 64, 220)):
        q, k, v = inputs(N, L, L, H, E, BF16, seed=L)
        v[0, left // 2, 1, 3] = float("inf")
        k[0, L - 9, 0, 2] = float("nan")
        check(q, k, v, left, 0, 4, True)


@pytest.mark.parametrize("dtype", DTYPES, ids=NAME.get)
@pytest.mark.parametrize("shape", [(9, 1, 700, 32, 128, 500), (9, 16, 700, 32, 64, 500), (9, 17, 300, 32, 64, 260),
                                   (9, 32, 300, 32, 128, 30), (17, 33, 90, 32, 32, 20)],
                         ids=lambda s: "-".join(map(str, s)))
def test_few_rows_of_many_sequences(cuda, dtype, shape):
    N, L, S, H, E, left = shape
    check(*inputs(N, L, S, H, E, dtype, seed=L), left, 0, 4, True)
