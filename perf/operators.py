"""The operators of a long-running server's cache, as cases that can be timed and checked.

- ``window``: ``flash_attn_window_func``, a prompt whose tokens see the last tokens
  before them (a sliding window) and the first few of the sequence (sinks);
- ``step``: ``flash_attn_window_with_kvcache``, one new token per sequence over the
  paged cache, with a window and sinks;
- ``quant``: ``reshape_and_cache_fp8``, tokens written as 8-bit codes with one scale
  per page and head;
- ``step8``: ``flash_attn_with_kvcache_fp8``, one new token per sequence over that cache;
- ``copy``: ``copy_blocks``, pages copied within the caches of several layers (a forked
  sequence's last page, a compacted cache).

With ``own`` false ``run`` computes them from elementary torch operations.
"""

import math
import os
import random
import sys

import torch

own = False

_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "cpu-attention_amd")
if _PKG not in sys.path:
    sys.path.insert(0, _PKG)

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
ESIZE = {"bf16": 2, "fp32": 4}
F8 = torch.float8_e4m3fn
F8_MAX = 448.0
MIN_EXP = -100  # the smallest scale is 2^-100


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def window_case(dtype, batch, rows, keys, heads, dim, left, right, sinks, causal, **name):
    return dict(name, op="window", dtype=dtype, batch=batch, rows=rows, keys=keys, heads=heads, dim=dim, left=left,
                right=right, sinks=sinks, causal=causal)


def step_case(op, dtype, batch, heads, dim, page, shortest, longest, left, sinks, new, checks, lens_seed=0, **name):
    """Lengths spread from ``shortest`` to ``longest`` (both among them); ``left`` -1: no
    window; ``new`` tokens appended per sequence (0 or 1); ``checks``: the lengths are
    checked on the host."""
    return dict(name, op=op, dtype=dtype, batch=batch, heads=heads, dim=dim, page=page, shortest=shortest,
                longest=longest, left=left, sinks=sinks, new=new, checks=checks, lens_seed=lens_seed)


def quant_case(dtype, batch, heads, dim, page, shortest, longest, step, lens_seed=0, **name):
    """``step`` false: whole prompts, one token in ten a padding slot; true: the token
    after each sequence's cached ones."""
    return dict(name, op="quant", dtype=dtype, batch=batch, heads=heads, dim=dim, page=page, shortest=shortest,
                longest=longest, step=step, lens_seed=lens_seed)


def copy_case(dtype, layers, blocks, pairs, heads, dim, page, **name):
    return dict(name, op="copy", dtype=dtype, layers=layers, blocks=blocks, pairs=pairs, heads=heads, dim=dim, page=page)


def listed():
    return [
        # A short chat prompt with a window shorter than it: launch and latency.
        window_case("bf16", 1, 128, 128, 16, 64, 63, 0, 4, True, name="window_short"),
        # A batch of prompts twice as long as the window.
        window_case("bf16", 4, 2048, 2048, 32, 128, 1023, 0, 4, True, name="window_prompts"),
        # A long prompt: the largest.
        window_case("bf16", 1, 8192, 8192, 32, 128, 2047, 0, 16, True, name="window_long"),
        # The next piece of a prompt in 32-bit floats, odd sizes.
        window_case("fp32", 1, 333, 2500, 12, 64, 511, 0, 5, True, name="window_piece_fp32"),
        # One user's chat far past the window.
        step_case("step", "bf16", 1, 32, 128, 16, 8191, 8191, 1023, 4, 1, False, name="step_one"),
        # A full batch of mixed lengths, most of them longer than the window.
        step_case("step", "bf16", 64, 32, 128, 32, 17, 8000, 2047, 4, 1, False, name="step_batch"),
        # The new tokens of a small batch, stored at their slots.
        quant_case("bf16", 8, 16, 64, 16, 17, 2047, True, name="quant_step"),
        # The prompts of a large batch.
        quant_case("bf16", 128, 32, 128, 16, 64, 1024, False, name="quant_prompts"),
        # One user's chat over the 8-bit cache, called with the defaults.
        step_case("step8", "bf16", 1, 32, 128, 16, 4095, 4095, -1, 0, 1, True, name="step8_one"),
        # A full batch of mixed lengths over the 8-bit cache.
        step_case("step8", "bf16", 64, 32, 128, 32, 17, 4095, -1, 0, 0, False, name="step8_batch"),
        # Forked sequences: their last, partial pages in the 8-bit caches of a few layers.
        copy_case("fp8", 4, 512, 8, 16, 64, 16, name="copy_forks"),
        # A cache compacted after many sequences have ended.
        copy_case("bf16", 2, 6000, 2048, 32, 128, 16, name="copy_compact"),
    ]


def _log(rng, lo, hi):
    """A whole number from lo to hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


MOST_FLOPS = {"bf16": 2.0e11, "fp32": 3e10}  # of a drawn prefill
MOST_PAIRS = 2 ** 31                         # its (row, key) pairs over all heads
MOST_BYTES = 1.0e9                           # of any drawn case
MOST_CACHE = 4.0e9                           # of its cache


def draw(rng):
    while True:
        case = _draw(rng)
        w = work(case)
        if w["bytes"] > MOST_BYTES:
            continue
        if case["op"] == "window":
            pairs = case["batch"] * case["heads"] * case["rows"] * case["keys"]
            if w["flops"] > MOST_FLOPS[case["dtype"]] or pairs > MOST_PAIRS:
                continue
        elif case["op"] != "copy":
            if sum(lens_of(case)) * case["heads"] * case["dim"] * 4 > MOST_CACHE:
                continue
        return case


def _draw(rng):
    dtype = rng.choice(("bf16", "bf16", "bf16", "fp32"))
    heads, dim = rng.choice((8, 12, 16, 20, 32)), rng.choice((32, 64, 64, 128, 128))
    page = rng.choice((16, 32, 64))
    kind = rng.choice(("window", "window", "window", "step", "step", "quant", "step8", "step8", "copy"))
    if kind == "window":
        keys = _log(rng, 16, 8192)
        rows = keys if rng.random() < 0.7 else max(1, min(keys, _log(rng, 1, 2048)))
        causal = rng.random() < 0.8
        right = 0 if causal else _log(rng, 1, 512)
        return window_case(dtype, _log(rng, 1, 8), rows, keys, heads, dim, _log(rng, 16, max(17, keys)), right,
                           rng.choice((0, 1, 4, 5, 16, 64)), causal)
    if kind in ("step", "step8"):
        longest = _log(rng, 64, 16384)
        left = -1 if kind == "step8" and rng.random() < 0.6 else _log(rng, 16, 4096)
        return step_case(kind, dtype, _log(rng, 1, 128), heads, dim, page, _log(rng, 1, longest), longest, left,
                         rng.choice((0, 1, 4, 16)) if left >= 0 else 0, rng.choice((0, 1)), rng.random() < 0.3,
                         lens_seed=rng.randrange(1000))
    if kind == "quant":
        longest = _log(rng, 16, 4096)
        return quant_case(dtype, _log(rng, 1, 128), heads, dim, page, _log(rng, 1, longest), longest,
                          rng.random() < 0.4, lens_seed=rng.randrange(1000))
    blocks = _log(rng, 64, 4096)
    return copy_case(rng.choice(("bf16", "fp32", "fp8")), rng.randint(1, 4), blocks, _log(rng, 1, blocks // 2), heads,
                     dim, page)


def lens_of(case):
    """Cached tokens before an append; tokens of a prompt."""
    r = random.Random(case["lens_seed"])
    lens = [r.randint(case["shortest"], case["longest"]) for _ in range(case["batch"])]
    lens[-1] = case["shortest"]
    lens[0] = case["longest"]
    return lens


def span_of(case, n):
    """(lo, s): the newest of ``n`` tokens sees keys [0, s) and [lo, n)."""
    lo = max(0, n - 1 - case["left"]) if case["left"] >= 0 else 0
    return lo, min(case["sinks"], lo)


def visible(case):
    """Visible (row, key) pairs of one (batch, head) of a prefill."""
    rows, keys, total = case["rows"], case["keys"], 0
    for i in range(rows):
        p = i + keys - rows
        end = max(0, min(keys, p + 1 + case["right"]))
        lo = min(max(0, p - case["left"]), end)
        total += end - lo + min(case["sinks"], lo)
    return total


def work(case):
    heads, dim = case["heads"], case["dim"]
    if case["op"] == "copy":
        page = heads * case["page"] * dim * {"bf16": 2, "fp32": 4, "fp8": 1}[case["dtype"]]
        scales = 4 * heads if case["dtype"] == "fp8" else 0
        return {"bytes": case["layers"] * case["pairs"] * 4 * (page + scales) + 16 * case["pairs"], "flops": 0}
    es, batch = ESIZE[case["dtype"]], case["batch"]
    row = heads * dim * es
    if case["op"] == "window":
        rows, keys = case["rows"], case["keys"]
        used = min(keys, case["sinks"] + rows + case["left"] + case["right"])  # keys that a row sees
        return {"bytes": batch * row * 2 * (rows + used), "flops": 4 * dim * heads * batch * visible(case)}
    lens = lens_of(case)
    if case["op"] == "quant":
        tokens = batch if case["step"] else sum(n - n // 10 for n in lens)
        pages = batch if case["step"] else sum(-(-n // case["page"]) for n in lens)
        return {"bytes": tokens * (2 * row + 2 * heads * dim + 8) + pages * heads * 8, "flops": 0}
    kv = heads * dim * (es if case["op"] == "step" else 1)
    seen = 0
    for n in lens:
        lo, s = span_of(case, n + case["new"])
        seen += n + case["new"] - lo + s
    return {"bytes": 2 * seen * kv + 2 * batch * row + 2 * batch * case["new"] * (row + kv) + 4 * seen // case["page"]
            + (0 if case["op"] == "step" else 8 * heads * seen // case["page"]),
            "flops": 4 * heads * dim * seen}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _tokens(g, dtype, n, heads, dim):
    """Keys or values of ``n`` tokens: tokens differ in size, as a model's do."""
    return (_randn(g, n, heads, dim) * torch.exp(0.5 * _randn(g, n, heads, 1))).to(DTYPES[dtype])


def _cache(g, dtype, blocks, heads, page, dim):
    if dtype != "fp8":
        return torch.randn(blocks, heads, page, dim, generator=g, device="cuda", dtype=DTYPES[dtype])
    codes = torch.randn(blocks, heads, page, dim, generator=g, device="cuda", dtype=torch.float16) * 90
    return codes.clamp_(-F8_MAX, F8_MAX).to(F8)


def _power(k):
    """2^k of whole numbers, exactly (a power function may be an ulp off): the bits of a float."""
    return (k.int() + 127 << 23).view(torch.float32)


def _scales(g, blocks, heads):
    return _power(torch.randint(-8, -4, (blocks, heads), generator=g, device="cuda"))


def _paging(case, seed, lens):
    """A page table over blocks in random order, and the number of blocks."""
    need = [-(-n // case["page"]) for n in lens]
    order = list(range(sum(need)))
    random.Random(seed).shuffle(order)
    width = max(need)
    table = torch.zeros(len(lens), width, dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = torch.tensor(order[at:at + n], dtype=torch.int32)
        at += n
    return table, at


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    heads, dim = case["heads"], case["dim"]
    state = dict(case)
    if case["op"] == "window":
        dtype = DTYPES[case["dtype"]]
        state["q"], state["k"], state["v"] = (
            torch.randn(case["batch"], n, heads, dim, generator=g, device="cuda", dtype=dtype)
            for n in (case["rows"], case["keys"], case["keys"]))
        return state
    if case["op"] == "copy":
        args = (g, case["dtype"], case["blocks"], heads, case["page"], dim)
        state["kc"] = [_cache(*args) for _ in range(case["layers"])]
        state["vc"] = [_cache(*args) for _ in range(case["layers"])]
        state["ks"] = state["vs"] = None
        if case["dtype"] == "fp8":
            state["ks"] = [_scales(g, case["blocks"], heads) for _ in range(case["layers"])]
            state["vs"] = [_scales(g, case["blocks"], heads) for _ in range(case["layers"])]
        order = torch.randperm(case["blocks"], generator=g, device="cuda")[:2 * case["pairs"]]
        state["mapping"] = order.view(2, -1).t().contiguous()
        return state
    lens = lens_of(case)
    grow = 1 if case["op"] != "quant" or case["step"] else 0
    table, blocks = _paging(case, seed, [n + grow for n in lens])
    state["table"], state["lens"] = table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda()
    cache = "fp8" if case["op"] in ("quant", "step8") else case["dtype"]
    state["kc"], state["vc"] = (_cache(g, cache, blocks, heads, case["page"], dim) for _ in range(2))
    if cache == "fp8":
        state["ks"], state["vs"] = _scales(g, blocks, heads), _scales(g, blocks, heads)
    if case["op"] == "quant":
        page = case["page"]
        if case["step"]:
            pos = torch.tensor(lens)
            slots = table.gather(1, (pos // page)[:, None].long())[:, 0].long() * page + pos % page
        else:
            slots = torch.cat([(table[i, :-(-n // page)].long()[:, None] * page + torch.arange(page)).flatten()[:n]
                               for i, n in enumerate(lens)])
            slots[9::10] = -1  # padding
        state["slots"] = slots.cuda()
        state["k"], state["v"] = (_tokens(g, case["dtype"], slots.numel(), heads, dim) for _ in range(2))
        return state
    state["q"] = _randn(g, case["batch"], 1, heads, dim).to(DTYPES[case["dtype"]])
    if case["new"]:
        state["k"], state["v"] = (_tokens(g, case["dtype"], case["batch"], heads, dim)[:, None] for _ in range(2))
    return state


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------
def _plain_window(s):
    """Every logit of every row, masked, in 32 bits."""
    q, k, v = (s[x].float().transpose(1, 2).contiguous() for x in "qkv")
    p = torch.arange(s["rows"], device=q.device)[:, None] + (s["keys"] - s["rows"])
    j = torch.arange(s["keys"], device=q.device)
    seen = ((j >= p - s["left"]) | (j < s["sinks"])) & (j <= p + s["right"])
    logits = torch.matmul(q, k.transpose(2, 3).contiguous()).mul_(s["dim"] ** -0.5)
    logits.masked_fill_(~seen, -math.inf)
    top = logits.amax(-1, keepdim=True)
    weight = logits.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = weight.sum(-1, keepdim=True)
    out = torch.matmul(weight, v) / torch.where(total == 0, 1.0, total)
    return out.transpose(1, 2).contiguous().to(s["q"].dtype)


def _words(cache, page):
    """The K cache's elements as [block, head, word, position, element of the word]: a
    page holds 32-bit words of neighbouring dims, word by word."""
    blocks, heads, _, dim = cache.shape
    per = 4 // cache.element_size()
    return cache.view(blocks, heads, dim // per, page, per)


def _bytes(x):
    return x.view(torch.uint8) if x.dtype == F8 else x


def _typed(x, dtype):
    return x.contiguous().view(dtype) if dtype == F8 else x


def _plain_step(s):
    """One query per sequence over the gathered keys that it sees, in 32 bits."""
    lens, page, dim = s["lens"].long() + s["new"], s["page"], s["dim"]
    most = s["longest"] + s["new"]
    lo = torch.zeros_like(lens)
    if s["left"] >= 0:
        lo = (lens - 1 - s["left"]).clamp(min=0)
        most = min(most, s["sinks"] + s["left"] + 1)
    first = lo.clamp(max=s["sinks"])
    j = torch.arange(most, device=lens.device)
    pos = torch.where(j < first[:, None], j, (lo - first)[:, None] + j)
    seen = pos < lens[:, None]
    pos = torch.where(seen, pos, 0)
    block, at = s["table"].long().gather(1, pos // page), pos % page
    k = _words(_bytes(s["kc"]), page).permute(0, 3, 1, 2, 4)[block, at]
    k = _typed(k.flatten(3), s["kc"].dtype).float()
    v = _typed(_bytes(s["vc"]).transpose(1, 2)[block, at], s["vc"].dtype).float()
    if s["op"] == "step8":
        k.mul_(s["ks"][block][..., None])
        v.mul_(s["vs"][block][..., None])
    logits = k.mul_(s["q"].float()).sum(-1) * dim ** -0.5
    logits.masked_fill_(~seen[..., None], -math.inf)
    weight = (logits - logits.amax(1, keepdim=True)).exp()
    out = v.mul_(weight[..., None]).sum(1) / weight.sum(1)[..., None]
    return out[:, None].to(s["q"].dtype)


def _slots(s):
    """The slots of the tokens after each sequence's cached ones."""
    lens, page = s["lens"].long(), s["page"]
    return s["table"].long().gather(1, (lens // page)[:, None])[:, 0] * page + lens % page


def _plain_store(s, slots):
    """The new tokens' elements into the 16- or 32-bit cache."""
    block, at = slots // s["page"], slots % s["page"]
    words = _words(s["kc"], s["page"])
    words[block, :, :, at] = s["k"][:, 0].view(s["batch"], s["heads"], -1, words.shape[-1])
    s["vc"][block, :, at] = s["v"][:, 0]


def _scale_for(top):
    """The smallest power of two, 2^-100 or more, that takes values up to ``top`` to 448."""
    part, power = torch.frexp(top)
    power = power.int() - torch.where(part <= 0.875, 9, 8)
    return _power(power.clamp(min=MIN_EXP))


def _plain_quant(s, key, value, slots):
    """Tokens into the 8-bit cache: each page's scale, its earlier codes at a scale that
    grew, then the tokens' codes."""
    blocks, heads, page = s["kc"].shape[0], s["heads"], s["page"]
    stored = slots >= 0
    block = torch.where(stored, slots // page, blocks)  # padding goes to a page past the last
    touched = torch.unique(block)
    touched = touched[touched < blocks]
    starts = torch.zeros(blocks + 1, dtype=torch.int32, device=slots.device)
    starts.scatter_reduce_(0, block, (slots % page == 0).int(), "amax")
    for x, cache, scales in ((key, s["kc"], s["ks"]), (value, s["vc"], s["vs"])):
        x = x.float()
        top = torch.where(x.isfinite(), x, 0.0).abs().amax(-1)
        most = torch.zeros(blocks + 1, heads, device=x.device)
        most.scatter_reduce_(0, block[:, None].expand(-1, heads), top, "amax")
        need = _scale_for(most[touched])
        old = scales[touched].clamp(min=2.0 ** MIN_EXP)
        anew = (starts[touched] > 0)[:, None]
        new = torch.where(anew, need, torch.maximum(old, need))
        ratio = torch.where(anew, 1.0, old / new)
        raw = cache.view(torch.uint8)
        codes = raw[touched].view(F8).float() * ratio[..., None, None]
        raw[touched] = codes.to(F8).view(torch.uint8)
        scales[touched] = new
        x, at, to = x[stored], slots[stored] % page, block[stored]
        codes = (x / scales[to][..., None]).to(F8).view(torch.uint8)
        if cache is s["kc"]:
            _words(raw, page)[to, :, :, at] = codes.view(*codes.shape[:2], -1, 4)
        else:
            raw[to, :, at] = codes


def _plain_copy(s):
    src, dst = s["mapping"][:, 0], s["mapping"][:, 1]
    for x in s["kc"] + s["vc"] + (s["ks"] or []) + (s["vs"] or []):
        x = _bytes(x)
        x[dst] = x[src]


def run(state):
    s = state
    op = s["op"]
    if own:
        return _own(s)
    if op == "window":
        return _plain_window(s)
    if op == "quant":
        _plain_quant(s, s["k"], s["v"], s["slots"])
        return [s["kc"], s["vc"], s["ks"], s["vs"]]
    if op == "copy":
        _plain_copy(s)
        return [s["kc"], s["vc"], s["ks"], s["vs"]]
    if s["new"] and op == "step":
        _plain_store(s, _slots(s))
    elif s["new"]:
        _plain_quant(s, s["k"][:, 0], s["v"][:, 0], _slots(s))
    return _after_step(s, _plain_step(s))


def _after_step(s, out):
    if not s["new"]:
        return [out]
    return [out, s["kc"], s["vc"]] + ([s["ks"], s["vs"]] if s["op"] == "step8" else [])


def _own(s):
    import cpu_attention as C
    from cpu_attention import _kernel

    if s["op"] == "window":
        return C.flash_attn_window_func(s["q"], s["k"], s["v"], window_size=(s["left"], s["right"]),
                                        sink_tokens=s["sinks"], causal=s["causal"])
    _kernel.set_host_checks(s.get("checks", False))
    if s["op"] == "quant":
        C.reshape_and_cache_fp8(s["k"], s["v"], s["kc"], s["vc"], s["ks"], s["vs"], s["slots"])
        return [s["kc"], s["vc"], s["ks"], s["vs"]]
    if s["op"] == "copy":
        C.copy_blocks(s["kc"], s["vc"], s["mapping"], key_scales=s["ks"], value_scales=s["vs"])
        return [s["kc"], s["vc"], s["ks"], s["vs"]]
    more = dict(k=s.get("k"), v=s.get("v"), cache_seqlens=s["lens"], page_table=s["table"],
                window_size=(s["left"], 0 if s["left"] >= 0 else -1), sink_tokens=s["sinks"])
    if s["op"] == "step":
        return _after_step(s, C.flash_attn_window_with_kvcache(s["q"], s["kc"], s["vc"], **more))
    return _after_step(s, C.flash_attn_with_kvcache_fp8(s["q"], s["kc"], s["vc"], s["ks"], s["vs"], **more))


# ---------------------------------------------------------------------------
# 64 bits
# ---------------------------------------------------------------------------
def _power64(k):
    return (k.long() + 1023 << 52).view(torch.float64)


def _e4m3(x):
    """``x`` (float64) rounded to e4m3's values: 3 bits after the leading one, ties to
    even, steps of 2^-9 below 2^-6; not finite: NaN."""
    size = x.abs()
    step = _power64(torch.frexp(torch.where(size.isfinite(), size, 0.0))[1].clamp(min=-5) - 4)
    return torch.where(size.isfinite(), torch.round(x / step) * step, math.nan)


def _exact_quant(s, key, value, slots):
    """The caches and scales after a store, in 64 bits, page by page as the scales' rule
    says it (in one go over the tokens sorted by page)."""
    blocks, heads, page, dim = s["kc"].shape
    keep = slots >= 0
    slots = slots[keep]
    order = torch.argsort(slots)
    slots = slots[order]
    page_of, counts = torch.unique_consecutive(slots // page, return_counts=True)
    begins = torch.cat([counts.new_zeros(1), counts.cumsum(0)[:-1]])
    anew = slots[begins] % page == 0
    result = []
    for x, cache, scales, is_k in ((key, s["kc"], s["ks"], True), (value, s["vc"], s["vs"], False)):
        x = x[keep][order].double()
        top = torch.nan_to_num(x, nan=0.0, posinf=0.0, neginf=0.0).abs().amax(-1)
        group = torch.repeat_interleave(torch.arange(len(counts), device=x.device), counts)
        most = torch.zeros(len(counts), heads, dtype=torch.float64, device=x.device)
        most.index_reduce_(0, group, top, "amax")
        need = torch.log2(torch.clamp(most / F8_MAX, min=2.0 ** MIN_EXP)).floor().int() - 1
        for _ in range(3):  # from below, up to the first that is enough
            need = need + (F8_MAX * _power64(need) < most)
        need = _power64(need.clamp(min=MIN_EXP))
        new, codes = scales.double().clone(), cache.float().double()
        old = new[page_of].clamp(min=2.0 ** MIN_EXP)
        now = torch.where(anew[:, None], need, torch.maximum(old, need))
        grew = (now > old) & ~anew[:, None]
        codes[page_of] = torch.where(grew[..., None, None], _e4m3(codes[page_of] * (old / now)[..., None, None]),
                                     codes[page_of])
        new[page_of] = now
        rows = _e4m3(x / now[group][..., None])
        b, t = slots // page, slots % page
        if is_k:
            codes.view(blocks, heads, dim // 4, page, 4)[b, :, :, t] = rows.view(len(b), heads, dim // 4, 4)
        else:
            codes[b, :, t] = rows
        result.append((codes, new))
    return [result[0][0], result[1][0], result[0][1], result[1][1]]


def _exact_step(s, caches):
    kc, vc, ks, vs = caches
    blocks, heads, page, dim = kc.shape
    per = 4 // (1 if s["op"] == "step8" else ESIZE[s["dtype"]])
    keys = kc.view(blocks, heads, dim // per, page, per)
    rows = []
    for i, n in enumerate(lens_of(s)):
        n += s["new"]
        lo, first = span_of(s, n)
        pos = torch.cat([torch.arange(first), torch.arange(lo, n)]).cuda()
        b, t = s["table"][i].long()[pos // page], pos % page
        k = keys[b, :, :, t].flatten(2).double()
        v = vc[b, :, t].double()
        if ks is not None:
            k, v = k * ks[b][..., None], v * vs[b][..., None]
        weight = torch.softmax((k * s["q"][i].double()).sum(-1) * dim ** -0.5, 0)
        rows.append((weight[..., None] * v).sum(0))
    return torch.stack(rows)[:, None]


def _exact_window(s):
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    j = torch.arange(s["keys"], device="cuda")
    at_most = max(1, int(2 ** 27 // s["keys"]))
    for b in range(s["batch"]):
        for h in range(s["heads"]):
            k, v = s["k"][b, :, h].double(), s["v"][b, :, h].double()
            for r in range(0, s["rows"], at_most):
                q = s["q"][b, r:r + at_most, h].double()
                p = torch.arange(r, r + len(q), device="cuda")[:, None] + s["keys"] - s["rows"]
                behind = p - j
                seen = (behind >= -s["right"]) & ((behind <= s["left"]) | (j[None] < s["sinks"]))
                logits = torch.where(seen, q @ k.T * s["dim"] ** -0.5, -math.inf)
                out[b, r:r + at_most, h] = torch.nan_to_num(torch.softmax(logits, -1), nan=0.0) @ v
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "window":
        return _exact_window(s)
    if s["op"] == "quant":
        return _exact_quant(s, s["k"], s["v"], s["slots"])
    if s["op"] == "copy":
        mapping = s["mapping"].tolist()
        src, dst = (torch.tensor(x, device="cuda") for x in zip(*mapping))
        lists = []
        for name in ("kc", "vc", "ks", "vs"):
            lists.append(None if s[name] is None else [])
            for x in s[name] or []:
                y = x.float().clone()
                y.index_copy_(0, dst, x.float().index_select(0, src))
                lists[-1].append(y)
        return lists
    if s["op"] == "step":
        kc, vc = s["kc"].clone(), s["vc"].clone()
        if s["new"]:
            for i, n in enumerate(lens_of(s)):
                b, t = int(s["table"][i, n // s["page"]]), n % s["page"]
                per = 4 // ESIZE[s["dtype"]]
                kc[b].view(s["heads"], s["dim"] // per, s["page"], per)[:, :, t] = s["k"][i, 0].view(s["heads"], -1, per)
                vc[b, :, t] = s["v"][i, 0]
        out = _exact_step(s, (kc, vc, None, None))
        return [out, kc, vc] if s["new"] else [out]
    caches = [s["kc"].float(), s["vc"].float(), s["ks"].double(), s["vs"].double()]
    if s["new"]:
        caches = _exact_quant(s, s["k"][:, 0], s["v"][:, 0], _slots(s))
    out = _exact_step(s, caches)
    return [out] + caches if s["new"] else [out]
