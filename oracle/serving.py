"""A sliding window with sinks, the 8-bit cache and copies of pages, in float64 numpy.

TEST INFRASTRUCTURE (see oracle/__init__.py).  These ops have no counterpart in the
reference; the definitions are those of ``include/cpu_attention_hip.h``, and
``tests/test_serving_oracle.py`` pins them (e4m3 against torch's conversion, the store's
rule against its statements, the window against a loop over single pairs).
"""

import numpy as np


def sees(pos, keys, left, right, sinks):
    """Which of ``keys`` keys the rows at positions ``pos`` see: bool [rows, keys]."""
    p, j = np.asarray(pos)[:, None], np.arange(keys)[None]
    ok = np.ones((len(pos), keys), bool)
    if right >= 0:
        ok &= j <= p + right
    if left >= 0:
        ok &= (j >= p - left) | (j < sinks)
    return ok


class Rows:
    """Attention rows in float64, and what bounds a kernel's error on them: ``out`` [..., E],
    ``size`` [..., E] (sum of p |v|), ``logit`` (the largest sum of |q k| scale of the
    visible pairs, in natural units) and ``keys``."""

    def __init__(self, out, size, logit, keys):
        self.out, self.size, self.logit, self.keys = out, size, logit, keys

    def bound(self, dtype, rounds_p):
        """How far a kernel's fp32 arithmetic may be off: the output's own rounding (half a
        step: bf16 2^-8, fp32 2^-24), P's to bf16 where the kernel rounds it (2^-8 of each
        term), and fp32's: each logit a sum of E products (at most E + 8 roundings of
        2^-24 of the sum of magnitudes, which moves p by as much relatively, in numerator and
        denominator), and sums over the keys (each addition 2^-24 of what it holds, twice),
        exponentials and scales (2^-18)."""
        own = 2.0 ** -8 if dtype == "bf16" else 2.0 ** -24
        e = self.out.shape[-1]
        terms = 2 * (e + 8) * 2.0 ** -24 * self.logit + (self.keys + 64) * 2.0 ** -23 + 2.0 ** -18
        if rounds_p:
            terms += 2.0 ** -8
        return own * np.abs(self.out) + (1 + own) * terms * self.size + 1e-30


def rows_of(q, k, v, scale, seen):
    """One (batch, head): q [L, E], k/v [S, E], seen [L, S]; a row without keys is 0.  Only
    visible values are used."""
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.where(seen, (q @ k.T) * scale, -np.inf)
        mag = np.where(seen, (np.abs(q) @ np.abs(k).T) * scale, 0.0)
        m = w.max(-1, keepdims=True, initial=-np.inf)
        e = np.where(seen, np.exp(w - np.where(np.isneginf(m), 0.0, m)), 0.0)
        p = e / np.maximum(e.sum(-1, keepdims=True), 1e-300)
    # 0 * inf and 0 * nan do not occur: unseen values are replaced, row by row if need be
    if np.isfinite(v).all():
        return p @ v, p @ np.abs(v), mag
    out = np.stack([pr[s] @ v[s] for pr, s in zip(p, seen)])
    return out, np.stack([pr[s] @ np.abs(v[s]) for pr, s in zip(p, seen)]), mag


def window(q, k, v, scale, left, right, sinks, causal):
    """flash_attn_window_func: q [b, L, h, E], k/v [b, S, h, E] -> Rows."""
    if causal:
        right = 0
    b, L, h, _ = q.shape
    S = k.shape[1]
    seen = sees(np.arange(L) + S - L, S, left, right, sinks)
    out, size, logit = np.zeros(q.shape), np.zeros(q.shape), 0.0
    for i in range(b):
        for j in range(h):
            out[i, :, j], size[i, :, j], mag = rows_of(q[i, :, j], k[i, :, j], v[i, :, j], scale, seen)
            logit = max(logit, float(np.nan_to_num(mag, nan=0.0, posinf=0.0).max(initial=0.0)))
    return Rows(out, size, logit, int(seen.sum(1).max(initial=0)))


def decode(q, ks, vs, scale, left, sinks):
    """One query per sequence: q [n, h, E], ks/vs lists of [len, h, E] -> Rows."""
    out, size, logit, most = np.zeros(q.shape), np.zeros(q.shape), 0.0, 0
    for i, (k, v) in enumerate(zip(ks, vs)):
        n = len(k)
        seen = sees([n - 1], n, left, -1, sinks)
        most = max(most, int(seen.sum()))
        for j in range(q.shape[1]):
            o, s, mag = rows_of(q[i, j][None], k[:, j], v[:, j], scale, seen)
            out[i, j], size[i, j] = o[0], s[0]
            logit = max(logit, float(np.nan_to_num(mag, nan=0.0, posinf=0.0).max(initial=0.0)))
    return Rows(out, size, logit, most)


# ---------------------------------------------------------------------------
# e4m3
# ---------------------------------------------------------------------------
def e4m3_values():
    """The 256 codes' values: sign, 4 exponent bits (bias 7), 3 mantissa bits; no
    infinities, 0x7f and 0xff NaN."""
    c = np.arange(256)
    e, m = (c >> 3) & 15, c & 7
    v = np.where(e > 0, (1 + m / 8.0) * 2.0 ** (e - 7), m / 8.0 * 2.0 ** -6)
    v = np.where((e == 15) & (m == 7), np.nan, v)
    return np.where(c >= 128, -v, v)


_VALUES = e4m3_values()
_POSITIVE = _VALUES[:127]  # 0 .. 448, rising


def e4m3_codes(x):
    """Codes of ``x`` (float64, magnitudes up to 448), to nearest, ties to the even code;
    not finite: NaN (0x7f)."""
    x = np.asarray(x, np.float64)
    size = np.where(np.isfinite(x), np.abs(x), 0.0)
    hi = np.clip(np.searchsorted(_POSITIVE, size), 0, 126)
    lo = np.maximum(hi - 1, 0)
    below, above = size - _POSITIVE[lo], _POSITIVE[hi] - size
    code = np.where((above < below) | ((above == below) & (hi % 2 == 0)) | (above == 0), hi, lo)
    code = code + np.where(np.signbit(x), 128, 0)
    return np.where(np.isfinite(x), code, 0x7f).astype(np.uint8)


def e4m3_decode(codes):
    return _VALUES[np.asarray(codes, np.uint8)]


def scale_for(top):
    """The smallest 2^k, k >= -100, with top <= 448 * 2^k."""
    k = -100
    while 448.0 * 2.0 ** k < top:
        k += 1
    return 2.0 ** k


class Cache8:
    """An 8-bit cache by its rule: codes [blocks, heads, page, E] of K and V (K not
    transposed here) and scales [blocks, heads]."""

    def __init__(self, k, v, k_scale, v_scale):
        self.codes, self.scales = [k, v], [k_scale, v_scale]

    def store(self, key, value, slots):
        blocks, heads, page, _ = self.codes[0].shape
        last = {}
        for i, s in enumerate(slots):
            if 0 <= s < blocks * page:
                last[int(s)] = i
        pages = sorted({s // page for s in last})
        for b in pages:
            mine = {s % page: i for s, i in last.items() if s // page == b}
            at, tok = np.array(list(mine)), np.array(list(mine.values()))
            for x, codes, scales in zip((key, value), self.codes, self.scales):
                rows = np.asarray(x, np.float64)[tok]  # [tokens, heads, E]
                for h in range(heads):
                    r = rows[:, h]
                    need = scale_for(np.abs(r[np.isfinite(r)]).max(initial=0.0))
                    if 0 in mine:
                        new = need
                    else:
                        old = max(float(scales[b, h]), 2.0 ** -100)
                        new = max(old, need)
                        if new > old:
                            codes[b, h] = e4m3_codes(e4m3_decode(codes[b, h]) * (old / new))
                    scales[b, h] = new
                    codes[b, h, at] = e4m3_codes(r / new)

    def values(self, which):
        return e4m3_decode(self.codes[which]) * np.asarray(self.scales[which], np.float64)[..., None, None]


def k_words(codes):
    """K codes [blocks, heads, page, E] in the cache's layout: 32-bit words of 4 dims, word
    by word, each for the page's positions in turn."""
    b, h, p, e = codes.shape
    return np.ascontiguousarray(codes.reshape(b, h, p, e // 4, 4).transpose(0, 1, 3, 2, 4)).reshape(b, h, p, e)


def k_rows(words):
    """The inverse of ``k_words``."""
    b, h, p, e = words.shape
    return np.ascontiguousarray(words.reshape(b, h, e // 4, p, 4).transpose(0, 1, 3, 2, 4)).reshape(b, h, p, e)


def copy_pages(array, pairs):
    """Pages copied as if at once; pairs with a negative page are padding."""
    out = array.copy()
    for s, d in pairs:
        if s >= 0 and d >= 0:
            out[d] = array[s]
    return out
