"""The operators together, as a server runs them: prompts through the window prefill, their
keys and values into the cache, sequences forked, decoded token by token, the cache
compacted.  Every step against the float64 oracle of the whole history."""

import numpy as np
import pytest
import torch

import cpu_attention as C
from helpers import values
from oracle import serving as R
from serving_helpers import close, same_bytes

pytestmark = pytest.mark.gpu
LAYERS, HEADS, DIM, PAGE, WINDOW, SINKS = 2, 3, 64, 16, 40, 3


class Server:
    """A paged cache of a few layers with the pages' bookkeeping on the host."""

    def __init__(self, blocks, dtype, fp8, device):
        self.dtype, self.fp8, self.device, self.blocks = dtype, fp8, device, blocks
        kind = torch.float8_e4m3fn if fp8 else dtype
        self.kc, self.vc = ([torch.zeros(blocks, HEADS, PAGE, DIM, dtype=kind, device=device) for _ in range(LAYERS)]
                            for _ in range(2))
        self.ks, self.vs = ([torch.zeros(blocks, HEADS, device=device) for _ in range(LAYERS)] for _ in range(2))
        self.free = list(np.random.default_rng(0).permutation(blocks))
        self.pages, self.lens, self.history = [], [], []
        empty = [np.zeros((blocks, HEADS, PAGE, DIM), np.uint8) for _ in range(2)]
        self.ref = [R.Cache8(empty[0].copy(), empty[1].copy(), np.zeros((blocks, HEADS)), np.zeros((blocks, HEADS)))
                    for _ in range(LAYERS)]

    def grow(self, i, n):
        while len(self.pages[i]) * PAGE < n:
            self.pages[i].append(int(self.free.pop()))

    def slots(self, i, start, n):
        return [self.pages[i][t // PAGE] * PAGE + t % PAGE for t in range(start, start + n)]

    def prompt(self, lens, g):
        """Prompts of one batch: attention layer by layer, then the cache writes."""
        S = max(lens)
        for n in lens:
            self.pages.append([])
            self.grow(len(self.pages) - 1, n)
            self.lens.append(n)
            self.history.append([[] for _ in range(LAYERS)])
        slots = np.full((len(lens), S), -1)
        for i, n in enumerate(lens):
            slots[i, :n] = self.slots(i, 0, n)
        slots_t = torch.from_numpy(slots).flatten().to(self.device)
        for layer in range(LAYERS):
            qkv = torch.randn(len(lens), S, 3, HEADS, DIM, generator=g).to(self.dtype).to(self.device)
            q, k, v = qkv.unbind(2)
            out = C.flash_attn_window_func(q, k, v, window_size=(WINDOW, 0), sink_tokens=SINKS, causal=True)
            close(out, R.window(values(q), values(k), values(v), DIM ** -0.5, WINDOW, 0, SINKS, True), self.dtype,
                  rounds_p=self.dtype == torch.bfloat16)
            k, v = (x.reshape(-1, HEADS, DIM) for x in (k, v))
            if self.fp8:
                C.reshape_and_cache_fp8(k, v, self.kc[layer], self.vc[layer], self.ks[layer], self.vs[layer], slots_t)
            else:
                C.reshape_and_cache(k, v, self.kc[layer], self.vc[layer], slots_t)
            self.ref[layer].store(values(k), values(v), slots.flatten())
            for i, n in enumerate(lens):
                self.history[i][layer] = [values(x).reshape(len(lens), S, HEADS, DIM)[i, :n] for x in (k, v)]

    def fork(self, i):
        """A child of sequence i: whole pages shared, the partial one copied."""
        whole = self.lens[i] // PAGE
        self.pages.append(self.pages[i][:whole])
        self.lens.append(self.lens[i])
        self.history.append([[x.copy() for x in layer] for layer in self.history[i]])
        if self.lens[i] % PAGE:
            self.grow(len(self.pages) - 1, self.lens[i])
            self.copy([(self.pages[i][whole], self.pages[-1][whole])])

    def copy(self, pairs):
        kw = dict(key_scales=self.ks, value_scales=self.vs) if self.fp8 else {}
        C.copy_blocks(self.kc, self.vc, torch.tensor(pairs), **kw)
        for r in self.ref:
            r.codes = [R.copy_pages(x, pairs) for x in r.codes]
            r.scales = [R.copy_pages(x, pairs) for x in r.scales]

    def table(self):
        width = max(map(len, self.pages))
        return torch.tensor([p + [-1] * (width - len(p)) for p in self.pages], dtype=torch.int32, device=self.device)

    def step(self, g, n=1, append=True):
        """One token for every sequence; returns the outputs."""
        outs = []
        for i in range(len(self.pages)):
            self.grow(i, self.lens[i] + n)
        lens = torch.tensor(self.lens, dtype=torch.int32, device=self.device)
        for layer in range(LAYERS):
            q = torch.randn(len(self.lens), 1, HEADS, DIM, generator=g).to(self.dtype).to(self.device)
            kv = torch.randn(2, len(self.lens), n, HEADS, DIM, generator=g) * 2.0 ** int(torch.randint(-2, 4, (1,), generator=g))
            k, v = kv.to(self.dtype).to(self.device)
            new = dict(k=k, v=v) if append else {}
            kw = dict(cache_seqlens=lens, page_table=self.table(), window_size=(WINDOW, 0), sink_tokens=SINKS, **new)
            if self.fp8:
                out = C.flash_attn_with_kvcache_fp8(q, self.kc[layer], self.vc[layer], self.ks[layer], self.vs[layer], **kw)
            else:
                out = C.flash_attn_window_with_kvcache(q, self.kc[layer], self.vc[layer], **kw)
            if append:
                slots = [s for i in range(len(self.lens)) for s in self.slots(i, self.lens[i], n)]
                self.ref[layer].store(values(k).reshape(-1, HEADS, DIM), values(v).reshape(-1, HEADS, DIM), slots)
                for i in range(len(self.lens)):
                    self.history[i][layer] = [np.concatenate([h, values(x)[i]]) for h, x in zip(self.history[i][layer], (k, v))]
            close(out, R.decode(values(q)[:, 0], *self.seen(layer), DIM ** -0.5, WINDOW, SINKS), self.dtype)
            outs.append(out)
        if append:
            self.lens = [x + n for x in self.lens]
        return outs

    def seen(self, layer):
        """Each sequence's keys and values: the history, or what the 8-bit cache stands for."""
        if not self.fp8:
            return tuple([h[layer][w] for h in self.history] for w in (0, 1))
        n = [len(h[layer][0]) for h in self.history]
        return tuple([np.concatenate([self.ref[layer].values(w)[b].transpose(1, 0, 2) for b in self.pages[i]])[:n[i]]
                      for i in range(len(n))] for w in (0, 1))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("fp8", [False, True], ids=["cache", "fp8"])
def test_a_server(cuda, dtype, fp8):
    g = torch.Generator().manual_seed(1)
    s = Server(80, dtype, fp8, cuda)
    s.prompt([70, 5, 33, 1], g)
    s.step(g)
    s.fork(0)       # in the middle of a page
    s.step(g)
    s.step(g, n=20)
    s.fork(2)
    for _ in range(17):  # over a page's end
        s.step(g)
    if fp8:
        for layer in range(LAYERS):
            for got, want in zip((s.ks, s.vs), s.ref[layer].scales):
                used = sorted({b for p in s.pages for b in p})
                assert np.array_equal(got[layer].cpu().numpy()[used], want[used].astype(np.float32))
    # sequence 1 ends; the cache is compacted onto the first pages, and nothing changes
    state = g.get_state()
    before = s.step(g, append=False)
    ended = s.pages.pop(1)
    s.lens.pop(1)
    s.history.pop(1)
    used = sorted({b for p in s.pages for b in p})
    free = [b for b in range(s.blocks) if b not in used]
    moves = [(src, dst) for src, dst in zip(reversed(used), free) if dst < src]
    s.copy(moves)
    to = dict(moves)
    s.pages = [[to.get(b, b) for b in p] for p in s.pages]
    assert ended and max(b for p in s.pages for b in p) == len(used) - 1
    s.free = [b for b in range(s.blocks) if b not in {b for p in s.pages for b in p}]
    keep = [0, 2, 3, 4, 5]
    g.set_state(state)
    layer = 0
    q = torch.randn(6, 1, HEADS, DIM, generator=g).to(dtype).to(cuda)[keep]
    lens = torch.tensor(s.lens, dtype=torch.int32, device=cuda)
    kw = dict(cache_seqlens=lens, page_table=s.table(), window_size=(WINDOW, 0), sink_tokens=SINKS)
    if fp8:
        out = C.flash_attn_with_kvcache_fp8(q, s.kc[layer], s.vc[layer], s.ks[layer], s.vs[layer], **kw)
    else:
        out = C.flash_attn_window_with_kvcache(q, s.kc[layer], s.vc[layer], **kw)
    assert same_bytes(out, before[0][keep])
    for _ in range(3):
        s.step(g)
