"""Shared by the tests of the window, the 8-bit cache and the page copies."""

import numpy as np
import torch

from helpers import values
from oracle import serving as R

NAME = {torch.float32: "fp32", torch.bfloat16: "bf16"}


def close(out, rows, dtype, rounds_p=False):
    """``out`` within the derived bound of the oracle's rows; NaN where and only where they
    are."""
    got = values(out).reshape(rows.out.shape)
    nan = np.isnan(rows.out)
    assert np.array_equal(np.isnan(got), nan), "NaN in other places"
    fine = np.isfinite(rows.out)
    assert np.array_equal(got[~fine & ~nan], rows.out[~fine & ~nan])
    err, tol = np.abs(got - rows.out)[fine], rows.bound(NAME[dtype], rounds_p)[fine]
    worst = int(np.argmax(err / tol)) if err.size else 0
    assert err.size == 0 or err[worst] <= tol[worst], (err[worst], tol[worst])



class Paged:
    """Sequences in a paged cache written here, token by token, in the cache's layout: pages
    in random order, everything else NaN, and the table's unused entries out of range."""

    def __init__(self, lens, heads, dim, page, dtype, seed, device, fp8=False, spare=0):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.page, self.heads, self.dim, self.dtype = list(lens), page, heads, dim, dtype
        need = [-(-(n + spare) // page) for n in lens]
        total = sum(need) + 2
        order = torch.randperm(total, generator=g)
        table = torch.full((len(lens), max(need + [1]) + 1), 1 << 30, dtype=torch.int32)
        at = 0
        for i, n in enumerate(need):
            table[i, :n] = order[at:at + n].int()
            at += n
        self.table = table.to(device)
        self.blocks = total
        self.lens_t = torch.tensor(self.lens, dtype=torch.int32, device=device)
        self.q = torch.randn(len(lens), 1, heads, dim, generator=g).to(dtype).to(device)
        ks = [torch.randn(n, heads, dim, generator=g) for n in lens]
        vs = [torch.randn(n, heads, dim, generator=g) for n in lens]
        if fp8:
            # codes and scales of every page; a page not in use holds NaN codes and a NaN scale
            kc = torch.full((total, heads, page, dim), 0x7f, dtype=torch.uint8)
            vc = kc.clone()
            kscale, vscale = (torch.full((total, heads), float("nan")) for _ in range(2))
            self.ks, self.vs = [], []
            for i, n in enumerate(lens):
                rows = []
                for x, cache, scale in ((ks[i], kc, kscale), (vs[i], vc, vscale)):
                    val = np.zeros((n, heads, dim))
                    for b in range(-(-n // page)):
                        blk = int(table[i, b])
                        for h in range(heads):
                            s = 2.0 ** int(torch.randint(-9, -5, (1,), generator=g))
                            scale[blk, h] = s
                            part = x[b * page:(b + 1) * page, h].double().numpy()
                            code = R.e4m3_codes(np.clip(part / s, -448, 448))
                            cache[blk, h, :len(part)] = torch.from_numpy(code)
                            val[b * page:(b + 1) * page, h] = R.e4m3_decode(code) * s
                    rows.append(val)
                self.ks.append(rows[0])
                self.vs.append(rows[1])
            self.rows = [kc.numpy(), vc.numpy()]
            self.kc = torch.from_numpy(R.k_words(kc.numpy())).view(torch.float8_e4m3fn).to(device)
            self.vc = vc.view(torch.float8_e4m3fn).to(device)
            self.kscale, self.vscale = kscale.to(device), vscale.to(device)
            return
        kc = torch.full((total, heads, page, dim), float("nan"), dtype=dtype)
        vc = kc.clone()
        for i, n in enumerate(lens):
            for b in range(-(-n // page)):
                blk = int(table[i, b])
                part = slice(b * page, min(n, (b + 1) * page))
                kc[blk, :, :part.stop - part.start] = ks[i][part].to(dtype).transpose(0, 1)
                vc[blk, :, :part.stop - part.start] = vs[i][part].to(dtype).transpose(0, 1)
        per = 4 // kc.element_size()
        self.kc = kc.view(total, heads, page, dim // per, per).transpose(2, 3).contiguous().view(total, heads, page, dim).to(device)
        self.vc = vc.to(device)
        self.ks = [values(x.to(dtype)) for x in ks]
        self.vs = [values(x.to(dtype)) for x in vs]

    def rows_of(self):
        """K as [blocks, heads, page, dim] rows (the layout undone) and V, on the CPU."""
        per = 4 // self.kc.element_size()
        k = self.kc.cpu().contiguous().view(torch.uint8).view(self.blocks, self.heads, self.dim // per, self.page, 4)
        k = k.transpose(2, 3).reshape(self.blocks, self.heads, self.page, -1)
        return k, self.vc.cpu().view(torch.uint8)


def capture(fn, warm=2):
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(warm):
            fn()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = fn()
    return graph, out


def same_bytes(a, b):
    return torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))
