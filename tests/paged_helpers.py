"""Shared by the paged-cache tests: pools filled through plain indexing, the float64 definition of the
attention and of the prologue, and the tolerance of an f32-accurate result."""
import math

import numpy as np
import torch

from bitgpu_amd import engine as E

DEV = "cuda"


def slot_order(page):
    """(tile, panel, index) of every slot of a page in the transposed V tiles."""
    s = np.arange(page)
    j = s % 32
    return s // 32, 2 * (j // 16) + (j % 8) // 4, 4 * ((j % 16) // 8) + j % 4


class Pool:
    """A one-layer cache with known contents; unwritten slots and unlisted pages hold NaN (f32, f16) or
    codes under NaN scales (q8)."""

    def __init__(self, KV, D, kv, page, n_pages, layers=1, seed=0, q8_block=32):
        self.cache = E.PagedKvCache(layers, KV, D, kv, n_pages=n_pages, page_size=page, q8_block=q8_block)
        self.KV, self.D, self.kv, self.page = KV, D, kv, page
        c = self.cache
        if kv == "q8":
            c.k.fill_(77)
            c.v.fill_(-77)
            c.k_scale.fill_(math.nan)
            c.v_scale.fill_(math.nan)
        else:
            c.k.fill_(math.nan)
            c.v.fill_(math.nan)
        self.gen = torch.Generator().manual_seed(seed)

    def fill(self, table, n, layer=0, k_amp=1.0, v_amp=1.0):
        """Random contents for positions [0, n) of a page list (shared pages are filled once more)."""
        c, KV, D, P = self.cache, self.KV, self.D, self.page
        tile, panel, index = slot_order(P)
        for i in range(-(-n // P)):
            m = min(P, n - i * P)
            at = [torch.from_numpy(x[:m]).to(DEV) for x in (np.arange(P), tile, panel, index)]
            id_ = table[i]
            if self.kv == "q8":
                k = torch.randint(-127, 128, (m, KV, D), generator=self.gen).to(torch.int8)
                v = torch.randint(-127, 128, (m, KV, D), generator=self.gen).to(torch.int8)
                ks = torch.rand(m, KV, D // 32, generator=self.gen) * k_amp + 0.2 * k_amp
                vs = torch.rand(m, KV, D // 32, generator=self.gen) * v_amp + 0.2 * v_amp
                c.k_scale[layer, id_, :, at[0]] = ks.to(DEV).transpose(0, 1)
                c.v_scale[layer, id_, :, at[0]] = vs.to(DEV).transpose(0, 1)
            else:
                k = torch.randn(m, KV, D, generator=self.gen) * k_amp
                v = torch.randn(m, KV, D, generator=self.gen) * v_amp
            c.k[layer, id_, :, at[0]] = k.to(DEV, c.k.dtype).transpose(0, 1)
            c.v[layer, id_][:, at[1], at[2], :, at[3]] = v.to(DEV, c.v.dtype)

    def values(self, table, n, layer=0):
        """The stored K and V of positions [0, n) as float64 [n, KV, D] on the host."""
        c, D, P = self.cache, self.D, self.page
        at = torch.tensor(table[:-(-n // P)], device=DEV)
        tile, panel, index = (torch.from_numpy(x).to(DEV) for x in slot_order(P))
        k = c.k[layer][at].transpose(1, 2).reshape(-1, self.KV, D)[:n].cpu().double()
        v = c.v[layer][at][:, :, tile, panel, :, index].transpose(0, 1).reshape(-1, self.KV, D)[:n].cpu().double()
        if self.kv == "q8":
            ks, vs = (s[layer][at].transpose(1, 2).reshape(-1, self.KV, D // 32)[:n].cpu().double().repeat_interleave(32, -1)
                      for s in (c.k_scale, c.v_scale))
            k, v = k * ks / 127, v * vs / 127
        return k, v


def attention64(q, kvs, rows, lens, scale=None, gate=None):
    """The definition in float64: q [T, H, D]; kvs: one (k, v) [lens, KV, D] a sequence. Returns the result
    and, for each row, the largest |score| sum (for the tolerance) times the largest |v|."""
    T, H, D = q.shape
    scale = 1 / math.sqrt(D) if scale is None else scale
    out, tol, t = torch.zeros(T, H, D, dtype=torch.float64), torch.zeros(T, H, 1, dtype=torch.float64), 0
    for (k, v), r, n in zip(kvs, rows, lens):
        G = H // k.shape[1] if r else 1
        for i in range(r):
            m = n - r + i + 1
            kk, vv = k[:m].repeat_interleave(G, 1), v[:m].repeat_interleave(G, 1)   # [m, H, D]
            x = torch.einsum("hd,mhd->hm", q[t].double(), kk) * scale
            p = torch.softmax(x, -1)
            out[t] = torch.einsum("hm,mhd->hd", p, vv)
            size = torch.einsum("hd,mhd->hm", q[t].double().abs(), kk.abs()).amax(-1) * scale
            tol[t] = tolerance(size, D, m)[:, None] * vv.abs().amax(0).amax(-1, keepdim=True)
            t += 1
    if gate is not None:
        out = out / (1 + torch.exp(-gate.double()))
    return out, tol


def tolerance(size, D, m):
    """Error of an f32-accurate attention relative to the largest |v|. A score is a sum of D products (two
    parts each, 2^-22 of the value) accumulated in f32: its error grows as sqrt(D) 2^-24 of the sum of
    their sizes; as an exponent it moves p by that much relatively, twice (numerator and sum). The sums
    over m positions add sqrt(m) 2^-24, the parts of p 2^-21. Factor 4: the largest of many outputs."""
    return 4 * (2 * size * math.sqrt(D) * 2.0 ** -24 + math.sqrt(m) * 2.0 ** -24 + 2.0 ** -21)


def make_batch(rng, B, page, rows_of, prefix, max_tail, forks=()):
    """rows, lens, tables: B sequences behind `prefix` shared pages; (a, b, n) in forks makes b share n
    pages with a."""
    ids = list(range(4 * B * (prefix + max_tail // page + 2)))
    rng.shuffle(ids)
    at = iter(ids)
    pre = [next(at) for _ in range(prefix)]
    rows, lens, tables = [], [], []
    for b in range(B):
        r = rows_of(b)
        n = prefix * page + rng.randint(r, max(r, max_tail))
        tables.append(pre + [next(at) for _ in range(-(-n // page) - prefix)])
        rows.append(r)
        lens.append(n)
    for a, b, n in forks:
        n = min(n, (lens[a] - rows[a]) // page, (lens[b] - rows[b]) // page)
        tables[b][:n] = tables[a][:n]
    return rows, lens, tables, len(ids)


def set_batch(cache, H, rows, lens, tables, positions=None):
    b = E.PagedBatch(cache, H, max_seqs=max(1, len(rows)), max_tokens=max(1, sum(rows)), max_pages=max(1, sum(map(len, tables))))
    b.set(rows, lens, tables, positions=positions)
    return b
