"""Restatement of the paged 4-bit KV cache in numpy, one element at a time in the
format and in 64 bits in the attention; shares no code with the product.

Quantising follows the product's definition step by step in float32 (its codes
are compared byte for byte); reading, planning and attention follow theirs.
"""
from __future__ import annotations

import numpy as np

TILE = 16


def tile_bytes(dim: int, group: int) -> int:
    return 16 * dim + 128 * (dim // group)


def head_bytes(dim: int, group: int, page: int) -> int:
    return page // TILE * tile_bytes(dim, group)


def k_spot(dim: int, tok: int, d: int):
    """(byte in the tile, shift) of a K code."""
    sd = min(dim, 128)
    slab, x = divmod(d, sd)
    i, y = divmod(x, 32)
    t, z = divmod(y, 8)
    k, h = divmod(z, 2)
    nib = 4 * h + k
    return 4 * (((slab * 16 + tok) * 4 + t) * (sd // 32) + i) + nib // 2, 4 * (nib % 2)


def v_spot(dim: int, tok: int, d: int):
    sd = min(dim, 128)
    slab, x = divmod(d, sd)
    j, y = divmod(x, 32)
    k, g = divmod(y, 8)
    p, r = divmod(tok, 8)
    t, b = divmod(r, 2)
    half = ((((slab * 2 + p) * 8 + g) * 4 + t) * (sd // 32) + j) * 2 + b
    return 8 * dim + 2 * half + k // 2, 4 * (k % 2)


def quantise(x: np.ndarray, group: int):
    """float32 [..., dim] -> (codes uint8 [..., dim], float16 [..., dim/group, 2])."""
    f = np.float32
    x = x.astype(f).reshape(*x.shape[:-1], -1, group)
    nan = np.isnan(x).any(-1, keepdims=True)
    x = np.clip(np.where(np.isnan(x), f(0), x), f(-65000), f(65000))
    lo, hi = x.min(-1, keepdims=True), x.max(-1, keepdims=True)
    scale = np.where(nan, f(np.nan), (hi - lo) / f(15)).astype(np.float16)
    s = scale.astype(f)
    offset = (lo + f(8) * s).astype(np.float16)
    with np.errstate(divide="ignore", invalid="ignore"):
        step = np.where(s > 0, f(1) / s, f(0)).astype(f)
        c = np.where(s > 0, np.rint((x - offset.astype(f)) * step), 0)
    c = np.clip(c, -8, 7) + 8
    par = np.concatenate([scale, offset], -1)
    return c.astype(np.uint8).reshape(*c.shape[:-2], -1), par


class Pages:
    """The bytes of a cache, [num_pages, layers, heads, bytes]."""

    def __init__(self, data: np.ndarray, dim: int, page: int, group: int):
        self.data, self.dim, self.page, self.group = data, dim, page, group
        self.tb = tile_bytes(dim, group)
        self.ks = [[k_spot(dim, t, d) for d in range(dim)] for t in range(TILE)]
        self.vs = [[v_spot(dim, t, d) for d in range(dim)] for t in range(TILE)]
        self.kb = np.array([[s[0] for s in r] for r in self.ks])
        self.kh = np.array([[s[1] for s in r] for r in self.ks], np.uint8)
        self.vb = np.array([[s[0] for s in r] for r in self.vs])
        self.vh = np.array([[s[1] for s in r] for r in self.vs], np.uint8)

    def _tile(self, layer, slot):
        page, off = divmod(int(slot), self.page)
        t, tok = divmod(off, TILE)
        return self.data[page, layer][:, t * self.tb:(t + 1) * self.tb], tok

    def append(self, layer, k, v, slots):
        ng = self.dim // self.group
        for x, byte, shift, par_at in ((k, self.kb, self.kh, 16 * self.dim),
                                       (v, self.vb, self.vh, 16 * self.dim + 64 * ng)):
            codes, par = quantise(x, self.group)
            for n, slot in enumerate(slots):
                if slot < 0 or slot >= self.data.shape[0] * self.page:
                    continue
                tile, tok = self._tile(layer, slot)
                for h in range(tile.shape[0]):
                    for d in range(self.dim):
                        b, s = byte[tok, d], shift[tok, d]
                        tile[h, b] = (tile[h, b] & (0xF0 >> s)) | (codes[n, h, d] << s)
                    a = par_at + tok * ng * 4
                    tile[h, a:a + 4 * ng] = np.ascontiguousarray(par[n, h]).view(np.uint8).reshape(-1)

    def read(self, layer, slots):
        """float64 (K, V) [n, heads, dim]: exact values, NaN where the group is."""
        ng = self.dim // self.group
        out = []
        for byte, shift, par_at in ((self.kb, self.kh, 16 * self.dim), (self.vb, self.vh, 16 * self.dim + 64 * ng)):
            rows = np.zeros((len(slots), self.data.shape[2], self.dim))
            for n, slot in enumerate(slots):
                if slot < 0 or slot >= self.data.shape[0] * self.page:
                    continue
                tile, tok = self._tile(layer, slot)
                code = (tile[:, byte[tok]] >> shift[tok]) & 15
                a = par_at + tok * ng * 4
                par = np.ascontiguousarray(tile[:, a:a + 4 * ng]).view(np.float16).reshape(-1, ng, 2).astype(np.float64)
                par = np.repeat(par, self.group, 1)
                rows[n] = par[..., 1] + par[..., 0] * (code.astype(np.float64) - 8)
            out.append(rows)
        return out


def attend(q, k, v, kv_len, causal, scale):
    """One request: q [n, heads, dim], k, v [kv_len, kv_heads, dim] in float64 ->
    (out, lse, slack) where slack bounds what a kernel with 16-bit operands in
    its two products may be off before its output is rounded: half a step of
    fp16, 2^-11, on every k, p and v, with sums in 32 bits (2^-16 on a sum of
    absolute values covers those)."""
    n, heads, dim = q.shape
    ratio = heads // k.shape[1]
    out = np.zeros((n, heads, dim))
    lse = np.full((n, heads), -np.inf)
    slack = np.zeros((n, heads))
    e = 2.0 ** -11 + 2.0 ** -16
    for r in range(n):
        limit = kv_len - (n - 1 - r) if causal else kv_len
        if limit <= 0:
            continue
        for h in range(heads):
            kk, vv = k[:limit, h // ratio], v[:limit, h // ratio]
            s = kk @ q[r, h] * scale
            top = s.max()
            p = np.exp(s - top)
            out[r, h] = p @ vv / p.sum()
            lse[r, h] = top + np.log(p.sum())
            wide = (np.abs(kk) @ np.abs(q[r, h])).max() * abs(scale) * e  # of a score
            # a score off by w moves p by e^w - 1; the weights sum to 1 before and after
            slack[r, h] = np.abs(vv).max() * (2 * np.expm1(wide) + 4 * e)
    return out, lse, slack


def params(pages: Pages, layer, slots):
    """float64 (scale, offset) of K and of V, each [n, heads, dim]."""
    ng = pages.dim // pages.group
    out = []
    for par_at in (16 * pages.dim, 16 * pages.dim + 64 * ng):
        par = np.zeros((len(slots), pages.data.shape[2], ng, 2))
        for n, slot in enumerate(slots):
            tile, tok = pages._tile(layer, slot)
            a = par_at + tok * ng * 4
            par[n] = np.ascontiguousarray(tile[:, a:a + 4 * ng]).view(np.float16).reshape(-1, ng, 2)
        out.append(tuple(np.repeat(par[..., i], pages.group, 2) for i in (0, 1)))
    return out


# Roundings of distinct values are taken as independent and of either sign: a sum of
# them, each at most a_t, passes 7.5 * sqrt(sum a_t^2) once in 10^12 (Hoeffding).
SIGMAS = 7.5


def attend_bounds(q, k, v, kv_len, causal, scale, par=None):
    """One request, as attend() -> (out, lse, tol_out [n, heads, dim], tol_lse [n, heads]):
    how far a kernel may be off before its output is rounded to its type.

    With ``par`` (params() of its tokens) for the kernel of few rows, which multiplies
    raw codes (exact in fp16) and rounds only p * scale_v to fp16; without, for the kernel
    of many rows, whose K, V and p are fp16. e(x) below is 2^-x.

    Sums of products are in 32 bits, with low bits cut off: a step of 16 terms costs
    e(22) of the largest value that the running sum takes. A score: dim / 16 steps of
    up to sum |q| * 15 scale (codes) or sum |q k|; the kernel of few rows also takes sum(q) (dim / 8
    + 4 additions of e(24)) times offset - 8 scale. Its exponential: the argument to e(24)
    relative, the result to e(22). The sum of weights: kv_len / 8 additions of e(24).
    Outputs: kv_len / 16 steps on the running sum; codes are uncentred, 15 scale each, for 8
    tiles of 16 tokens at a time.
    A weight below 2^-14 of the largest, in fp16: e(25) of the largest."""
    n, heads, dim = q.shape
    ratio = heads // k.shape[1]
    few = par is not None
    e = lambda x: 2.0 ** -x  # noqa: E731
    out, lse = np.zeros((n, heads, dim)), np.full((n, heads), -np.inf)
    tol, tol_l = np.zeros((n, heads, dim)), np.zeros((n, heads))
    for r in range(n):
        limit = kv_len - (n - 1 - r) if causal else kv_len
        if limit <= 0:
            continue
        for h in range(heads):
            j = h // ratio
            kk, vv, qq = k[:limit, j], v[:limit, j], q[r, h]
            s = kk @ qq * scale
            p = np.exp(s - s.max())
            total = p.sum()
            lse[r, h] = s.max() + np.log(total)
            p /= total
            o = p @ vv
            out[r, h] = o
            a, extra, extra_l = np.abs(qq), 0.0, 0.0
            if few:
                (ks, ko), (vs, vo) = [tuple(x[:limit, j] for x in both) for both in par]
                w = ((dim / 16 + 1) * e(22) * (15 * ks @ a)
                     + ((dim / 8 + 4) * e(24) + e(22)) * ((np.abs(ko) + 8 * ks) @ a)) * abs(scale)
                c = vv - vo  # scale * (code - 8)
                round_p = SIGMAS * e(11) * np.sqrt(((p[:, None] * c) ** 2).sum(0))
                round_p += limit * e(22) * (p[:, None] * vs).max()  # weights that are subnormal
                steps = 8 * e(22) * 15 * (p[:, None] * vs).sum(0) * 2
                steps += (limit / 16 + 1) * e(22) * np.abs(np.cumsum(p[:, None] * c, 0)).max(0)
                steps += (limit / 8 + 16) * e(24) * (p[:, None] * np.abs(vo)).sum(0)
            else:
                k16, v16 = kk.astype(np.float16).astype(np.float64), vv.astype(np.float16).astype(np.float64)
                s16 = k16 @ qq * scale
                p16 = np.exp(s16 - s16.max())
                extra_l = np.abs(s16.max() + np.log(p16.sum()) - lse[r, h])
                p16 /= p16.sum()
                extra = np.abs(p16 @ v16 - o)
                w = (dim / 16 + 2) * e(22) * (np.abs(kk) @ a) * abs(scale)
                round_p = SIGMAS * e(11) * np.sqrt(((p[:, None] * vv) ** 2).sum(0))
                round_p += limit * e(25) * p.max() * np.abs(vv).max(0)
                steps = (limit / 16 + 1) * e(22) * np.abs(np.cumsum(p[:, None] * vv, 0)).max(0)
            w = np.expm1(w + e(22) + e(23) * (1 + np.abs(s).max()))
            sums = (limit / 8 + 16) * e(24)
            tol[r, h] = (p * w) @ np.abs(vv - o) * 2 + round_p + steps + sums * np.abs(o) + extra
            tol_l[r, h] = (p * w).sum() * 2 + sums + e(22) * (1 + np.abs(lse[r, h])) + extra_l
    return out, lse, tol, tol_l


class Table:
    """PageTable.plan, row by row."""

    def __init__(self, table, kv_lens, borrowed, free, free_count, num_pages, page):
        self.table, self.kv_lens, self.borrowed = table.copy(), kv_lens.copy(), borrowed.copy()
        self.free, self.count, self.num_pages, self.page = list(free[:free_count]), int(free_count), num_pages, page

    def plan(self, q_lens, tokens, done=None):
        ps = self.page
        pages = lambda n: -(-n // ps)  # noqa: E731
        rows, columns = self.table.shape
        if done is not None:
            for r in range(rows):
                if done[r]:
                    self.free += self.table[r, self.borrowed[r]:pages(self.kv_lens[r])].tolist()
                    self.kv_lens[r] = self.borrowed[r] = 0
        slots, pos = np.full(tokens, -1, np.int64), np.zeros(tokens, np.int32)
        start, status = [0], []
        asked = 0  # pages that the rows so far need
        stack = len(self.free)
        for r in range(rows):
            q, length = max(int(q_lens[r]), 0), int(self.kv_lens[r])
            a, b = start[-1], start[-1] + q
            start.append(b)
            fits = b <= tokens and length + q <= columns * ps
            need = pages(length + q) - pages(length) if fits else 0
            asked += need
            ok = fits and (need == 0 or asked <= stack)
            status.append(0 if ok else 2)
            if ok:
                for c in range(pages(length), pages(length) + need):
                    self.table[r, c] = self.free.pop()
            for j in range(a, min(b, tokens)):
                p = length + j - a
                pos[j] = p
                if ok:
                    slots[j] = int(self.table[r, p // ps]) * ps + p % ps
            if ok:
                self.kv_lens[r] = length + q
        return slots, pos, np.array(start, np.int32), np.array(status, np.uint8)
