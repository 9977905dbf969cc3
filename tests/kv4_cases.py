"""What the GPU tests of attention over 4-bit pages share: a call held to the oracle's
bounds, and which row tile the library takes for a number of rows."""
import numpy as np
import torch

import cascade_cpp
from cascade_cpp import _lib as L
from oracle import kv4 as O
from test_gpu_kv4 import DEV, TYPES, make, nums, tables

DIMS = [(64, 32), (64, 64), (128, 32), (128, 64), (128, 128), (256, 32), (256, 64), (256, 128), (256, 256)]


def row_tile(dim, group, rows):
    """Rows of a tile of the kernel for few rows, from the workspace that the library asks
    for: 2 * rows * (dim + 2) floats and 21 bytes for every warp of a launch."""
    sms = min(torch.cuda.get_device_properties(0).multi_processor_count & ~1, 256)
    form = L.cb_kv4_cache(4096, 1 << 20, None, 4, 1, 1, dim, 16, group, 0, 0)
    a = L.cb_kv4_attend_args(q=4096, out=4096, block_table=4096, kv_lens=4096, table_stride=1, requests=1, columns=1,
                             total_q=1, q_heads=rows, max_q=1)
    need = cascade_cpp._native_lib().cb_kv4_attend_workspace(form, a)
    found = [n for n in (8, 16, 32) for warps in [sms * 8 * (2 if n == 8 and dim <= 128 else 1)]
             if need == (warps * (21 + 8 * n * (dim + 2)) + 31) // 16 * 16]
    assert len(found) == 1, (need, found)
    return found[0]


def row_tiles(dim, group):
    """{rows of a tile: the least and the most rows of a request that take it}."""
    out = {}
    for rows in range(1, 65):
        out.setdefault(row_tile(dim, group, rows), []).append(rows)
    return {t: (r[0], r[-1]) for t, r in out.items()}


def hold(got, lse, q, cache_ref, layer, table, lens, qs, dtype, causal=True, scale=None, few=None):
    """out and lse of a call against the definition; ``few`` says which kernel a request
    takes (by its rows of a KV head unless given)."""
    heads, dim = q.shape[1:]
    ref, page = cache_ref, cache_ref.page
    ratio = heads // ref.data.shape[2]
    half = torch.finfo(TYPES[dtype]).eps / 2
    at = 0
    for r, (n, m) in enumerate(zip(lens, qs)):
        if not m:
            continue
        slots = [int(table[r, t // page]) * page + t % page for t in range(n)]
        k, v = ref.read(layer, slots)
        is_few = dim == 256 or m * ratio <= 64 if few is None else few
        par = O.params(ref, layer, slots) if is_few else None
        bad = np.isnan(v)
        if par:
            par = [par[0], tuple(np.where(bad, 0.0, x) for x in par[1])]
        want, wl, tol, tol_l = O.attend_bounds(nums(q[at:at + m]).astype(np.float64), k, np.where(bad, 0.0, v), n,
                                               causal, dim ** -0.5 if scale is None else scale, par)
        o = nums(got[at:at + m]).astype(np.float64)
        for i in range(m):  # a NaN of V: in every row that sees it, in its dims
            sees = n - (m - 1 - i) if causal else n
            hit = bad[:max(sees, 0)].any(0).repeat(ratio, 0)
            assert np.array_equal(np.isnan(o[i]), hit), (r, i)
        off = np.abs(o - want)
        limit = np.abs(want) * half * (1 + half) + tol * (1 + half) + 2.0 ** -25  # 2^-25: half of fp16's smallest step
        assert (off <= limit)[~np.isnan(o)].all(), (r, float(np.nanmax(off / limit)))
        if lse is not None:
            le = nums(lse[at:at + m]).astype(np.float64)
            empty = np.isinf(wl)
            assert np.array_equal(np.isneginf(le), empty)
            far = np.abs(le[~empty] - wl[~empty]) / (tol_l[~empty] + 1e-30)
            assert (far <= 1).all(), (r, float(far.max()))
        at += m


def held_call(dtype, dim, group, page, kv_heads, ratio, lens, qs, seed, max_q=None, causal=True, wide=1.0):
    """A call on random pages, held to the bounds."""
    rng = np.random.default_rng(seed)
    pages = sum(-(-n // page) for n in lens) + 1
    cache, ref = make(pages, 2, kv_heads, dim, page, group, seed=seed)
    table = tables(rng, lens, pages, page)
    start = torch.from_numpy(np.concatenate([[0], np.cumsum(qs)]).astype(np.int32)).to(DEV)
    q = torch.from_numpy(rng.standard_normal((sum(qs), kv_heads * ratio, dim)) * wide).to(TYPES[dtype]).to(DEV)
    out, lse = cache.attend(1, q, torch.from_numpy(table).to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV),
                            q_start=start, max_q=max_q, causal=causal, return_lse=True)
    hold(out, lse, q, ref, 1, table, lens, qs, dtype, causal,
         few=True if dim == 256 or (max_q or sum(qs)) * ratio <= 64 else None)
    cache.check()
