"""The bounds that attention over 4-bit pages is held to, on the CPU: what a lost or
a repeated part of a long row would change is beyond them."""
import numpy as np
import pytest

from oracle import kv4 as O


def pages(n, heads, dim, group, seed):
    rng = np.random.default_rng(seed)
    count, tb, ng = -(-n // 16), O.tile_bytes(dim, group), dim // group
    data = np.zeros((count, 1, heads, tb), np.uint8)
    data[..., :16 * dim] = rng.integers(0, 256, data[..., :16 * dim].shape, dtype=np.uint8)
    par = np.empty((count, 1, heads, 32 * ng, 2), np.float16)
    par[..., 0] = rng.uniform(0.02, 0.5, par.shape[:-1])
    par[..., 1] = rng.standard_normal(par.shape[:-1]) * 0.4
    data[..., 16 * dim:] = par.view(np.uint8).reshape(count, 1, heads, -1)
    return O.Pages(data, dim, 16, group)


@pytest.mark.parametrize("n,dim,group", [(9000, 128, 128), (4000, 64, 32), (700, 256, 64)])
@pytest.mark.parametrize("few", [True, False])
def test_a_lost_tile_of_a_long_row_is_beyond_the_bounds(n, dim, group, few):
    ref = pages(n, 1, dim, group, seed=n)
    slots = np.arange(n)
    k, v = ref.read(0, slots)
    par = O.params(ref, 0, slots)
    q = np.random.default_rng(1).standard_normal((1, 4, dim)).astype(np.float16).astype(np.float64)
    want, lse, tol, tol_l = O.attend_bounds(q, k, v, n, True, dim ** -0.5, par if few else None)
    for lost in (0, n // 32 * 16, n // 16 * 16 - 16):
        keep = np.ones(n, bool)
        keep[lost:lost + 16] = False
        got, got_l, *_ = O.attend_bounds(q, k[keep], v[keep], n - 16, True, dim ** -0.5)
        assert (np.abs(got_l - lse) > tol_l + 1e-5).all()
        assert (np.abs(got - want) > np.abs(want) * 2.0 ** -11 + tol).any()  # an fp16 output's rounding


def test_scales_and_offsets_give_the_values():
    ref = pages(40, 2, 128, 32, seed=3)
    slots = np.arange(40)
    for x, (scale, offset) in zip(ref.read(0, slots), O.params(ref, 0, slots)):
        code = (x - offset) / scale + 8
        assert np.abs(code - np.rint(code)).max() < 1e-9 and code.min() > -1e-9 and code.max() < 15 + 1e-9
