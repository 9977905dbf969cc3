"""Calls on the paged 4-bit KV cache that are answered without a GPU."""
import pytest

import cascade_cpp
from cascade_cpp import _lib as L
from cascade_cpp import kv4
from oracle import kv4 as O

torch = pytest.importorskip("torch")


def test_a_fill_needs_what_it_fills():
    lib = cascade_cpp._native_lib()
    cache = L.cb_kv4_cache(4096, O.head_bytes(64, 32, 16), None, 4, 1, 1, 64, 16, 32, 0, 0)
    a = dict(q=4096, out=8192, lse=None, block_table=4096, kv_lens=4096, q_start=4096, table_stride=1, scale=1.0,
             columns=1, requests=0, total_q=3, q_heads=2, max_q=1)
    for kw in (dict(fill=L.CB_KV4_FILL_LSE), dict(fill=L.CB_KV4_FILL_OUT, out=None)):
        assert lib.cb_kv4_attend(cache, L.cb_kv4_attend_args(**{**a, **kw}), None) == L.CB_ERR_ARG
    assert lib.cb_kv4_attend(cache, L.cb_kv4_attend_args(**a), None) == L.CB_OK  # no request, nothing to do
    assert lib.cb_kv4_attend(cache, L.cb_kv4_attend_args(**{**a, "total_q": 0, "fill": 3}), None) == L.CB_OK


def test_overlap_of_out_and_q():
    import itertools
    raw = torch.zeros(400, dtype=torch.int16)
    heads, dim, n = 2, 4, 3
    seen = [0, 0]
    for row, head, q_at, out_at in itertools.product((8, 9, 16, 40, 60), (4, 6, 30), (0, 7, 50), range(0, 200, 3)):
        q = raw.as_strided((n, heads, dim), (row, head, 1), q_at)
        out = raw[out_at:out_at + n * heads * dim].view(n, heads, dim)
        mine = {q_at + r * row + h * head + d for r in range(n) for h in range(heads) for d in range(dim)}
        meet = bool(mine & set(range(out_at, out_at + n * heads * dim)))
        said = kv4._overlap(q, out)
        assert said or not meet  # never missed
        if row >= head + dim:  # rows apart from one another: exact but for gaps between heads
            seen[said == meet] += 1
    assert seen[1] > 10 * seen[0]
    assert not kv4._overlap(raw[:0].view(0, 2, 4), raw[:0].view(0, 2, 4))
    one = raw[8:16].view(1, 2, 4)
    assert not kv4._overlap(one, raw[16:24].view(1, 2, 4)) and not kv4._overlap(one, raw[:8].view(1, 2, 4))
    assert kv4._overlap(one, raw[1:9].view(1, 2, 4)) and kv4._overlap(one, raw[15:23].view(1, 2, 4))
