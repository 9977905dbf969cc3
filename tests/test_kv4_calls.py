"""Calls on the paged 4-bit KV cache that are answered without a GPU."""
import pytest

import cascade_cpp
from cascade_cpp import _lib as L
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
