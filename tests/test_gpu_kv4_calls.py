"""Calls on the paged 4-bit KV cache that are easy to get wrong: after a refused one, with
values that are not finite, padded, on other streams, on tensors with gradients."""
import pytest

import cascade_cpp
from cascade_cpp import _lib as L

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from test_gpu_kv4 import DEV, make  # noqa: E402


def i32(*x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def test_a_refused_call_does_not_break_the_next():
    cache, _ = make(4, 1, 2, 64, 16, 32, seed=1)
    table, lens = torch.arange(4, dtype=torch.int32, device=DEV).view(2, 2), i32(20, 31)
    q = torch.randn(2, 6, 64, device=DEV).half()
    want = make(4, 1, 2, 64, 16, 32, seed=1)[0].attend(0, q, table, lens)
    for layer, x in ((1, q), (-1, q), (0, q.float())):
        with pytest.raises((TypeError, cascade_cpp.CascadeError)):
            cache.attend(layer, x, table, lens)
        assert torch.equal(cache.attend(0, q, table, lens), want)


def test_a_failed_call_leaves_no_error_behind():
    cache, _ = make(2, 1, 1, 64, 16, 64, seed=1)
    lib = cascade_cpp._native_lib()
    x = torch.randn(3, 1, 64, device=DEV).half()
    at = torch.arange(3, device=DEV)
    nowhere = L.cb_kv4_cache(cache.base, cache.stride, None, 2, 1, 1, 64, 16, 64, 99, 0)  # no such device
    call = (0, L.CB_KV4_F16, x.data_ptr(), x.data_ptr(), 3, 64, 64, 64, 64, at.data_ptr(), None)
    assert lib.cb_kv4_append(nowhere, *call) == L.CB_ERR_CUDA
    assert lib.cb_kv4_append(cache._form, *call) == L.CB_OK
    assert lib.cb_kv4_append(nowhere, *call) == L.CB_ERR_CUDA
    (x + 1).sum().item()

