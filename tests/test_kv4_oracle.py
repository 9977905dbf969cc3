"""The 4-bit page format on the CPU: the oracle's places of codes against a
second statement of the format, its quantiser's error, and the page table's
rules; and the refusals of the C entry points that need no GPU."""
import ctypes as C

import numpy as np
import pytest

import cascade_cpp
from cascade_cpp import _lib as L
from cascade_cpp import kv4
from oracle import kv4 as O

torch = pytest.importorskip("torch")


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_every_code_has_a_place_of_its_own(dim):
    spots = set()
    for tok in range(16):
        for d in range(dim):
            for byte, shift in (O.k_spot(dim, tok, d), O.v_spot(dim, tok, d)):
                assert shift in (0, 4)
                spots.add((byte, shift))
    assert len(spots) == 2 * 16 * dim
    assert {b for b, _ in spots} == set(range(16 * dim))


@pytest.mark.parametrize("dim,group,page", [(64, 32, 16), (128, 128, 32), (256, 64, 64)])
def test_page_bytes_and_round_trip(dim, group, page):
    layers, heads = 2, 3
    n = kv4.page_bytes(layers, heads, dim, page, group)
    assert n == layers * heads * O.head_bytes(dim, group, page)
    pages = O.Pages(np.zeros((2, layers, heads, n // layers // heads), np.uint8), dim, page, group)
    rng = np.random.default_rng(dim)
    x = rng.standard_normal((20, heads, dim)).astype(np.float16).astype(np.float32)
    slots = rng.permutation(2 * page)[:20]
    pages.append(1, x, -x, slots)
    k, v = pages.read(1, slots)
    span = x.reshape(20, heads, -1, group)
    span = (span.max(-1) - span.min(-1)).max()
    # half a code step, and the fp16 roundings of scale (x15) and offset
    assert np.abs(k - x).max() <= span / 30 + span * 2.0 ** -10 + np.abs(x).max() * 2.0 ** -10
    assert np.abs(v + x).max() <= span / 30 + span * 2.0 ** -10 + np.abs(x).max() * 2.0 ** -10
    assert not pages.data[:, 0].any()  # the other layer is untouched


def test_a_constant_group_is_kept_and_a_nan_shows():
    c, par = O.quantise(np.full((1, 1, 64), 1.5, np.float32), 32)
    assert (c == 8).all() and (par[..., 0] == 0).all() and (par[..., 1] == 1.5).all()
    x = np.zeros((1, 1, 64), np.float32)
    x[0, 0, 3] = np.nan
    _, par = O.quantise(x, 32)
    assert np.isnan(par[0, 0, 0]).all() and not np.isnan(par[0, 0, 1]).any()


@pytest.mark.parametrize("form", [(1, 1, 96, 16, 32), (1, 1, 128, 24, 32), (1, 1, 64, 16, 128), (0, 1, 64, 16, 64),
                                  (1, 1, 128, 8, 64), (1, 1, 128, 16, 16)])
def test_forms_that_are_not_offered(form):
    with pytest.raises(ValueError):
        kv4.page_bytes(*form)
    assert cascade_cpp._native_lib().cb_kv4_page_bytes(*form) == 0


def test_c_entry_points_refuse_before_they_touch_a_gpu():
    lib = cascade_cpp._native_lib()
    good = dict(pages=4096, page_stride=2 * 4 * O.head_bytes(128, 64, 16), errors=None, num_pages=4, layers=2,
                kv_heads=4, head_dim=128, page_size=16, group=64, device=0)

    def cache(**kw):
        return L.cb_kv4_cache(**{**good, **kw})

    def append(c, layer=0, dtype=0, n=1, ptr=4096):
        return lib.cb_kv4_append(c, layer, dtype, ptr, ptr, n, 512, 128, 512, 128, ptr, None)

    bad = [cache(pages=None), cache(pages=4100), cache(page_stride=16), cache(head_dim=80), cache(group=256),
           cache(num_pages=0), cache(page_stride=good["page_stride"] + 8)]
    for c in bad:
        assert append(c) == L.CB_ERR_ARG
        assert lib.cb_kv4_read(c, 0, 0, 4096, 4096, 1, 4096, None) == L.CB_ERR_ARG
        assert lib.cb_kv4_attend(c, L.cb_kv4_attend_args(), None) == L.CB_ERR_ARG
        assert lib.cb_last_error(None)
    c = cache()
    assert append(c, layer=2) == append(c, layer=-1) == append(c, dtype=3) == append(c, n=-1) == L.CB_ERR_ARG
    assert append(c, ptr=None) == append(None) == L.CB_ERR_ARG
    assert append(c, n=0) == L.CB_OK
    assert lib.cb_kv4_read(c, 0, 7, 4096, 4096, 1, 4096, None) == L.CB_ERR_ARG
    assert lib.cb_kv4_read(c, 0, 0, None, 4096, 1, 4096, None) == L.CB_ERR_ARG

    def attend(**kw):
        a = dict(q=4096, out=8192, block_table=4096, kv_lens=4096, table_stride=3, q_token_stride=512,
                 q_head_stride=128, scale=1.0, layer=0, dtype=0, requests=2, columns=3, total_q=2, q_heads=8, max_q=1)
        return lib.cb_kv4_attend(c, L.cb_kv4_attend_args(**{**a, **kw}), None)

    for kw in (dict(dtype=2), dict(q_heads=6), dict(q_heads=0), dict(columns=0), dict(table_stride=-1), dict(total_q=3), dict(out=8200),
               dict(q=None), dict(out=None), dict(kv_lens=None), dict(layer=5), dict(requests=-1),
               dict(columns=1 << 28, table_stride=1 << 28)):
        assert attend(**kw) == L.CB_ERR_ARG, kw
    assert attend(requests=0, total_q=0) == L.CB_OK
    assert lib.cb_kv4_attend(c, None, None) == L.CB_ERR_ARG
    p = dict(q_lens=4096, kv_lens=4096, kv_lens_out=4096, borrowed=4096, block_table=4096, free=4096, free_count=4096,
             free_count_out=4096, slots=4096, positions=4096, q_start=4096, status=4096, table_stride=4, requests=1,
             columns=4, num_pages=8, page_size=16, tokens=1)
    for kw in (dict(requests=-1), dict(tokens=-1), dict(columns=0), dict(page_size=0), dict(table_stride=3),
               dict(num_pages=0), dict(free=None), dict(q_lens=None), dict(slots=None), dict(status=None),
               dict(done=4096, borrowed=None), dict(columns=1 << 28, table_stride=1 << 28)):
        assert lib.cb_kv4_plan(L.cb_kv4_plan_args(**{**p, **kw}), None) == L.CB_ERR_ARG, kw
    assert lib.cb_kv4_plan(None, None) == L.CB_ERR_ARG


def test_struct_layouts_match_c(tmp_path):
    import os
    import subprocess
    header = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")
    lines, want = [], []
    for cls in (L.cb_kv4_cache, L.cb_kv4_plan_args, L.cb_kv4_attend_args):
        lines.append(f'printf("%zu\\n", sizeof({cls.__name__}));')
        want.append(C.sizeof(cls))
        for f, _ in cls._fields_:
            lines.append(f'printf("%zu\\n", offsetof({cls.__name__}, {f}));')
            want.append(getattr(cls, f).offset)
    prog = tmp_path / "layout.c"
    prog.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "cascade_b200.h"\n'
                    "int main(void){" + "".join(lines) + "return 0;}\n")
    subprocess.run(["gcc", "-I", header, str(prog), "-o", str(tmp_path / "layout")], check=True)
    got = subprocess.run([str(tmp_path / "layout")], capture_output=True, text=True).stdout.split()
    assert [int(x) for x in got] == want


def test_python_refuses_host_tensors_and_devices():
    with pytest.raises(TypeError):
        kv4.KV4Cache.over(torch.zeros(2, 1, 1, O.head_bytes(64, 32, 16), dtype=torch.uint8), head_dim=64, group=32)
    with pytest.raises(TypeError):
        kv4.KV4Cache(4, 1, 1, 64, device="cpu")
    with pytest.raises(TypeError):
        kv4.PageTable(2, 4, 8, device="cpu")
    with pytest.raises(ValueError):
        kv4.PageTable(2, 0, 8)
    with pytest.raises(ValueError):
        kv4.PageTable(2, 1 << 28, 8)


def test_table_rules():
    t = O.Table(np.zeros((4, 3), np.int32), np.zeros(4, np.int32), np.zeros(4, np.int32), np.arange(5), 5, 5, 16)
    slots, pos, start, status = t.plan([17, 0, 40, 16], 100)
    # rows 0 and 2 take 2 + 3 pages; row 3 finds none left
    assert status.tolist() == [0, 0, 0, 2] and start.tolist() == [0, 17, 17, 57, 73]
    assert slots[0] == 4 * 16 and slots[16] == 3 * 16 and slots[17] == 2 * 16 and (slots[57:] == -1).all()
    assert t.kv_lens.tolist() == [17, 0, 40, 0]
    slots, *_, status = t.plan([0, 5, 0, 20], 100, done=[1, 0, 0, 0])
    assert status.tolist() == [0, 0, 0, 2]  # row 1 took one of the two pages; row 3 needs two
    assert t.kv_lens.tolist() == [0, 5, 40, 0]
