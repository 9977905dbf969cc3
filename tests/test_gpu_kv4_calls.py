"""Calls on the paged 4-bit KV cache that are easy to get wrong: after a refused one, with
values that are not finite, padded, on other streams, on tensors with gradients."""
import numpy as np
import pytest

import cascade_cpp
from cascade_cpp import _lib as L
from cascade_cpp import kv4

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from kv4_cases import hold  # noqa: E402
from test_gpu_kv4 import DEV, make, tables  # noqa: E402


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


def nan_case(token, far, n=100, group=32, which=1):
    """One request of 200 tokens and n rows; a group of a token's V (which 1) or K is NaN.
    ``far``: the token's weight is nothing."""
    cache, ref = make(14, 1, 1, 128, 16, group, seed=7)
    table = np.random.default_rng(3).permutation(14)[None, :13].astype(np.int32)
    kv = [torch.randn(1, 1, 128, device=DEV), torch.randn(1, 1, 128, device=DEV)]
    if far:
        kv[0] = torch.full((1, 1, 128), -60.0, device=DEV)
    kv[which][..., 70] = float("nan")
    slot = int(table[0, token // 16]) * 16 + token % 16
    cache.append(0, *kv, torch.tensor([slot], device=DEV))
    ref.data[:] = cache.cache.cpu().numpy()
    gen = torch.Generator(device=DEV).manual_seed(5)
    q = (1.0 + 0.2 * torch.randn(n, 2, 128, generator=gen, device=DEV)).half()
    return cache, ref, table, q


@pytest.mark.parametrize("token", [40, 198])  # in a full tile; in the last one, which two rows see
@pytest.mark.parametrize("far", [False, True])
@pytest.mark.parametrize("hint", [1, None])   # the kernel for few rows, and for many
@pytest.mark.parametrize("group", [32, 64, 128])
def test_a_nan_group_of_v_is_nan_in_its_dims_whatever_its_weight(token, far, hint, group):
    cache, ref, table, q = nan_case(token, far, group=group)
    out, lse = cache.attend(0, q, torch.from_numpy(table).to(DEV), i32(200), q_start=i32(0, 100), max_q=hint,
                            return_lse=True)
    hold(out, lse, q, ref, 0, table, [200], [100], "fp16", few=hint == 1)


@pytest.mark.parametrize("hint", [1, None])
@pytest.mark.parametrize("group", [32, 64])
def test_a_nan_group_of_v_costs_the_other_groups_of_its_token_nothing(hint, group):
    cache, ref, table, q = nan_case(40, False, group=group)
    v = torch.randn(1, 1, 128, device=DEV)
    v[..., 70] = float("nan")
    slot = int(table[0, 2]) * 16 + 8
    cache.append(0, torch.full_like(v, 60.0), v, torch.tensor([slot], device=DEV))  # nearly all the weight
    ref.data[:] = cache.cache.cpu().numpy()
    out, lse = cache.attend(0, q, torch.from_numpy(table).to(DEV), i32(200), q_start=i32(0, 100), max_q=hint,
                            return_lse=True)
    hold(out, lse, q, ref, 0, table, [200], [100], "fp16", few=hint == 1)


@pytest.mark.parametrize("hint", [1, None])
def test_a_nan_group_of_k_is_nan_in_the_row_and_its_lse(hint):
    cache, ref, table, q = nan_case(198, False, which=0)
    out, lse = cache.attend(0, q, torch.from_numpy(table).to(DEV), i32(200), q_start=i32(0, 100), max_q=hint,
                            return_lse=True)
    assert torch.isnan(out[-2:]).all() and torch.isnan(lse[-2:]).all()
    assert torch.isfinite(out[:-2]).all() and torch.isfinite(lse[:-2]).all()


@pytest.mark.parametrize("rows,hint", [(1, None), (3, None), (70, None)])
def test_a_nan_group_of_v_in_one_part_of_a_long_row(rows, hint):
    cache, ref = make(300, 1, 1, 64, 16, 32, seed=2)
    table = tables(np.random.default_rng(2), [4700], 300, 16)
    v = torch.randn(1, 1, 64, device=DEV)
    v[..., 40] = float("nan")
    slot = int(table[0, 2000 // 16]) * 16 + 2000 % 16
    cache.append(0, torch.zeros_like(v), v, torch.tensor([slot], device=DEV))
    ref.data[:] = cache.cache.cpu().numpy()
    q = torch.randn(rows, 1, 64, device=DEV).half()
    out, lse = cache.attend(0, q, torch.from_numpy(table).to(DEV), i32(4700), q_start=i32(0, rows), return_lse=True)
    hold(out, lse, q, ref, 0, table, [4700], [rows], "fp16")


@pytest.mark.parametrize("dim,qs", [(64, [3, 7]), (128, [1, 1]), (128, [100, 2]), (256, [20, 1])])
@pytest.mark.parametrize("first", [0, 2])
def test_rows_of_no_request_are_zeros_in_a_new_out(dim, qs, first):
    cache, ref = make(20, 1, 2, dim, 16, 64, seed=4)
    table, lens = torch.randperm(20, device=DEV).to(torch.int32).view(2, 10), i32(160, 75)
    start = i32(first, first + qs[0], first + sum(qs))
    rows = first + sum(qs) + 9
    q = torch.randn(rows, 4, dim, device=DEV).bfloat16()
    nan = [torch.full((rows, 4, dim), float("nan"), device=DEV).bfloat16(), torch.full((rows, 4), float("nan"), device=DEV)]
    del nan  # what the allocator hands out next
    out, lse = cache.attend(0, q, table, lens, q_start=start, return_lse=True)
    mine = torch.zeros(rows, dtype=torch.bool, device=DEV)
    mine[first:first + sum(qs)] = True
    assert (out[~mine] == 0).all() and torch.isneginf(lse[~mine]).all()
    hold(out[mine], lse[mine], q[mine], ref, 0, table.cpu().numpy(), [160, 75], qs, "bf16")
    # a given out keeps them
    given = torch.full_like(out, 7.0)
    again, lse = cache.attend(0, q, table, lens, q_start=start, out=given, return_lse=True)
    assert again is given and (given[~mine] == 7).all() and torch.equal(given[mine], out[mine])
    assert torch.isneginf(lse[~mine]).all()


def test_without_requests_every_row_is_zeros():
    cache, _ = make(2, 1, 2, 64, 16, 64, seed=4)
    q = torch.randn(5, 4, 64, device=DEV).half()
    nan = torch.full_like(q, float("nan"))
    del nan
    none = torch.empty(0, dtype=torch.int32, device=DEV)
    out, lse = cache.attend(0, q, torch.empty(0, 3, dtype=torch.int32, device=DEV), none, q_start=i32(0), return_lse=True)
    assert (out == 0).all() and torch.isneginf(lse).all()


def test_a_padded_step_is_captured_and_replayed():
    # the number of tokens of a step moves on inside a graph of a fixed token axis
    cache, _ = make(30, 1, 2, 128, 16, 64, seed=4)
    table, lens = torch.arange(30, dtype=torch.int32, device=DEV).view(3, 10), i32(90, 150, 31)
    start = i32(0, 1, 2, 3)
    q = torch.randn(16, 8, 128, device=DEV).bfloat16()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        cache.attend(0, q, table, lens, q_start=start, max_q=8)
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = cache.attend(0, q, table, lens, q_start=start, max_q=8)
    for now in ([0, 8, 12, 16], [0, 1, 2, 3], [0, 0, 0, 1]):
        start.copy_(i32(*now))
        g.replay()
        want = torch.zeros_like(out)
        cache.attend(0, q, table, lens, q_start=start, max_q=8, out=want)
        assert torch.equal(out, want) and (out[now[-1]:] == 0).all()


def test_a_dry_plan_names_pages_behind_the_rows_and_changes_nothing_else():
    t = kv4.PageTable(3, 8, 20, 16, device=DEV)
    t.plan(i32(20, 0, 33), 53)
    t.block_table[:, 5:] = -1
    before = [x.clone() for x in (t.kv_lens, t.borrowed, t.free, t.free_count, t.block_table)]
    dry = t.plan(i32(40, 3, 0), 50, commit=False)
    assert all(torch.equal(a, b) for a, b in zip(before, (t.kv_lens, t.borrowed, t.free, t.free_count)))
    held = [2, 0, 3]
    for r, n in enumerate(held):
        assert torch.equal(t.block_table[r, :n], before[4][r, :n])
    # the plan's slots are in the table, as its program will read them
    row = torch.tensor([0] * 40 + [1] * 3, device=DEV)
    pos = dry.positions[:43].long()
    assert torch.equal(t.block_table[row, pos // 16].long() * 16 + pos % 16, dry.slots[:43])
    wet = t.plan(i32(40, 3, 0), 50)
    assert all(torch.equal(a, b) for a, b in zip(dry, wet))


def test_a_dry_plan_writes_all_tensors_of_an_earlier_one():
    t = kv4.PageTable(3, 8, 20, 16, device=DEV)
    dry = t.plan(i32(20, 0, 33), 53, commit=False)
    again = t.plan(i32(1, 2, 3), 53, commit=False, out=dry)
    assert all(a.data_ptr() == b.data_ptr() for a, b in zip(again, dry))
    assert dry.kv_lens.tolist() == [1, 2, 3] and dry.free_count.item() == 17 and t.kv_lens.tolist() == [0, 0, 0]
    # a committed plan's lengths are the table's: a dry one never writes those
    wet = t.plan(i32(1, 2, 3), 53, out=dry)
    assert wet.kv_lens is t.kv_lens and wet.free_count is t.free_count
    more = t.plan(i32(5, 5, 5), 53, commit=False, out=wet)
    assert t.kv_lens.tolist() == [1, 2, 3] and t.free_count.item() == 17
    assert more.kv_lens.tolist() == [6, 7, 8] and more.slots.data_ptr() == wet.slots.data_ptr()
    with pytest.raises(ValueError):
        t.plan(i32(1, 1, 1), 53, commit=False, out=dry._replace(kv_lens=i32(0, 0)))


def test_a_page_is_not_given_back_twice():
    t = kv4.PageTable(2, 4, 6, 16, device=DEV)
    pages = t.take(3)
    with pytest.raises(ValueError):
        t.give([pages[0], pages[0]])
    t.give(pages[:1])
    with pytest.raises(ValueError):
        t.give(pages[:2])  # the first one is free already
    assert t.free_count.item() == 4
    t.give(pages[1:])
    assert sorted(t.free.tolist()) == list(range(6))
    with pytest.raises(ValueError):
        t.attach(0, [2, 2], 20)
    t.attach(0, [2, 2], 32, borrowed=True)


def test_tensors_with_gradients_or_tangents_are_refused():
    cache, ref = make(2, 1, 2, 64, 16, 64, seed=4)
    table, lens = torch.zeros(3, 1, dtype=torch.int32, device=DEV), i32(3, 4, 5)
    q, k = torch.randn(3, 4, 64, device=DEV), torch.randn(3, 2, 64, device=DEV)
    at = torch.arange(3, device=DEV)
    before = cache.cache.clone()
    for bad in ((k.clone().requires_grad_(), k), (k, k.clone().requires_grad_())):
        with pytest.raises(ValueError):
            cache.append(0, *bad, at)
    with pytest.raises(ValueError):
        cache.attend(0, q.half(), table, lens, out=torch.empty_like(q).half().requires_grad_())
    import torch.autograd.forward_ad as fwd
    with fwd.dual_level():
        with pytest.raises(ValueError):
            cache.append(0, k, fwd.make_dual(k, k), at)
        with pytest.raises(ValueError):
            cache.attend(0, fwd.make_dual(q.half(), q.half()), table, lens)
        cache.attend(0, q.half(), table, lens)
    assert torch.equal(cache.cache, before)
    with torch.no_grad():
        cache.append(0, k.clone().requires_grad_(), k, at)
        cache.attend(0, q.half().requires_grad_(), table, lens)


def test_out_may_not_overlap_q():
    cache, _ = make(4, 1, 2, 64, 16, 64, seed=4)
    table, lens = torch.zeros(6, 1, dtype=torch.int32, device=DEV), i32(1, 2, 3, 4, 5, 6)
    raw = torch.randn(7, 4, 64, device=DEV).half()
    with pytest.raises(ValueError):
        cache.attend(0, raw[:6], table, lens, out=raw[1:])
    both = torch.randn(12, 4, 64, device=DEV).half()
    want = cache.attend(0, both[:6], table, lens)
    assert torch.equal(cache.attend(0, both[:6], table, lens, out=both[6:]), want)


def test_check_waits_for_calls_on_every_stream():
    cache, _ = make(2, 1, 1, 64, 16, 64, seed=4)
    table = kv4.PageTable(1, 2, 2, 16, device=DEV)
    x = torch.randn(1, 1, 64, device=DEV).half()
    at = torch.tensor([777], device=DEV)
    one, lens = i32(1), i32(-9)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        torch.cuda._sleep(200_000_000)  # about 0.1 s
        cache.append(0, x, x, at)
        table.kv_lens.copy_(lens)
        table.plan(one, 1)
    with pytest.raises(cascade_cpp.CascadeError):
        cache.check()
    with pytest.raises(cascade_cpp.CascadeError):
        table.check()


def test_calls_from_several_threads_on_streams_of_their_own():
    import threading
    cache, _ = make(300, 1, 2, 128, 16, 64, seed=9)
    table = torch.from_numpy(tables(np.random.default_rng(9), [2500, 1300], 300, 16)).to(DEV)
    lens, start = i32(2500, 1300), i32(0, 90, 92)
    qs = [torch.randn(92, 8, 128, device=DEV).bfloat16() for _ in range(4)]
    want = [cache.attend(0, q, table, lens, q_start=start, return_lse=True) for q in qs]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(30):
                got = cache.attend(0, qs[i], table, lens, q_start=start, return_lse=True)
                if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                    wrong.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(qs))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong
    cache.check()


def test_sizes_past_32_bits_are_refused_and_not_wrapped():
    cache, _ = make(2, 1, 1, 64, 16, 64, seed=9)
    x = torch.randn(1, 1, 64, device=DEV).half()
    at, table, lens = torch.tensor([3], device=DEV), torch.zeros(1, 1, dtype=torch.int32, device=DEV), i32(9)
    before = cache.cache.clone()
    for layer in (1 << 32, -(1 << 32)):
        with pytest.raises(cascade_cpp.CascadeError):
            cache.append(layer, x, x, at)
        with pytest.raises(cascade_cpp.CascadeError):
            cache.read(layer, at)
        with pytest.raises(cascade_cpp.CascadeError):
            cache.attend(layer, x, table, lens)
    assert torch.equal(cache.cache, before)
    want = cache.attend(0, x, table, lens)
    assert torch.equal(cache.attend(0, x, table, lens, max_q=(1 << 32) + 1), want)
    with pytest.raises(ValueError):
        kv4.PageTable(1, 2, 2, 16, device=DEV).plan(i32(1), 1 << 32)


def test_a_plan_of_many_tokens_is_captured_and_replayed():
    # the largest cluster, rows that finish and start anew, in a graph
    rng = np.random.default_rng(6)
    eager, graph = (kv4.PageTable(300, 20, 4000, 16, device=DEV) for _ in range(2))
    q, done = torch.zeros(300, dtype=torch.int32, device=DEV), torch.zeros(300, dtype=torch.bool, device=DEV)
    steps = [(torch.from_numpy(rng.integers(0, 130, 300).astype(np.int32)).to(DEV),
              torch.from_numpy(rng.random(300) < 0.5).to(DEV)) for _ in range(8)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        graph.plan(q, 30000, done=done)
    torch.cuda.current_stream().wait_stream(s)
    eager.plan(q, 30000, done=done)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = graph.plan(q, 30000, done=done)
    for a, b in steps:
        q.copy_(a)
        done.copy_(b)
        want = eager.plan(q, 30000, done=done)
        g.replay()
        assert all(torch.equal(x, y) for x, y in zip(got, want))
        assert torch.equal(graph.block_table, eager.block_table)
    graph.check()
