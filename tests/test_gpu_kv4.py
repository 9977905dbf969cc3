"""Paged KV cache held in 4 bits (cascade_cpp.kv4) on the GPU against the numpy
restatement in oracle/kv4.py: page bytes and read values exactly, plans exactly,
attention within half a step of its output type plus what 16-bit operands in the
two products may cost (``slack`` of the oracle, derived there)."""
import ctypes as C

import numpy as np
import pytest

import cascade_cpp
from cascade_cpp import _lib as L
from cascade_cpp import kv4
from oracle import kv4 as O

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DEV = "cuda:0"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def make(pages, layers, heads, dim, page, group, seed=None, store=None):
    """A cache and its oracle twin; with a seed, full of random codes and sane
    parameters, and NaN parameters in the layers that are not used."""
    n = O.head_bytes(dim, group, page)
    data = np.zeros((pages, layers, heads, n), np.uint8)
    if seed is not None:
        rng = np.random.default_rng(seed)
        tb, ng = O.tile_bytes(dim, group), dim // group
        tiles = data.reshape(pages, layers, heads, page // 16, tb)
        tiles[..., :16 * dim] = rng.integers(0, 256, tiles[..., :16 * dim].shape, dtype=np.uint8)
        par = np.empty((pages, layers, heads, page // 16, 2 * 16 * ng, 2), np.float16)
        par[..., 0] = rng.uniform(0.02, 0.5, par.shape[:-1])
        par[..., 1] = rng.standard_normal(par.shape[:-1]) * 0.4
        tiles[..., 16 * dim:] = par.view(np.uint8).reshape(*par.shape[:-2], -1)
    cache = kv4.KV4Cache.over(torch.from_numpy(data.copy()).to(DEV), head_dim=dim, page_size=page, group=group,
                              store=store)
    return cache, O.Pages(data, dim, page, group)


def nums(t):
    return t.detach().float().cpu().numpy()


def rounded(x, dtype):
    """float64 -> the values of a type, through float32 as the product defines it."""
    return torch.from_numpy(x.astype(np.float32)).to(dtype)


FORMS = [("bf16", 128, 128, 16, 4), ("fp16", 128, 32, 32, 3), ("fp32", 64, 64, 16, 1), ("bf16", 64, 32, 64, 5),
         ("fp16", 256, 64, 16, 2), ("bf16", 256, 256, 128, 1), ("fp16", 128, 64, 256, 2)]


@pytest.mark.parametrize("dtype,dim,group,page,heads", FORMS)
@pytest.mark.parametrize("n", [1, 37])
def test_append_and_read_match_the_format(dtype, dim, group, page, heads, n):
    rng = np.random.default_rng(dim + group + n)
    cache, ref = make(5, 2, heads, dim, page, group)
    x = rng.standard_normal((2, n, heads, dim)) * rng.choice([1e-4, 1.0, 30.0], (2, n, heads, 1))
    k, v = (torch.from_numpy(a).to(TYPES[dtype]).to(DEV) for a in x)
    slots = rng.permutation(5 * page)[:n].astype(np.int64)
    if n > 4:
        slots[[1, n - 1]] = -1
        k[2, 0, :3] = torch.tensor([70000.0, -1e30, 3.0]) if dtype != "fp16" else 65504.0
        k[3] = 0.25  # constant groups
    cache.append(1, k, v, torch.from_numpy(slots).to(DEV))
    ref.append(1, nums(k), nums(v), slots)
    assert np.array_equal(cache.cache.cpu().numpy(), ref.data)
    cache.check()
    back = cache.read(1, torch.from_numpy(slots).to(DEV), dtype=TYPES[dtype])
    for got, want in zip(back, ref.read(1, slots)):
        assert got.dtype == TYPES[dtype]
        assert torch.equal(got.cpu(), rounded(want, TYPES[dtype]))


def test_append_takes_slices_of_a_fused_projection_and_odd_addresses():
    rng = np.random.default_rng(3)
    for shift in (0, 1, 8):  # elements: 1 leaves no 16-byte boundary
        cache, ref = make(3, 1, 4, 128, 16, 64)
        width = (12 + 2 * 4) * 128 + 16
        flat = torch.from_numpy(rng.standard_normal(23 * width + 8)).to(torch.bfloat16).to(DEV)
        qkv = flat[shift:shift + 23 * width].view(23, width)
        k = qkv[:, 12 * 128:16 * 128].view(23, 4, 128)
        v = qkv[:, 16 * 128:20 * 128].view(23, 4, 128).flip(1).as_strided((23, 4, 128), (4 * 128, 128, 1))
        slots = torch.from_numpy(rng.permutation(48)[:23].astype(np.int64)).to(DEV)
        cache.append(0, k, v, slots)
        ref.append(0, nums(k), nums(v), slots.cpu().numpy())
        assert np.array_equal(cache.cache.cpu().numpy(), ref.data)


def test_nan_shows_and_stays_in_its_group():
    cache, ref = make(1, 1, 1, 128, 16, 32)
    k = torch.randn(2, 1, 128, device=DEV)
    k[1, 0, 40] = float("nan")
    at = torch.arange(2, device=DEV)
    cache.append(0, k, k, at)
    got, _ = cache.read(0, at, dtype=torch.float32)
    bad = torch.isnan(got).cpu().numpy()
    assert bad[1, 0, 32:64].all() and bad.sum() == 32


def test_slots_outside_the_cache_are_skipped_and_reported():
    cache, ref = make(2, 1, 2, 64, 16, 32, seed=1)
    k = torch.randn(4, 2, 64, device=DEV).half()
    slots = torch.tensor([32, 5, 1 << 40, -7], device=DEV)
    cache.append(0, k, k, slots)
    ref.append(0, nums(k), nums(k), slots.cpu().numpy())
    assert np.array_equal(cache.cache.cpu().numpy(), ref.data)
    with pytest.raises(cascade_cpp.CascadeError):
        cache.check()
    cache.check()  # reported once
    a, b = cache.read(0, slots, dtype=torch.float16)
    assert not a[[0, 2, 3]].any() and not b[[0, 2, 3]].any() and a[1].any()
    with pytest.raises(cascade_cpp.CascadeError):
        cache.check()
    empty = torch.empty(0, dtype=torch.int64, device=DEV)
    cache.append(0, k[:0], k[:0], empty)
    assert cache.read(0, empty)[0].shape == (0, 2, 64)
    cache.check()


def test_pages_depend_on_their_tokens_alone_and_deduplicate():
    cfg = cascade_cpp.DistributedConfig()
    cfg.gpu_capacity_per_device = 64 << 20
    cfg.dram_capacity = 0
    cfg.device = 0
    store = cascade_cpp.DistributedStore(cfg)
    cache = kv4.KV4Cache(8, 2, 4, 128, 32, 64, device=DEV, store=store)
    k = torch.randn(64, 4, 128, device=DEV, dtype=torch.bfloat16)
    v = torch.randn(64, 4, 128, device=DEV, dtype=torch.bfloat16)
    at = torch.arange(64, device=DEV)
    for layer in range(2):
        cache.append(layer, k, v, at)                              # pages 0 and 1 at once
        for j in torch.randperm(64).tolist():                      # pages 5 and 3, a token at a time
            cache.append(layer, k[j:j + 1], v[j:j + 1], torch.tensor([(5 if j < 32 else 3) * 32 + j % 32], device=DEV))
    assert torch.equal(cache.cache[[5, 3]], cache.cache[:2])
    ids, status = cache.save([0, 1, 5, 3], return_status=True)
    assert status == [0, 0, 1, 1] and ids[:2] == ids[2:]
    assert cache.load(ids[:2], [6, 7]) == [True, True]
    assert torch.equal(cache.cache[6:], cache.cache[:2])
    store.close()


# ------------------------------------------------------------------- the plan

def same_table(t, ref, plan, want):
    slots, pos, start, status = want
    assert plan.slots.tolist() == slots.tolist()
    assert plan.positions.tolist() == pos.tolist()
    assert plan.q_start.tolist() == start.tolist()
    assert plan.status.tolist() == status.tolist()
    assert plan.kv_lens.tolist() == ref.kv_lens.tolist()
    assert plan.free_count.tolist() == [len(ref.free)]
    assert t.free[:len(ref.free)].tolist() == ref.free
    ps = ref.page
    for r in range(len(ref.kv_lens)):
        n = -(-int(ref.kv_lens[r]) // ps)
        assert t.block_table[r, :n].tolist() == ref.table[r, :n].tolist()


@pytest.mark.parametrize("rows,columns,pages,page,most", [(1, 40, 64, 16, 30), (7, 12, 40, 16, 60), (37, 9, 200, 32, 90),
                                                          (1300, 6, 4000, 16, 20), (5, 700, 3500, 16, 9000)])
def test_steps_of_a_page_table(rows, columns, pages, page, most):
    rng = np.random.default_rng(rows)
    t = kv4.PageTable(rows, columns, pages, page, device=DEV)
    ref = O.Table(t.block_table.cpu().numpy(), np.zeros(rows, np.int32), np.zeros(rows, np.int32),
                  t.free.cpu().numpy(), pages, pages, page)
    refused = 0
    for step in range(6):
        q = rng.integers(0, most + 1, rows).astype(np.int32)
        q[rng.random(rows) < 0.3] = 0
        if step == 2:
            q[0] = -5
        done = rng.random(rows) < 0.4 if step else None
        tokens = int(q.clip(0).sum()) + (3 if step != 3 else -int(q.clip(0).sum()) // 3)
        d = None if done is None else torch.from_numpy(done).to(DEV)
        plan = t.plan(torch.from_numpy(q).to(DEV), tokens, done=d)
        want = ref.plan(q, tokens, done)
        same_table(t, ref, plan, want)
        refused += int((want[3] != 0).sum())
    assert refused or rows == 1
    t.check()


def test_a_dry_plan_leaves_the_table_and_a_borrowed_prefix_its_owner():
    t = kv4.PageTable(3, 8, 20, 16, device=DEV)
    assert t.take(2) == [0, 1]
    t.attach(0, [0, 1], 32, borrowed=True)
    t.attach(2, [0, 1], 32, borrowed=True)
    q = torch.tensor([5, 16, 33], dtype=torch.int32, device=DEV)
    before = [x.clone() for x in (t.kv_lens, t.free_count, t.borrowed)]
    dry = t.plan(q, 54, commit=False)
    assert all(torch.equal(a, b) for a, b in zip(before, (t.kv_lens, t.free_count, t.borrowed)))
    wet = t.plan(q, 54)
    assert all(torch.equal(a, b) for a, b in zip(dry, wet))
    assert wet.slots[:5].tolist() == [2 * 16 + i for i in range(5)] and wet.positions[0] == 32
    done = torch.ones(3, dtype=torch.bool, device=DEV)
    again = t.plan(torch.zeros_like(q), 54, done=done, out=wet)
    assert again.slots.data_ptr() == wet.slots.data_ptr() and (again.slots == -1).all()
    assert t.free_count.item() == 18 and sorted(t.free[:18].tolist()) == list(range(2, 20))
    t.give([0, 1])
    assert t.free_count.item() == 20
    with pytest.raises(cascade_cpp.CascadeError):
        t.give([3])
    with pytest.raises(cascade_cpp.CascadeError):
        t.take(21)
    with pytest.raises(ValueError):
        t.plan(q, 54, done=done, commit=False)
    with pytest.raises(ValueError):
        t.attach(0, [1], 12, borrowed=True)
    with pytest.raises(IndexError):
        t.attach(3, [], 0)
    t.attach(1, [4], 9)
    with pytest.raises(ValueError):
        t.attach(1, [5], 3)  # not empty


def test_a_table_set_wrongly_is_reported_and_harms_nothing():
    t = kv4.PageTable(3, 4, 8, 16, device=DEV)
    t.kv_lens.copy_(torch.tensor([-3, 1000, 20]))
    t.block_table[2, :2] = torch.tensor([3, 77])
    p = t.plan(torch.tensor([1, 1, 1], dtype=torch.int32, device=DEV), 3)
    assert p.status.tolist() == [2, 2, 0] and p.slots.tolist() == [-1, -1, -1]
    with pytest.raises(cascade_cpp.CascadeError):
        t.check()
    t.plan(torch.zeros(3, dtype=torch.int32, device=DEV), 0, done=torch.ones(3, dtype=torch.uint8, device=DEV))
    assert 0 <= t.free_count.item() <= 8
    with pytest.raises(cascade_cpp.CascadeError):
        t.check()


def test_plans_without_rows_or_tokens():
    t = kv4.PageTable(0, 4, 8, 16, device=DEV)
    p = t.plan(torch.empty(0, dtype=torch.int32, device=DEV), 5)
    assert p.slots.tolist() == [-1] * 5 and p.q_start.tolist() == [0] and p.free_count.item() == 8
    t = kv4.PageTable(2, 4, 8, 16, device=DEV)
    p = t.plan(torch.tensor([0, 3], dtype=torch.int32, device=DEV), 0)
    assert p.status.tolist() == [0, 2] and p.q_start.tolist() == [0, 0, 3] and t.kv_lens.tolist() == [0, 0]


# ------------------------------------------------------------------ attention

def tables(rng, lens, pages, page, spare=1):
    cols = max(1, max(-(-n // page) for n in lens)) + spare
    table = rng.integers(0, pages, (len(lens), cols)).astype(np.int32)
    ids = rng.permutation(pages)
    at = 0
    for r, n in enumerate(lens):
        m = -(-n // page)
        table[r, :m] = ids[at:at + m]
        at += m
    assert at <= pages
    return table


def attend_case(dtype, dim, group, page, kv_heads, ratio, lens, qs, causal=True, seed=0, scale=None, lse=True,
                spare_rows=0, one_row=False, wide=1.0, max_q=None):
    rng = np.random.default_rng(seed)
    total_pages = sum(-(-n // page) for n in lens) + 3
    cache, ref = make(total_pages, 2, kv_heads, dim, page, group, seed=seed)
    table = tables(rng, lens, total_pages, page)
    # what no row may see holds NaN and infinity in its parameters
    tb, ng = O.tile_bytes(dim, group), dim // group
    seen = np.zeros((total_pages, page), bool)
    for r, n in enumerate(lens):
        for t in range(n):
            seen[table[r, t // page], t % page] = True
    par = ref.data.reshape(total_pages, 2, kv_heads, page // 16, tb)[..., 16 * dim:].copy()
    par = par.view(np.float16).reshape(total_pages, 2, kv_heads, page // 16, 2, 16, ng, 2)
    hidden = ~seen.reshape(total_pages, page // 16, 16)
    for p in range(total_pages):
        for i in range(page // 16):
            par[p, :, :, i][:, :, :, hidden[p, i]] = [np.nan, np.inf]
    ref.data.reshape(total_pages, 2, kv_heads, page // 16, tb)[..., 16 * dim:] = \
        par.reshape(total_pages, 2, kv_heads, page // 16, -1).view(np.uint8)
    cache.cache.copy_(torch.from_numpy(ref.data))
    start = np.concatenate([[0], np.cumsum(qs)]).astype(np.int32)
    rows = int(start[-1]) + spare_rows
    fused = torch.from_numpy(rng.standard_normal((rows, kv_heads * ratio + 2, dim)) * wide).to(TYPES[dtype]).to(DEV)
    q = fused[:, 1:-1]
    out = torch.full((rows, kv_heads * ratio, dim), 7.0, dtype=TYPES[dtype], device=DEV)
    got = cache.attend(1, q, torch.from_numpy(table).to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV),
                       q_start=None if one_row else torch.from_numpy(start).to(DEV), max_q=max_q, causal=causal,
                       scale=scale, out=out, return_lse=lse)
    o, e = got if lse else (got, None)
    assert o is out
    sc = dim ** -0.5 if scale is None else scale
    half = torch.finfo(TYPES[dtype]).eps / 2
    for r, n in enumerate(lens):
        a, b = start[r], start[r + 1]
        if a == b:
            continue
        k, v = ref.read(1, [int(table[r, t // page]) * page + t % page for t in range(n)])
        want, wl, slack = O.attend(nums(q[a:b]).astype(np.float64), k, v, n, causal, sc)
        off = np.abs(nums(o[a:b]) - want)
        tol = np.abs(want) * half * (1 + half) + slack[..., None] + 1e-7
        assert (off <= tol).all(), (r, n, float((off / tol).max()))
        if lse:
            le = nums(e[a:b])
            empty = np.isinf(wl)
            assert np.array_equal(np.isneginf(le), empty)
            # a score is off by what 16-bit keys cost, the sum of weights by no more; sums are in 32 bits
            wide_l = (np.abs(k).reshape(n, kv_heads, dim).max((0, 2)).repeat(ratio)[None]
                      * np.abs(nums(q[a:b])).sum(-1) * abs(sc)) * (2.0 ** -11 + 2.0 ** -16) if n else 0.0
            wide_l = np.broadcast_to(wide_l, wl.shape)[~empty]
            assert (np.abs(le[~empty] - wl[~empty]) <= wide_l + 1e-5 * (1 + np.abs(wl[~empty]))).all()
    if spare_rows:
        assert (o[start[-1]:] == 7.0).all()
    cache.check()
    return cache


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("dim,group", [(64, 32), (64, 64), (128, 32), (128, 64), (128, 128), (256, 32), (256, 64),
                                       (256, 128), (256, 256)])
def test_attend_single_tokens(dtype, dim, group):
    lens = [0, 1, 15, 16, 17, 130, 301]
    attend_case(dtype, dim, group, 16, 2, 7, lens, [1] * len(lens), seed=dim + group, one_row=True)


@pytest.mark.parametrize("ratio", [1, 2, 5, 8, 9, 16, 33])
@pytest.mark.parametrize("page", [16, 64, 256])
def test_attend_head_groups_and_pages(ratio, page):
    attend_case("bf16", 128, 64, page, 3, ratio, [77, 3, 200], [1, 1, 1], seed=ratio)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dim,ratio", [(64, 4), (128, 1), (128, 7), (256, 3)])
def test_attend_several_tokens(causal, dim, ratio):
    # rows of no request, requests of no rows, more rows than tokens (rows that see nothing)
    attend_case("fp16", dim, 64, 32, 2, ratio, [40, 100, 5, 0, 33, 64], [3, 0, 9, 2, 33, 1], causal=causal, seed=ratio,
                spare_rows=5)


@pytest.mark.parametrize("dim,group,ratio", [(64, 32, 8), (128, 128, 7), (128, 32, 1), (128, 64, 4), (256, 64, 2)])
def test_attend_prompt_chunks(dim, group, ratio):
    attend_case("bf16", dim, group, 16, 1, ratio, [300, 513, 140], [130, 65, 140], seed=dim + ratio, spare_rows=1)


@pytest.mark.parametrize("hint", [1, 3, 40, 5000])
def test_the_hint_does_not_change_what_is_right(hint):
    attend_case("bf16", 128, 64, 16, 2, 4, [90, 31], [37, 2], max_q=hint, seed=5)


def test_attend_long_rows_are_split_and_joined():
    attend_case("fp16", 128, 128, 64, 1, 4, [9000, 4000, 1], [1, 2, 1], seed=8)


def test_attend_many_rows():
    rng = np.random.default_rng(1)
    lens = rng.integers(0, 60, 300).tolist()
    attend_case("bf16", 64, 64, 16, 1, 2, lens, [1] * 300, seed=2, one_row=True)


def test_attend_a_prompt_behind_a_long_prefix():
    attend_case("bf16", 128, 128, 64, 1, 1, [6100], [70], seed=3)


def test_attend_many_requests_of_both_kinds():
    # single tokens beside chunks (each kernel takes its own), more requests than a block has threads
    rng = np.random.default_rng(4)
    qs = rng.choice([0, 1, 2, 17], 540).tolist()
    lens = [int(q + rng.integers(0, 25)) for q in qs]
    attend_case("fp16", 64, 64, 16, 1, 4, lens, qs, seed=4, max_q=17)


@pytest.mark.parametrize("rows", [2, 90])
def test_q_may_lie_on_odd_addresses(rows):
    cache, _ = make(8, 1, 2, 128, 16, 64, seed=3)
    table = torch.arange(8, dtype=torch.int32, device=DEV).view(1, 8)
    lens = torch.tensor([125], dtype=torch.int32, device=DEV)
    start = torch.tensor([0, rows], dtype=torch.int32, device=DEV)
    q = torch.randn(rows, 6, 128, device=DEV).bfloat16()
    odd = torch.empty(rows * 6 * 131 + 1, dtype=q.dtype, device=DEV)[1:].view(rows, 6, 131)[:, :, :128]
    odd.copy_(q)
    want = cache.attend(0, q, table, lens, q_start=start)
    assert torch.equal(cache.attend(0, odd, table, lens, q_start=start), want)


@pytest.mark.parametrize("wide,scale", [(300.0, None), (1e-3, None), (1.0, 0.0), (1.0, -0.5), (2e-6, 3e4)])
def test_attend_large_and_tiny_scores(wide, scale):
    attend_case("bf16", 128, 64, 16, 2, 4, [100, 65], [1, 40], seed=4, wide=wide, scale=scale)


def test_attend_without_rows():
    cache, _ = make(2, 1, 2, 64, 16, 32, seed=1)
    table = torch.zeros(0, 1, dtype=torch.int32, device=DEV)
    none = torch.empty(0, dtype=torch.int32, device=DEV)
    q = torch.empty(0, 4, 64, dtype=torch.float16, device=DEV)
    assert cache.attend(0, q, table, none).shape == (0, 4, 64)
    start = torch.zeros(3, dtype=torch.int32, device=DEV)
    table, lens = torch.zeros(2, 1, dtype=torch.int32, device=DEV), torch.tensor([5, 9], dtype=torch.int32, device=DEV)
    assert cache.attend(0, q, table, lens, q_start=start).shape == (0, 4, 64)


def test_pages_outside_the_cache_are_skipped_and_reported():
    cache, ref = make(4, 1, 1, 128, 16, 128, seed=3)
    table = np.array([[1, 9, 2, -4, 3]], np.int32)
    q = torch.randn(1, 4, 128, device=DEV).half()
    for rows in (1, 90):  # the kernels for few and for many rows
        qq = q.repeat(rows, 1, 1)
        got = cache.attend(0, qq, torch.from_numpy(table).to(DEV), torch.tensor([80], dtype=torch.int32, device=DEV),
                           q_start=torch.tensor([0, rows], dtype=torch.int32, device=DEV), causal=False)
        slots = [p * 16 + i for p in (1, 2, 3) for i in range(16)]
        k, v = ref.read(0, slots)
        want, _, slack = O.attend(nums(q).astype(np.float64), k, v, len(slots), False, 128 ** -0.5)
        assert (np.abs(nums(got) - want) <= np.abs(want) * 2.0 ** -11 + slack[..., None] + 1e-7).all()
        with pytest.raises(cascade_cpp.CascadeError):
            cache.check()


def test_lengths_outside_the_table_are_cut_and_reported():
    cache, ref = make(2, 1, 1, 64, 16, 64, seed=3)
    table = torch.tensor([[1], [0]], dtype=torch.int32, device=DEV)
    q = torch.randn(2, 1, 64, device=DEV).half()
    lens = torch.tensor([16, 0], dtype=torch.int32, device=DEV)
    want = cache.attend(0, q, table, lens)
    cache.check()
    got = cache.attend(0, q, table, torch.tensor([500, -2], dtype=torch.int32, device=DEV))
    assert torch.equal(got, want)
    with pytest.raises(cascade_cpp.CascadeError):
        cache.check()


def test_q_with_nan_or_infinity_keeps_to_its_rows():
    cache, _ = make(8, 1, 2, 128, 16, 64, seed=3)
    for n in (2, 100):
        q = torch.randn(n, 8, 128, device=DEV).bfloat16()
        table = torch.arange(8, dtype=torch.int32, device=DEV).view(1, 8)
        lens = torch.tensor([120], dtype=torch.int32, device=DEV)
        start = torch.tensor([0, n], dtype=torch.int32, device=DEV)
        want = cache.attend(0, q, table, lens, q_start=start)
        q[1, 3, 5] = float("nan")
        q[0, 6, 5] = float("inf")
        got = cache.attend(0, q, table, lens, q_start=start)
        assert torch.isnan(got[1, 3]).all() and torch.isnan(got[0, 6]).all()
        keep = torch.ones(n, 8, dtype=torch.bool, device=DEV)
        keep[1, 3] = keep[0, 6] = False
        assert torch.equal(got[keep], want[keep])


@pytest.mark.parametrize("n,ratio", [(3, 2), (100, 4)])  # the kernels for few and for many rows
@pytest.mark.parametrize("which", [0, 1])
def test_a_token_that_is_nan_stays_hidden_from_the_rows_before_it(n, ratio, which):
    cache, _ = make(16, 1, 1, 128, 16, 64, seed=6)
    table = torch.randperm(16, device=DEV).to(torch.int32).view(1, 16)
    lens = torch.tensor([250], dtype=torch.int32, device=DEV)
    start = torch.tensor([0, n], dtype=torch.int32, device=DEV)
    q = torch.randn(n, ratio, 128, device=DEV).bfloat16()
    want = cache.attend(0, q, table, lens, q_start=start)
    # the token that the last two rows see, behind what the others do
    slot = torch.tensor([int(table[0, 248 // 16]) * 16 + 248 % 16], device=DEV)
    kv = [torch.randn(1, 1, 128, device=DEV), torch.randn(1, 1, 128, device=DEV)]
    kv[which][:] = float("nan")
    cache.append(0, *kv, slot)
    got, lse = cache.attend(0, q, table, lens, q_start=start, return_lse=True)
    assert torch.equal(got[:-2], want[:-2]) and torch.isfinite(lse[:-2]).all()
    assert torch.isnan(got[-2:]).all()


def test_requests_may_share_one_row_of_a_table():
    cache, _ = make(4, 1, 2, 64, 16, 32, seed=1)
    table = torch.tensor([[2, 0, 3]], dtype=torch.int32, device=DEV)
    lens = torch.tensor([5, 40, 48], dtype=torch.int32, device=DEV)
    q = torch.randn(3, 4, 64, device=DEV).half()
    want = cache.attend(0, q, table.repeat(3, 1), lens)
    assert torch.equal(cache.attend(0, q, table.expand(3, 3), lens), want)
    wide = torch.zeros(3, 50, dtype=torch.int32, device=DEV)
    wide[:, 7:10] = table
    assert torch.equal(cache.attend(0, q, wide[:, 7:10], lens), want)


def test_a_cache_past_4_gib():
    # pages that lie 2.2 GiB apart: offsets pass 32 bits
    heads, dim = 1, 128
    n = O.head_bytes(dim, 128, 16)
    stride = (2200 << 20) // 16 * 16
    raw = torch.empty(2 * stride + n, dtype=torch.uint8, device=DEV)
    cache = kv4.KV4Cache.over(raw.as_strided((3, 1, heads, n), (stride, n, n, 1)), head_dim=dim, group=128)
    k = torch.randn(48, heads, dim, device=DEV).half()
    v = torch.randn(48, heads, dim, device=DEV).half()
    small, _ = make(3, 1, heads, dim, 16, 128)
    at = torch.arange(48, device=DEV)
    table = torch.tensor([[2, 0, 1]], dtype=torch.int32, device=DEV)
    lens = torch.tensor([48], dtype=torch.int32, device=DEV)
    outs = []
    for c in (cache, small):
        c.append(0, k, v, at)
        start = torch.tensor([0, 40], dtype=torch.int32, device=DEV)
        outs.append((*c.read(0, at), c.attend(0, k[:1], table, lens), c.attend(0, k[:40], table, lens, q_start=start)))
        c.check()
    assert all(torch.equal(a, b) for a, b in zip(*outs))


def test_results_do_not_change_from_run_to_run():
    rng = np.random.default_rng(9)
    cache, _ = make(700, 1, 2, 128, 16, 64, seed=9)
    lens = [4000, 3000, 900, 2500]
    table = torch.from_numpy(tables(rng, lens, 700, 16)).to(DEV)
    kv = torch.tensor(lens, dtype=torch.int32, device=DEV)
    for qs in ([1, 1, 1, 1], [150, 3, 60, 1]):
        start = torch.tensor(np.concatenate([[0], np.cumsum(qs)]), dtype=torch.int32, device=DEV)
        q = torch.randn(sum(qs), 8, 128, device=DEV).bfloat16()
        first = cache.attend(0, q, table, kv, q_start=start, return_lse=True)
        for _ in range(5):
            again = cache.attend(0, q, table, kv, q_start=start, return_lse=True)
            assert all(torch.equal(a, b) for a, b in zip(first, again))


# ---------------------------------------------------- together, as a program runs

def step_tensors(rng, heads, kv_heads, dim, n):
    mk = lambda h: torch.from_numpy(rng.standard_normal((n, h, dim))).to(torch.bfloat16).to(DEV)  # noqa: E731
    return mk(heads), mk(kv_heads), mk(kv_heads)


def run_steps(steps, layers=2, stream=None):
    """Two requests' prompts, then single tokens, then one leaves and another comes."""
    rng = np.random.default_rng(12)
    table = kv4.PageTable(3, 20, 40, 16, device=DEV)
    cache = kv4.KV4Cache(40, layers, 2, 128, 16, 64, device=DEV)
    outs = []
    for q_lens, done in steps:
        n = sum(q_lens)
        plan = table.plan(torch.tensor(q_lens, dtype=torch.int32, device=DEV), n,
                          done=None if done is None else torch.tensor(done, device=DEV))
        for layer in range(layers):
            q, k, v = step_tensors(rng, 8, 2, 128, n)
            cache.append(layer, k, v, plan.slots)
            outs.append(cache.attend(layer, q, table.block_table, table.kv_lens, q_start=plan.q_start))
    cache.check()
    table.check()
    return outs, table


STEPS = [([50, 0, 131], None), ([1, 0, 1], None), ([1, 20, 1], None), ([7, 1, 1], [True, False, False]),
         ([1, 1, 1], None)]


def test_steps_of_serving_match_attention_over_what_was_appended():
    outs, table = run_steps(STEPS)
    rng = np.random.default_rng(12)
    held = {(layer, r): ([], []) for layer in range(2) for r in range(3)}
    i = 0
    for q_lens, done in STEPS:
        for r in range(3):
            if done and done[r]:
                for layer in range(2):
                    held[layer, r] = ([], [])
        for layer in range(2):
            q, k, v = (nums(x).astype(np.float64) for x in step_tensors(rng, 8, 2, 128, sum(q_lens)))
            got, at = nums(outs[i]), 0
            i += 1
            for r, n in enumerate(q_lens):
                if not n:
                    continue
                for x, to in ((k, held[layer, r][0]), (v, held[layer, r][1])):
                    c, par = O.quantise(x[at:at + n], 64)
                    par = np.repeat(par.astype(np.float64), 64, -2)
                    to.extend(par[..., 1] + par[..., 0] * (c.astype(np.float64) - 8))
                kk, vv = (np.array(x) for x in held[layer, r])
                want, _, slack = O.attend(q[at:at + n], kk, vv, len(kk), True, 128 ** -0.5)
                off = np.abs(got[at:at + n] - want)
                assert (off <= np.abs(want) * 2.0 ** -8 + slack[..., None] + 1e-7).all()
                at += n
    assert table.kv_lens.tolist() == [8, 22, 135]


def test_steps_on_another_stream_give_the_same():
    want, _ = run_steps(STEPS)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got, _ = run_steps(STEPS)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))


def test_a_step_is_captured_and_replayed():
    # decode steps of one graph: the table moves on inside it
    rng = np.random.default_rng(2)
    tables_, caches = [], []
    for _ in range(2):
        tables_.append(kv4.PageTable(3, 20, 60, 16, device=DEV))
        caches.append(kv4.KV4Cache(60, 1, 2, 128, 16, 64, device=DEV))
    ql = torch.tensor([1, 1, 0], dtype=torch.int32, device=DEV)
    q, k, v = step_tensors(rng, 14, 2, 128, 3)
    news = [step_tensors(rng, 14, 2, 128, 3) for _ in range(40)]

    def step(i, buf):
        plan = tables_[i].plan(ql, 3)
        caches[i].append(0, buf[1], buf[2], plan.slots)
        out = torch.zeros_like(buf[0])
        return caches[i].attend(0, buf[0], tables_[i].block_table, tables_[i].kv_lens, q_start=plan.q_start, max_q=1,
                                out=out)

    want = [step(0, b) for b in news]
    buf = (q, k, v)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for x, y in zip(buf, news[0]):
            x.copy_(y)
        first = step(1, buf)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(first, want[0])
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step(1, buf)
    for b, w in zip(news[1:], want[1:]):
        for x, y in zip(buf, b):
            x.copy_(y)
        g.replay()
        assert torch.equal(out, w)
    assert torch.equal(tables_[0].kv_lens, tables_[1].kv_lens)
    assert torch.equal(caches[0].cache, caches[1].cache)


def test_two_graphs_replayed_at_once_do_not_disturb_each_other():
    cache, _ = make(600, 1, 2, 128, 16, 64, seed=9)
    rng = np.random.default_rng(9)
    lens = [5000, 4000]
    table = torch.from_numpy(tables(rng, lens, 600, 16)).to(DEV)
    kv = torch.tensor(lens, dtype=torch.int32, device=DEV)
    graphs = []
    for _ in range(2):
        q = torch.randn(2, 8, 128, device=DEV).bfloat16()
        want = cache.attend(0, q, table, kv)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = cache.attend(0, q, table, kv)
        graphs.append((g, out, want, torch.cuda.Stream(), q))  # q lives as long as its graph
    torch.cuda.synchronize()
    for _ in range(20):
        for g, _, _, s, _ in graphs:
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(out, want) for _, out, want, _, _ in graphs)


def test_refusals_of_the_python_layer():
    cache, _ = make(3, 1, 2, 64, 16, 32, seed=1)
    k = torch.zeros(4, 2, 64, device=DEV).half()
    at = torch.arange(4, device=DEV)
    for bad in (k[:, :1], k[:, :, :32], k[0], k.transpose(1, 2)):
        with pytest.raises(ValueError):
            cache.append(0, bad, bad, at)
    with pytest.raises(ValueError):
        cache.append(0, k, k[:2], at)
    with pytest.raises(ValueError):
        cache.append(0, k, k.float(), at)
    with pytest.raises(TypeError):
        cache.append(0, k.double(), k.double(), at)
    with pytest.raises(TypeError):
        cache.append(0, k, k, at.int())
    with pytest.raises(TypeError):
        cache.append(0, k, k, at.cpu())
    with pytest.raises(ValueError):
        cache.append(0, k, k, at[:3])
    with pytest.raises(cascade_cpp.CascadeError):
        cache.append(1, k, k, at)
    with pytest.raises(TypeError):
        cache.read(0, at, dtype=torch.int8)
    with pytest.raises(ValueError):
        cache.save([0])
    table, lens = torch.zeros(4, 1, dtype=torch.int32, device=DEV), torch.ones(4, dtype=torch.int32, device=DEV)
    q = torch.zeros(4, 6, 64, device=DEV).half()
    for bad in (q[:, :3], q[:, :, :32], q[0], q[:, :0], q[:3]):
        with pytest.raises(ValueError):
            cache.attend(0, bad, table, lens)
    with pytest.raises((TypeError, cascade_cpp.CascadeError)):
        cache.attend(0, q.float(), table, lens)
    with pytest.raises(TypeError):
        cache.attend(0, q, table.long(), lens)
    with pytest.raises(ValueError):
        cache.attend(0, q, table[:, :0], lens)
    with pytest.raises(ValueError):
        cache.attend(0, q, table, lens, q_start=torch.zeros(4, dtype=torch.int32, device=DEV))
    with pytest.raises(ValueError):
        cache.attend(0, q, table, lens, out=q)
    with pytest.raises(ValueError):
        cache.attend(0, q, table, lens, out=torch.empty_like(q).float())
    odd = torch.empty(q.numel() + 1, dtype=q.dtype, device=DEV)[1:].view_as(q)
    with pytest.raises(ValueError):
        cache.attend(0, q, table, lens, out=odd)
    with pytest.raises(ValueError):
        cache.attend(0, q.clone().requires_grad_(), table, lens)
    with pytest.raises(cascade_cpp.CascadeError):
        cache.attend(-1, q, table, lens)
    with pytest.raises(ValueError):
        kv4.KV4Cache.over(cache.cache, head_dim=64, group=64)
    t = kv4.PageTable(4, 2, 3, device=DEV)
    with pytest.raises(TypeError):
        t.plan(lens.long(), 4)
    with pytest.raises(ValueError):
        t.plan(lens[:3], 4)
    with pytest.raises(ValueError):
        t.plan(lens, -1)
    with pytest.raises(TypeError):
        t.plan(lens, 4, done=lens)


def test_a_workspace_that_is_too_small_is_refused():
    cache, _ = make(40, 1, 1, 128, 16, 64, seed=1)
    table = torch.arange(40, dtype=torch.int32, device=DEV).view(1, 40)
    lens = torch.tensor([600], dtype=torch.int32, device=DEV)
    q = torch.zeros(1, 4, 128, device=DEV).half()
    out = torch.empty_like(q)
    a = L.cb_kv4_attend_args(q.data_ptr(), out.data_ptr(), None, table.data_ptr(), lens.data_ptr(), None, None, 0, 40,
                             512, 128, 0.1, 0, L.CB_KV4_F16, 1, 40, 1, 4, 1, 1, 0)
    lib = cascade_cpp._native_lib()
    need = lib.cb_kv4_attend_workspace(cache._form, a)
    if not need:
        pytest.skip("this form needs no workspace")
    work = torch.empty(need, dtype=torch.uint8, device=DEV)
    for ptr, size in ((None, need), (work.data_ptr(), need - 1), (work.data_ptr() + 8, need)):
        a.workspace, a.workspace_bytes = ptr, size
        assert lib.cb_kv4_attend(cache._form, a, C.c_void_p(0)) == L.CB_ERR_ARG
