"""Cases and plain forms of the operators on a paged KV cache held in 4 bits.

Four operators that a serving program runs one after another:

* ``plan``: the page table. Finished requests give their pages back, the new
  tokens of every request get pages, slots and positions;
* ``append``: new keys and values are quantised into the pages at their slots,
  and read back as the values that the pages now stand for;
* ``read``: tokens of the cache as dense 16-bit keys and values;
* ``attend``: attention of the new tokens' queries over the cached ones.

Format of a page (one per layer and KV head): tiles of 16 tokens, each

    K codes 8*D bytes | V codes 8*D | K params 64*D/group | V params 64*D/group

with two fp16 numbers (scale, offset) per token and group of ``group``
dimensions, and x = offset + scale * (code - 8). Dimensions are split into
slabs of SD = min(D, 128). A K code (token, slab, dim 32 i + 8 t + 2 k + h) is
nibble 4 h + k of the 32-bit word ((slab*16 + token)*4 + t)*(SD/32) + i; a V
code (token 8 p + 2 t + b, slab, dim 32 j + 8 k + g) is nibble k of the 16-bit
word ((((slab*2 + p)*8 + g)*4 + t)*(SD/32) + j)*2 + b.
"""
import math
import os
import random
import sys

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ------------------------------------------------------------------ the cases

def _attend(name, q_heads, kv_heads, dim, group, page, dtype, requests, len_lo, len_hi, q_lo, q_hi, layers=1,
            lse=False):
    return {"name": name, "op": "attend", "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim, "group": group,
            "page": page, "dtype": dtype, "requests": requests, "len_lo": len_lo, "len_hi": len_hi, "q_lo": q_lo,
            "q_hi": q_hi, "layers": layers, "lse": lse}


def _tokens(name, op, heads, dim, group, page, dtype, tokens, layers=2):
    return {"name": name, "op": op, "kv_heads": heads, "dim": dim, "group": group, "page": page, "dtype": dtype,
            "tokens": tokens, "layers": layers}


def _plan(name, requests, len_lo, len_hi, q_lo, q_hi, page, restart):
    return {"name": name, "op": "plan", "requests": requests, "len_lo": len_lo, "len_hi": len_hi, "q_lo": q_lo,
            "q_hi": q_hi, "page": page, "restart": restart}


def listed():
    return [
        # one decode step of a small batch: one new token for each request
        _plan("plan decode 48", 48, 20, 6000, 1, 1, 16, False),
        # a busy step: most rows have finished and start anew with prompts of all lengths
        _plan("plan restart 700", 700, 5, 2500, 0, 700, 16, True),
        # the new tokens of a decode step (Qwen2.5-7B heads)
        _tokens("append decode 37", "append", 4, 128, 128, 16, "bf16", 37),
        # a prompt chunk (Qwen2.5-72B heads), fine groups
        _tokens("append prompt 8191", "append", 8, 128, 32, 16, "bf16", 8191),
        # a short prefix handed to an engine with a 16-bit cache
        _tokens("read prefix 333", "read", 4, 128, 64, 32, "fp16", 333),
        # a long document's prefix
        _tokens("read document 40000", "read", 8, 128, 128, 16, "bf16", 40000, layers=1),
        # one user, a short chat: latency
        _attend("decode one user", 28, 4, 128, 128, 16, "bf16", 1, 1100, 1100, 1, 1, layers=2, lse=True),
        # an ordinary batch, ragged lengths (Qwen2.5-7B heads)
        _attend("decode ragged 61", 28, 4, 128, 64, 16, "fp16", 61, 90, 8000, 1, 1, lse=True),
        # long contexts (Qwen2.5-72B heads): the largest cache
        _attend("decode long 48", 64, 8, 128, 128, 32, "bf16", 48, 9000, 32000, 1, 1),
        # a small model's heads, small groups
        _attend("decode D64 130", 32, 8, 64, 32, 64, "bf16", 130, 1, 3000, 1, 1, layers=2, lse=True),
        # drafted tokens checked in one step: a few query tokens each
        _attend("drafts 24", 64, 8, 128, 128, 16, "bf16", 24, 200, 7000, 2, 5),
        # prompt chunks behind cached prefixes loaded from the store
        _attend("prompt chunk 2", 64, 8, 128, 128, 16, "bf16", 2, 5200, 9100, 900, 1537),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["plan", "append", "read", "decode", "decode", "drafts", "prompt"])
    dim = rng.choice([64, 128, 128, 256])
    group = rng.choice([g for g in (32, 64, 128, 256) if g <= dim])
    page = rng.choice([16, 16, 32, 64])
    dtype = rng.choice(["bf16", "fp16"])
    heads = rng.choice([1, 2, 4, 5, 8])
    if kind == "plan":
        restart = rng.random() < 0.5
        hi = _log(rng, 2, 600) if restart else rng.choice([1, 1, 4])
        c = _plan("", _log(rng, 1, 700), 1, _log(rng, 8, 2400), 0 if restart else 1, hi, page, restart)
    elif kind in ("append", "read"):
        most = (8191 if kind == "append" else 40000) * 8 * 128 // (8 * 256)
        c = _tokens("", kind, heads, dim, group, page, dtype, _log(rng, 1, most), rng.choice([1, 2]))
    elif kind == "prompt":
        c = _attend("", heads * rng.choice([1, 4, 7]), heads, min(dim, 128), min(group, 64), page, dtype,
                    rng.choice([1, 2, 3]), 300, _log(rng, 900, 6000), _log(rng, 17, 200), _log(rng, 201, 900))
    else:
        ratio = rng.choice([1, 3, 7, 8, 16])
        requests = _log(rng, 1, 60)
        top = min(30000, 700000 // requests // max(1, dim // 128))
        hi = _log(rng, 40, top)
        q = (1, 1) if kind == "decode" else (1, rng.choice([2, 4, 6]))
        c = _attend("", heads * ratio, heads, dim, group, page, dtype, requests, rng.choice([1, 17, max(1, hi // 3)]),
                    hi, q[0], q[1], rng.choice([1, 2]))
    c.pop("name")
    return c


def _lens(case):
    """(cached length with the new tokens, new tokens) of each request: the
    same pairs whatever the seed, which only orders them."""
    n = case["requests"]
    r = random.Random(n * 1000003 + case["len_hi"] * 101 + case["q_hi"])
    q = [r.randint(case["q_lo"], case["q_hi"]) for _ in range(n)]
    total = [case["len_lo"] + (case["len_hi"] - case["len_lo"]) * i // max(1, n - 1) for i in range(n)]
    if n == 1:
        total = [case["len_hi"]]
    r.shuffle(total)
    if case["op"] == "attend":
        q = [min(a, b) for a, b in zip(q, total)]
    return total, q


def work(case):
    op = case["op"]
    if op == "plan":
        total, q = _lens(case)
        ps, new = case["page"], sum(q)
        if case["restart"]:
            moved = sum(-(-n // ps) for n in q)  # pages given back and taken again
            pages = 2 * moved
        else:
            pages = sum(-(-(a + b) // ps) - -(-a // ps) for a, b in zip(total, q))
        return {"bytes": 12 * new + 8 * pages + 28 * len(q), "flops": 0}
    h, d = case["kv_heads"], case["dim"]
    held = h * (d + 8 * (d // case["group"]))  # bytes of one cached token
    if op == "append":  # values in, pages out; pages in, values out
        n = case["tokens"]
        return {"bytes": n * (2 * 4 * h * d + 2 * held + 16), "flops": 0}
    if op == "read":
        n = case["tokens"]
        return {"bytes": n * (4 * h * d + held + 8), "flops": 0}
    total, q = _lens(case)
    pairs = sum(b * a - b * (b - 1) // 2 for a, b in zip(total, q))
    return {"bytes": sum(total) * held + 4 * sum(q) * case["q_heads"] * d, "flops": 4 * pairs * case["q_heads"] * d}


# ---------------------------------------------------------- the format, plain

def _tile_bytes(dim, group):
    return 16 * dim + 128 * (dim // group)


def _views(pages, dim, group, page):
    """K codes, V codes, K params and V params of ``pages``, as views."""
    lay, h = pages.shape[1:3]
    tiles = pages.view(-1, lay, h, page // 16, _tile_bytes(dim, group))
    sd = min(dim, 128)
    par = 64 * (dim // group)
    k = tiles[..., :8 * dim].unflatten(-1, (dim // sd, 16, sd // 2))
    v = tiles[..., 8 * dim:16 * dim].unflatten(-1, (dim // sd, 2, 8, 4, sd // 32, 2, 2))
    kp = tiles[..., 16 * dim:16 * dim + par].unflatten(-1, (16, par // 16))
    vp = tiles[..., 16 * dim + par:].unflatten(-1, (16, par // 16))
    return k, v, kp, vp


def _quantise(x, group):
    """Codes (int32) and parameters (fp16 pairs) of [n, heads, dim] values."""
    x = x.float().clamp(-65000.0, 65000.0).unflatten(-1, (-1, group))
    low, high = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    scale = ((high - low) / 15.0).half()
    offset = (low + 8.0 * scale.float()).half()
    s = scale.float()
    step = torch.where(s > 0, 1.0 / s, torch.zeros_like(s))
    code = torch.round((x - offset.float()) * step).clamp(-8.0, 7.0) + 8.0
    return code.to(torch.int32).flatten(-2), torch.cat([scale, offset], -1).flatten(-2)


def _bytes_k(code, sd):
    c = code.unflatten(-1, (-1, sd // 32, 4, 4, 2))  # slab, i, t, k, h
    c = c.movedim(-3, -4)                             # slab, t, i, k, h
    c = c.transpose(-1, -2).flatten(-2)               # slab, t, i, nibble
    return (c[..., 0::2] | c[..., 1::2] << 4).to(torch.uint8).flatten(-3)


def _bytes_v(code, sd):
    c = code.unflatten(-1, (-1, sd // 32, 4, 8))      # slab, j, k, g
    c = c.permute(*range(c.dim() - 3), -1, -3, -2)    # slab, g, j, k
    return (c[..., 0::2] | c[..., 1::2] << 4).to(torch.uint8)


def _place(slots, page):
    p, t = slots // page, slots % page
    return p, t // 16, t % 16


def _write(pages, layer, k, v, slots, dim, group, page):
    keep = slots >= 0
    p, tile, tok = _place(slots[keep], page)
    sd = min(dim, 128)
    vk, vv, vkp, vvp = _views(pages, dim, group, page)
    kc, kp = _quantise(k[keep], group)
    vc, vp = _quantise(v[keep], group)
    vk[p, layer, :, tile, :, tok] = _bytes_k(kc, sd)
    vv[p, layer, :, tile, :, tok // 8, :, tok % 8 // 2, :, tok % 2] = _bytes_v(vc, sd)
    vkp[p, layer, :, tile, tok] = kp.view(torch.uint8)
    vvp[p, layer, :, tile, tok] = vp.view(torch.uint8)


def _nibbles(b):
    return torch.stack([b & 15, b >> 4], -1).flatten(-2)


def _dequantise(code, par, group):
    par = par.contiguous().view(torch.float16).float().unflatten(-1, (-1, 2))
    x = code.float().unflatten(-1, (-1, group))
    return (par[..., 1:] + par[..., :1] * (x - 8.0)).flatten(-2)


def _read(pages, layer, slots, dim, group, page):
    """K and V of ``slots`` in 32 bits: [n, heads, dim]."""
    p, tile, tok = _place(slots.clamp(min=0), page)
    sd = min(dim, 128)
    vk, vv, vkp, vvp = _views(pages, dim, group, page)
    kc = _nibbles(vk[p, layer, :, tile, :, tok]).unflatten(-1, (4, sd // 32, 2, 4))  # t, i, h, k
    kc = kc.permute(*range(kc.dim() - 4), -3, -4, -1, -2).flatten(-5)
    vc = _nibbles(vv[p, layer, :, tile, :, tok // 8, :, tok % 8 // 2, :, tok % 2])   # slab, g, j, k
    vc = vc.permute(*range(vc.dim() - 3), -2, -1, -3).flatten(-4)
    k = _dequantise(kc, vkp[p, layer, :, tile, tok], group)
    v = _dequantise(vc, vvp[p, layer, :, tile, tok], group)
    none = (slots < 0)[:, None, None]
    return k.masked_fill(none, 0.0), v.masked_fill(none, 0.0)


# ------------------------------------------------------------------ the inputs

def _package():
    at = os.path.join(os.getcwd(), "kcj-cascade-v6_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    from cascade_cpp import kv4
    return kv4


def _values(gen, n, heads, dim, dtype, channel):
    """Keys have a few dimensions of larger spread and their own mean."""
    x = torch.randn(n, heads, dim, generator=gen, device=DEV)
    if channel is not None:
        x = x * channel[0] + channel[1]
    return x.to(DTYPES[dtype])


def _channels(gen, heads, dim):
    wide = torch.where(torch.rand(heads, dim, generator=gen, device=DEV) < 0.04, 4.0, 1.0)
    return wide, torch.randn(heads, dim, generator=gen, device=DEV) * 0.5


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    order = random.Random(seed)
    s = {"case": case}
    if case["op"] == "plan":
        total, q = _lens(case)
        both = list(zip(total, q))
        order.shuffle(both)
        total, q = [a for a, _ in both], [b for _, b in both]
        ps = case["page"]
        cols = -(-(case["len_hi"] + case["q_hi"]) // ps)
        held = [-(-n // ps) for n in total]
        pages = sum(max(a, -(-b // ps)) + 1 for a, b in zip(held, q)) + sum(
            -(-(a + b) // ps) for a, b in zip(total, q))
        ids = torch.randperm(pages, generator=gen, device=DEV, dtype=torch.int64).to(torch.int32)
        table = torch.zeros(len(q), cols, dtype=torch.int32, device=DEV)
        used = torch.arange(cols, device=DEV)[None, :] < torch.tensor(held, device=DEV)[:, None]
        n = sum(held)
        table[used] = ids[:n]
        s |= {"block_table": table, "kv_lens": torch.tensor(total, dtype=torch.int32, device=DEV),
              "q_lens": torch.tensor(q, dtype=torch.int32, device=DEV),
              "free": torch.cat([ids[n:], torch.zeros(n, dtype=torch.int32, device=DEV)]),
              "free_count": torch.tensor([pages - n], dtype=torch.int32, device=DEV),
              "borrowed": torch.zeros(len(q), dtype=torch.int32, device=DEV), "tokens": sum(q) + 3}
        if case["restart"]:  # the rows that start anew have finished
            s["done"] = s["q_lens"] > 0
        if own:  # the program's page table, in the state of the inputs
            kv4 = _package()
            t = kv4.PageTable(len(q), cols, pages, ps, device=DEV)
            for name in ("block_table", "kv_lens", "free", "free_count", "borrowed"):
                getattr(t, name).copy_(s[name])
                s[name] = getattr(t, name)
            s["table"] = t
        return s

    h, d, g, ps, lay = case["kv_heads"], case["dim"], case["group"], case["page"], case["layers"]
    if case["op"] == "attend":
        total, q = _lens(case)
        both = list(zip(total, q))
        order.shuffle(both)
        total, q = [a for a, _ in both], [b for _, b in both]
        cols = max(-(-n // ps) for n in total)
        pages = sum(-(-n // ps) for n in total) + 2
    else:
        pages = -(-case["tokens"] // ps) + 3
    cache = torch.zeros(pages, lay, h, ps // 16 * _tile_bytes(d, g), dtype=torch.uint8, device=DEV)
    layer = lay - 1
    s |= {"pages": cache, "layer": layer}
    ids = torch.randperm(pages, generator=gen, device=DEV)
    chan = _channels(gen, h, d)
    if case["op"] == "attend":
        table = torch.zeros(len(q), cols, dtype=torch.int32, device=DEV)
        used = torch.arange(cols, device=DEV)[None, :] < torch.tensor([-(-n // ps) for n in total], device=DEV)[:, None]
        table[used] = ids[:pages - 2].to(torch.int32)
        start = torch.tensor([0] + q, device=DEV).cumsum(0).to(torch.int32)
        s |= {"block_table": table, "kv_lens": torch.tensor(total, dtype=torch.int32, device=DEV), "q_start": start,
              "max_q": max(q),
              "q": _values(gen, sum(q), case["q_heads"], d, case["dtype"], None)}
    elif case["op"] == "append":
        n = case["tokens"]
        s |= {"k": _values(gen, n, h, d, case["dtype"], chan), "v": _values(gen, n, h, d, case["dtype"], None)}
    if case["op"] != "attend":  # tokens of one request, in order, with a padding slot among many
        n = case["tokens"]
        at = torch.arange(n, device=DEV)
        s["slots"] = ids[at // ps] * ps + at % ps
        if n > 8:
            s["slots"][n - 2] = -1
    if case["op"] != "append":  # every page full of quantised values
        step = max(1, (1 << 25) // (ps * h * d))
        for a in range(0, pages, step):
            b = min(pages, a + step)
            slots = torch.arange(a * ps, b * ps, device=DEV)
            _write(cache, layer, _values(gen, len(slots), h, d, case["dtype"], chan),
                   _values(gen, len(slots), h, d, case["dtype"], None), slots, d, g, ps)
    if own:  # the program's cache over these pages
        s["cache"] = _package().KV4Cache.over(cache, head_dim=d, page_size=ps, group=g)
    return s


# --------------------------------------------------------------------- a pass

def run(s):
    return {"plan": _run_plan, "append": _run_append, "read": _run_read, "attend": _run_attend}[s["case"]["op"]](s)


def _run_plan(s):
    restart = s["case"]["restart"]
    if own:
        p = s["table"].plan(s["q_lens"], s["tokens"], done=s.get("done"), commit=restart)
        return {"slots": p.slots, "positions": p.positions, "q_start": p.q_start, "status": p.status,
                "kv_lens": p.kv_lens, "free_count": p.free_count, "block_table": s["block_table"]}
    ps, table, n = s["case"]["page"], s["block_table"], s["tokens"]
    lens, q, count = s["kv_lens"].long(), s["q_lens"].long(), s["free_count"].long()
    held = (lens + ps - 1) // ps
    col = torch.arange(table.shape[1], device=DEV)
    if restart:
        back = s["done"][:, None] & (col >= s["borrowed"][:, None]) & (col < held[:, None])
        ids = table[back]
        s["free"][count + torch.arange(len(ids), device=DEV)] = ids
        count = count + len(ids)
        lens = torch.where(s["done"], 0, lens)
        held = torch.where(s["done"], 0, held)
    start = torch.cat([torch.zeros_like(q[:1]), q.cumsum(0)])
    fits = (start[1:] <= n) & (lens + q <= table.shape[1] * ps)
    need = torch.where(fits, (lens + q + ps - 1) // ps - held, 0)
    upto = need.cumsum(0)
    ok = fits & ((need == 0) | (upto <= count))
    take = torch.where(ok, need, 0)
    fresh = (col >= held[:, None]) & (col < (held + take)[:, None])
    table[fresh] = s["free"][count - 1 - torch.arange(int(take.sum()), device=DEV)]
    at = torch.arange(n, device=DEV)
    row = torch.searchsorted(start[1:], at, right=True)
    there = row < len(q)
    row = row.clamp(max=len(q) - 1)
    pos = torch.where(there, lens[row] + at - start[row], 0)
    slots = table[row, (pos // ps).clamp(max=table.shape[1] - 1)].long() * ps + pos % ps
    slots = torch.where(there & ok[row], slots, -1)
    after = torch.where(ok, lens + q, lens).to(torch.int32)
    left = (count - take.sum()).to(torch.int32)
    if restart:
        s["kv_lens"].copy_(after)
        s["free_count"].copy_(left)
        s["borrowed"].masked_fill_(s["done"], 0)
    return {"slots": slots, "positions": pos.to(torch.int32), "q_start": start.to(torch.int32),
            "status": torch.where(ok, 0, 2).to(torch.uint8), "kv_lens": after, "free_count": left,
            "block_table": table}


def _run_append(s):
    if own:
        s["cache"].append(s["layer"], s["k"], s["v"], s["slots"])
        return s["cache"].read(s["layer"], s["slots"], dtype=s["k"].dtype)
    c = s["case"]
    form = (c["dim"], c["group"], c["page"])
    _write(s["pages"], s["layer"], s["k"], s["v"], s["slots"], *form)
    k, v = _read(s["pages"], s["layer"], s["slots"], *form)
    return k.to(s["k"].dtype), v.to(s["k"].dtype)


def _run_read(s):
    c = s["case"]
    if own:
        return s["cache"].read(s["layer"], s["slots"], dtype=DTYPES[c["dtype"]])
    k, v = _read(s["pages"], s["layer"], s["slots"], c["dim"], c["group"], c["page"])
    return k.to(DTYPES[c["dtype"]]), v.to(DTYPES[c["dtype"]])


def _run_attend(s):
    c = s["case"]
    if own:
        r = s["cache"].attend(s["layer"], s["q"], s["block_table"], s["kv_lens"], q_start=s["q_start"],
                              max_q=s["max_q"], return_lse=c["lse"])
        return r
    ps, d, h, most = c["page"], c["dim"], c["kv_heads"], s["max_q"]
    table, lens, start, q = s["block_table"].long(), s["kv_lens"].long(), s["q_start"].long(), s["q"]
    rows, ratio = len(table), c["q_heads"] // h
    slots = (table[:, :, None] * ps + torch.arange(ps, device=DEV)).flatten()
    k, v = _read(s["pages"], s["layer"], slots, d, c["group"], ps)
    k = k.view(rows, -1, h, d).permute(0, 2, 3, 1)
    v = v.view(rows, -1, h, d).permute(0, 2, 1, 3)
    count = start[1:] - start[:-1]
    i = torch.arange(most, device=DEV)
    there = i < count[:, None]
    at = (start[:-1, None] + i).clamp(max=len(q) - 1)
    x = q[at].float().view(rows, most, h, ratio, d).permute(0, 2, 1, 3, 4).reshape(rows, h, most * ratio, d)
    score = (x @ k).view(rows, h, most, ratio, -1) * (1.0 / math.sqrt(d))
    seen = torch.arange(score.shape[-1], device=DEV) <= (lens - count)[:, None, None] + i[:, None]
    score.masked_fill_(~(seen & there[:, :, None])[:, None, :, None], float("-inf"))
    top = score.amax(-1, keepdim=True)
    top = torch.where(top == float("-inf"), torch.zeros_like(top), top)
    p = score.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    o = (p.view(rows, h, most * ratio, -1) @ v).view(rows, h, most, ratio, d) / total.clamp(min=1e-30)
    o = o.permute(0, 2, 1, 3, 4).reshape(rows, most, h * ratio, d)[there].to(q.dtype)
    if not c["lse"]:
        return o
    lse = (top + total.log())[..., 0].permute(0, 2, 1, 3).reshape(rows, most, h * ratio)[there]
    return o, lse


# ------------------------------------------------------- the definition, in 64

def _spots(dim, tok):
    """Byte within a tile and shift of every K and V code of one token."""
    sd = min(dim, 128)
    x = torch.arange(dim, device=DEV)
    slab, r = x // sd, x % sd
    word = ((slab * 16 + tok) * 4 + r % 32 // 8) * (sd // 32) + r // 32
    nib = 4 * (r % 2) + r % 8 // 2
    half = ((((slab * 2 + tok // 8) * 8 + r % 8) * 4 + tok % 8 // 2) * (sd // 32) + r // 32) * 2 + tok % 2
    vn = r % 32 // 8
    return word * 4 + nib // 2, nib % 2 * 4, 8 * dim + half * 2 + vn // 2, vn % 2 * 4


def _exact_kv(s, slots):
    c = s["case"]
    d, g, ps = c["dim"], c["group"], c["page"]
    flat, tb = s["pages"].view(-1), _tile_bytes(c["dim"], c["group"])
    head = torch.arange(c["kv_heads"], device=DEV)
    page, tok = slots // ps, slots % ps
    base = ((page[:, None] * c["layers"] + s["layer"]) * c["kv_heads"] + head) * (ps // 16 * tb)
    base = (base + (tok // 16 * tb)[:, None])[..., None]
    kb, ks, vb, vs = _spots(d, (tok % 16)[:, None, None])
    half = flat.view(torch.float16)
    dims = torch.arange(d, device=DEV) // g
    out = []
    for n, (byte, shift) in enumerate(((kb, ks), (vb, vs))):
        code = flat[base + byte] >> shift & 15
        par = (base + 16 * d + n * 64 * (d // g)) // 2 + ((tok % 16)[:, None, None] * (d // g) + dims) * 2
        out.append(half[par + 1].double() + half[par].double() * (code.double() - 8.0))
    return out


def _exact_values(x, slots, group):
    x = x.double().clamp(-65000.0, 65000.0).unflatten(-1, (-1, group))
    low, high = x.min(-1, keepdim=True).values, x.max(-1, keepdim=True).values
    scale = ((high - low) / 15.0).half().double()
    offset = (low + 8.0 * scale).half().double()
    code = torch.where(scale > 0, ((x - offset) / scale).round().clamp(-8.0, 7.0), torch.zeros_like(x))
    return (offset + scale * code).flatten(-2) * (slots >= 0)[:, None, None]


def exact(case, seed):
    if case["op"] == "plan":
        return None
    s = prepare(case, seed)
    if case["op"] == "append":
        return [_exact_values(s[x], s["slots"], case["group"]) for x in ("k", "v")]
    if case["op"] == "read":
        return [x * (s["slots"] >= 0)[:, None, None] for x in _exact_kv(s, s["slots"].clamp(min=0))]
    ps, h, d = case["page"], case["kv_heads"], case["dim"]
    ratio = case["q_heads"] // h
    start, lens = s["q_start"].tolist(), s["kv_lens"].tolist()
    outs, lses = [], []
    for b, n in enumerate(lens):
        t = torch.arange(n, device=DEV)
        k, v = _exact_kv(s, s["block_table"][b].long()[t // ps] * ps + t % ps)
        q = s["q"][start[b]:start[b + 1]].double()
        last = n - len(q) + torch.arange(len(q), device=DEV)
        hidden = (t > last[:, None])[:, None, :]
        o, e = torch.empty_like(q), torch.empty(q.shape[:2], dtype=torch.float64, device=DEV)
        for j in range(h):
            at = slice(j * ratio, (j + 1) * ratio)
            w = (torch.einsum("qrd,td->qrt", q[:, at], k[:, j]) / math.sqrt(d)).masked_fill(hidden, -math.inf)
            e[:, at] = torch.logsumexp(w, -1)
            o[:, at] = torch.einsum("qrt,td->qrd", torch.softmax(w, -1), v[:, j])
        outs.append(o)
        lses.append(e)
    return [torch.cat(outs), torch.cat(lses)] if case["lse"] else torch.cat(outs)
