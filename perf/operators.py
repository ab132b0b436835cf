"""The paged key/value cache's operators, as a serving loop calls them.

Three families:

* ``reserve``  block tables and slot maps from the requests' lengths: every request grows or
  shrinks by a number of tokens, pages come from and go back to a stack of free ones.  A pass
  is a step and its exact inverse (a server that rewinds, or finishes and admits again), so
  the state after it is the state before it;
* ``append``   new tokens' fused q|k|v rows: QK-RMSNorm, RoPE, the queries out, keys and values
  into the pages by slot;
* ``attend``   attention of one new token per request over its pages.

``run`` computes them in elementary torch operations, 32-bit, or with ``own`` set through
``syrinx_amd.paged``.  ``exact`` states each one again in 64 bits (or integers).
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEV = "cuda:0"
F64 = torch.float64
DTYPE = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
EPS = 1e-6
THETA = 1e6


# ---- the cases ------------------------------------------------------------------------

def listed():
    return [
        # one token for each of the decode engine's 16 streams: latency alone
        _reserve("reserve_step_16", 16, 64, 2048, "step", 0, 0),
        # a busy server's step: prompts admitted, finished requests dropped, the rest one token
        _reserve("reserve_mixed_512", 512, 16, 4096, "mixed", 16, 2000),
        # the same over thousands of requests, hundreds of thousands of new tokens
        _reserve("reserve_mixed_4096", 4096, 32, 8192, "mixed", 32, 1500),
        # one token of eight CosyVoice2 utterances (f32, rotate-half, no norm)
        _append("append_cv2_step_8", 8, 8, 8, 14, 2, 64, 16, "f32", "f32", False, False),
        # ragged Fish prompts of three requests, f32 activations into 16-bit pages
        _append("append_fish_prompt_1412", 1412, 1412, 3, 32, 8, 128, 64, "f32", "bf16", True, True),
        # an odd head width, a map longer than its tokens
        _append("append_f16_333", 333, 350, 7, 12, 3, 80, 32, "f16", "f16", True, False),
        # many prompts at once, all 16-bit
        _append("append_bf16_8192", 8192, 8192, 8, 32, 8, 128, 32, "bf16", "bf16", True, True),
        # one CosyVoice2 utterance: latency
        _attend("attend_cv2_1", "500", 0, 14, 2, 64, 16, "f32", "f32"),
        # 16 concurrent Fish streams with ragged caches, f32 queries over 16-bit pages
        _attend("attend_fish_16", "1203,414,1845,980,256,1677,733,2040,1390,577,1121,1958,301,861,1544,1099", 0, 32, 8,
                128, 64, "f32", "bf16"),
        # requests of no token, one token and sizes beside a page's, an idle row, an odd width
        _attend("attend_f16_edges", "0,1,33,4097,777,32", 1, 20, 4, 96, 32, "f16", "f16"),
        # one request over a very long cache: the split over its length carries it
        _attend("attend_long_131071", "131071", 0, 32, 8, 128, 16, "bf16", "bf16"),
        # a full batch of long requests: bandwidth
        _attend("attend_64_long", "spread:64:1000:16384", 0, 32, 8, 128, 32, "bf16", "bf16"),
    ]


def _reserve(name, n, page, max_len, mode, lo, hi):
    return {"name": name, "family": "reserve", "n": n, "page": page, "max_len": max_len, "mode": mode, "lo": lo, "hi": hi}


def _append(name, tokens, cap, requests, nh, nkv, hd, page, dtype, cache, norm, interleaved):
    return {"name": name, "family": "append", "tokens": tokens, "cap": cap, "requests": requests, "nh": nh, "nkv": nkv,
            "hd": hd, "page": page, "dtype": dtype, "cache": cache, "norm": norm, "interleaved": interleaved}


def _attend(name, lens, idle, nh, nkv, hd, page, dtype, cache):
    return {"name": name, "family": "attend", "lens": lens, "idle": idle, "nh": nh, "nkv": nkv, "hd": hd, "page": page,
            "dtype": dtype, "cache": cache}


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    family = rng.choice(["reserve", "append", "append", "attend", "attend", "attend"])
    page = rng.choice([16, 32, 64, 128])
    if family == "reserve":
        n, hi = _log(rng, 1, 4096), _log(rng, 32, 1500)
        case = _reserve("", n, page, _log(rng, 1600, 8192), rng.choice(["step", "mixed", "mixed"]), rng.randint(1, 32), hi)
    else:
        hd = rng.choice([64, 64, 80, 96, 128, 128, 256])
        nkv, group = rng.randint(1, 8), rng.choice([1, 2, 4, 5, 7, 8, 16])
        nh = nkv * group
        dtype, cache = rng.choice([("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16"), ("bf16", "bf16"), ("f16", "f16")])
        if family == "append":
            top = min(8192, 8192 * 48 * 128 // ((nh + 2 * nkv) * hd) // 2)
            tokens = _log(rng, 1, top)
            requests = rng.randint(1, min(tokens, 16)) if rng.random() < 0.7 else min(tokens, 256)
            cap = tokens + rng.choice([0, 0, rng.randint(1, 40)])
            case = _append("", tokens, cap, requests, nh, nkv, hd, page, dtype, cache, rng.random() < 0.5,
                           rng.random() < 0.5)
        else:
            n = _log(rng, 1, 256)
            # at most half of the positions and heads of the largest listed case
            top = 16384 * 8 * 128 * 8 // (nkv * hd * (SIZE[cache] // 2) * max(1, group // 4))
            hi = _log(rng, 32, max(33, min(131072, top // n)))
            if n <= 4:
                lens = ",".join(str(_log(rng, 1, hi)) for _ in range(n))
            else:
                lens = f"spread:{n}:{_log(rng, 1, hi)}:{hi}"
            case = _attend("", lens, rng.choice([0, 0, rng.randint(1, 3)]), nh, nkv, hd, page, dtype, cache)
    del case["name"]
    return case


def _spread(n, lo, hi):
    """n lengths between lo and hi, even over their logarithm, in a mixed order."""
    return [int(round(lo * (hi / lo) ** ((i * 0.6180339887498949) % 1.0))) for i in range(n)]


def _lens(case):
    if case["lens"].startswith("spread:"):
        return _spread(*(int(v) for v in case["lens"].split(":")[1:]))
    return [int(v) for v in case["lens"].split(",")]


# ---- seeded data ----------------------------------------------------------------------

def _gen(seed, path):
    return torch.Generator(device=DEV).manual_seed((seed * 1000003 + path) & 0x7FFFFFFFFFFF)


def _normal(shape, std, dtype, seed, path):
    return torch.randn(shape, generator=_gen(seed, path), device=DEV, dtype=dtype).mul_(std)


def _i32(values):
    return torch.as_tensor(np.asarray(values, dtype=np.int32)).to(DEV)


def _blocks(x, page):
    return (x + page - 1) // page


def _page_tables(lens, page, width, n_pages, rng):
    """A table of random distinct pages holding the lengths, and the pages left over."""
    order = rng.permutation(n_pages).astype(np.int32)
    table, at = np.full((len(lens), width), -1, np.int32), 0
    for i, n in enumerate(lens):
        b = _blocks(int(n), page)
        table[i, :b] = order[at:at + b]
        at += b
    return table, order[at:]


def _reserve_plan(case, seed):
    """lens, the tokens each request grows (or shrinks) by, and the inverse; the seed decides
    which of the requests that do the same holds which length."""
    rng, n, top = np.random.default_rng(seed), case["n"], case["max_len"]
    lens, add = np.asarray(_spread(n, 1, top - 1)), np.ones(n, np.int64)
    if case["mode"] == "step":
        kind = (np.arange(n) % 10 == 5).astype(int)
        add[kind == 1] = 0
    else:
        kind, size = np.arange(n) % 4, np.minimum(_spread(n, case["lo"], case["hi"]), top - 1)
        lens[kind == 1], add[kind == 1] = 0, size[kind == 1]
        lens[kind == 3], add[kind == 3] = size[kind == 3], -size[kind == 3]
    for group in range(4):
        at, mix = np.flatnonzero(kind == group), rng.permutation(int((kind == group).sum()))
        lens[at], add[at] = lens[at][mix], add[at][mix]
    return lens, add, -add


def _reserve_caps(case):
    _, add, back = _reserve_plan(case, 0)
    return int(add[add > 0].sum()), int(back[back > 0].sum())


def prepare(case, seed):
    st, page = dict(case), case["page"]
    if case["family"] == "reserve":
        lens, add, back = _reserve_plan(case, seed)
        width = _blocks(case["max_len"], page)
        used = int(_blocks(lens, page).sum())
        n_pages = used + int(_blocks(np.maximum(lens + add, 0), page).sum()) + 7
        table, free = _page_tables(lens, page, width, n_pages, np.random.default_rng(seed + 1))
        stack = np.full(n_pages, -1, np.int32)
        stack[:len(free)] = free
        st.update(add=_i32(add), back=_i32(back), lens=_i32(lens), table=_i32(table), free=_i32(stack),
                  free_count=_i32([len(free)]), caps=_reserve_caps(case))
        if own:
            cache = _cache(1, 64, n_pages, page, case["n"], case["max_len"], torch.bfloat16)
            for name in ("lens", "table", "free", "free_count"):
                getattr(cache, name).copy_(st[name])
                st[name] = getattr(cache, name)
            st["kv"] = cache
        return st
    nkv, hd, dt, cdt = case["nkv"], case["hd"], DTYPE[case["dtype"]], DTYPE[case["cache"]]
    rng = np.random.default_rng(seed)
    if case["family"] == "append":
        each = [case["tokens"] // case["requests"] + (i < case["tokens"] % case["requests"])
                for i in range(case["requests"])]
        start = rng.integers(0, 1000, case["requests"])
        lens, most = start + each, 1000 + np.asarray(each)
    else:
        lens = most = np.asarray(_lens(case))
    max_len = max(1, int(most.max()))
    n_pages = int(_blocks(most, page).sum()) + 3
    table, _ = _page_tables(lens, page, _blocks(max_len, page), n_pages, rng)
    shape = (n_pages, nkv, page, hd)
    st.update(k=_normal(shape, 1.0, cdt, seed, 1), v=_normal(shape, 1.0, cdt, seed, 2), lens=_i32(lens), table=_i32(table))
    if case["family"] == "append":
        row = np.repeat(np.arange(case["requests"]), each)
        pos = np.concatenate([np.arange(s, s + e) for s, e in zip(start, each)])
        slot = table[row, pos // page].astype(np.int64) * page + pos % page
        pad = np.full(case["cap"] - case["tokens"], -1)
        ang = np.arange(max_len)[:, None] * THETA ** (-2.0 * np.arange(hd // 2) / hd)
        st.update(rows=_i32(np.concatenate([row, pad])), pos=_i32(np.concatenate([pos, pad])),
                  slots=_i32(np.concatenate([slot, pad])),
                  cos=torch.as_tensor(np.cos(ang).astype(np.float32)).to(DEV),
                  sin=torch.as_tensor(np.sin(ang).astype(np.float32)).to(DEV),
                  qkv=_normal((case["cap"], (case["nh"] + 2 * nkv) * hd), 1.5, dt, seed, 3),
                  out=torch.zeros((case["cap"], case["nh"] * hd), dtype=dt, device=DEV))
        st["q_norm"] = 1.0 + _normal((hd,), 0.1, torch.float32, seed, 4) if case["norm"] else None
        st["k_norm"] = 1.0 + _normal((hd,), 0.1, torch.float32, seed, 5) if case["norm"] else None
    else:
        n, idle = len(lens), case["idle"]
        st.update(q=_normal((n + idle, case["nh"], hd), 2.0, dt, seed, 3), rows=_i32(list(range(n)) + [-1] * idle),
                  host_lens=[int(v) for v in lens],
                  out=torch.zeros((n + idle, case["nh"], hd), dtype=dt, device=DEV))
    if own:
        cache = _cache(nkv, hd, n_pages, page, len(lens), max_len, cdt)
        cache.k[0].copy_(st["k"])
        cache.v[0].copy_(st["v"])
        cache.lens.copy_(st["lens"])
        cache.table.copy_(st["table"])
        st.update(kv=cache, k=cache.k[0], v=cache.v[0])
        if case["family"] == "append":
            st["map"] = _slot_map(st)
    return st


def _cache(nkv, hd, n_pages, page, rows, max_len, dtype):
    from syrinx_amd.paged import PagedKvCache

    return PagedKvCache(1, nkv, hd, n_pages=n_pages, page_size=page, max_rows=rows, max_len=max_len, dtype=dtype,
                        device=DEV)


def _slot_map(st):
    from syrinx_amd.paged import SlotMap

    return SlotMap(slots=st["slots"], pos=st["pos"], rows=st["rows"])


# ---- the plain forms ------------------------------------------------------------------

def _reserve_plain(st, add, cap):
    page, table, free, count = st["page"], st["table"], st["free"].long(), st["free_count"].long()
    width, a, old = table.shape[1], add.long(), st["lens"].long()
    ob = _blocks(old, page)
    shrink = a < 0
    less, more = (old + a).clamp(min=0), old + a
    lb, mb = _blocks(less, page), _blocks(more, page)
    wide = ~shrink & (more > width * page)
    zero = torch.zeros_like(a)
    need, tok = torch.where(shrink | wide, zero, mb - ob), torch.where(shrink | wide, zero, a)
    freed = torch.where(shrink, ob - lb, zero)
    # pages given back: the first of them on top of the stack
    j = torch.arange(width, device=DEV)[None, :]
    gone = shrink[:, None] & (j >= lb[:, None]) & (j < ob[:, None])
    avail = count + freed.sum()
    rank = (torch.cumsum(freed, 0) - freed)[:, None] + j - lb[:, None]
    at = torch.where(gone, avail - 1 - rank, torch.full_like(rank, free.numel()))
    free = torch.cat([free, free.new_zeros(1)]).scatter_(0, at.reshape(-1), table.long().reshape(-1))[:-1]
    table = torch.where(gone, torch.full_like(table, -1), table)
    # who gets pages and room in the map
    dry = (need > 0) & (torch.cumsum(need, 0) > avail)
    full = (tok > 0) & (torch.cumsum(tok, 0) > cap)
    status = torch.where(wide, 2 + zero, torch.where(dry, 1 + zero, torch.where(full, 3 + zero, zero)))
    ok = ~shrink & (status == 0)
    need, tok = torch.where(ok, need, zero), torch.where(ok, tok, zero)
    fresh = ok[:, None] & (j >= ob[:, None]) & (j < mb[:, None])
    rank = (torch.cumsum(need, 0) - need)[:, None] + j - ob[:, None]
    pages = free[torch.where(fresh, avail - 1 - rank, torch.zeros_like(rank))]
    table = torch.where(fresh, pages.to(torch.int32), table)
    cu = torch.cat([zero[:1], torch.cumsum(tok, 0)])
    t = torch.arange(cap, device=DEV)
    row = torch.searchsorted(cu[1:].contiguous(), t, right=True).clamp(max=a.numel() - 1)
    live = t < cu[-1]
    pos = old[row] + t - cu[row]
    slot = table[row, (pos // page).clamp(0, width - 1)].long() * page + pos % page
    out = [torch.where(live, v, torch.full_like(t, -1)).to(torch.int32) for v in (slot, pos, row)]
    st["table"].copy_(table)
    st["free"].copy_(free)
    st["free_count"].copy_(avail - need.sum())
    st["lens"].copy_(torch.where(shrink, less, torch.where(ok, more, old)))
    return [cu.to(torch.int32), *out, status.to(torch.int32)]


def _rotate(x, c, s, interleaved):
    if interleaved:
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
    a, b = x.chunk(2, -1)
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def _append_plain(st):
    nh, nkv, hd, page = st["nh"], st["nkv"], st["hd"], st["page"]
    x = st["qkv"].float().view(-1, nh + 2 * nkv, hd)
    q, k, v = x.split([nh, nkv, nkv], 1)
    if st["norm"]:
        q = q / torch.sqrt((q * q).mean(-1, keepdim=True) + EPS) * st["q_norm"]
        k = k / torch.sqrt((k * k).mean(-1, keepdim=True) + EPS) * st["k_norm"]
    at = st["pos"].long().clamp(min=0)
    c, s = st["cos"][at][:, None], st["sin"][at][:, None]
    q, k = _rotate(q, c, s, st["interleaved"]), _rotate(k, c, s, st["interleaved"])
    tokens = st["tokens"]  # the map's tokens come first; a user's program knows their number
    slot = st["slots"][:tokens].long()
    st["k"][slot // page, :, slot % page] = k[:tokens].to(st["k"].dtype)
    st["v"][slot // page, :, slot % page] = v[:tokens].to(st["v"].dtype)
    st["out"][:tokens] = q[:tokens].reshape(tokens, -1).to(st["out"].dtype)
    return [st["out"], st["k"], st["v"]]


def _attend_plain(st):
    nh, nkv, hd, page, lens = st["nh"], st["nkv"], st["hd"], st["page"], st["host_lens"]
    scale, at = 1.0 / math.sqrt(hd), 0
    while at < len(lens):  # batches of requests whose padded keys stay within a gigabyte
        end, top = at, 1
        while end < len(lens) and (end == at or (end + 1 - at) * max(top, lens[end]) * nkv * hd <= 1 << 28):
            top, end = max(top, lens[end]), end + 1
        m, nb = end - at, _blocks(top, page)
        rows = st["rows"][at:end].long()
        pages = st["table"][rows, :nb].long().clamp(min=0)
        k = st["k"][pages].float().permute(0, 2, 4, 1, 3).reshape(m, nkv, hd, nb * page)
        v = st["v"][pages].float().permute(0, 2, 1, 3, 4).reshape(m, nkv, nb * page, hd)
        s = torch.matmul(st["q"][at:end].float().view(m, nkv, nh // nkv, hd), k) * scale
        gone = torch.arange(nb * page, device=DEV)[None, :] >= st["lens"][rows][:, None]
        s = s.masked_fill(gone[:, None, None, :], -math.inf)
        top_s = s.amax(-1, keepdim=True)
        p = torch.exp(s - torch.where(torch.isinf(top_s), torch.zeros_like(top_s), top_s))
        total = p.sum(-1, keepdim=True)
        o = torch.matmul(p, v) / torch.where(total == 0, torch.ones_like(total), total)
        st["out"][at:end] = o.view(m, nh, hd).to(st["out"].dtype)
        at = end
    return [st["out"]]


def run(st):
    if st["family"] == "reserve":
        if own:
            a = st["kv"].reserve(st["add"], st["caps"][0])
            b = st["kv"].reserve(st["back"], st["caps"][1])
            maps = [[m.cu, m.slots, m.pos, m.rows, m.status] for m in (a, b)]
        else:
            maps = [_reserve_plain(st, st["add"], st["caps"][0]), _reserve_plain(st, st["back"], st["caps"][1])]
        return [*maps[0], *maps[1], st["lens"], st["table"], st["free"], st["free_count"]]
    if st["family"] == "append":
        if not own:
            return _append_plain(st)
        st["kv"].append(0, st["qkv"], st["map"], n_heads=st["nh"], q_norm=st["q_norm"], k_norm=st["k_norm"], eps=EPS,
                        rope=(st["cos"], st["sin"]), interleaved=st["interleaved"], out=st["out"])
        return [st["out"], st["k"], st["v"]]
    if not own:
        return _attend_plain(st)
    return [st["kv"].attend(0, st["q"], rows=st["rows"], out=st["out"])]


# ---- what a pass cannot do without ----------------------------------------------------

def work(case):
    page = case["page"]
    if case["family"] == "reserve":
        lens, add, _ = _reserve_plan(case, 0)
        moved = np.abs(_blocks(np.maximum(lens + add, 0), page) - _blocks(lens, page)).sum()
        # both calls: lengths and growth in, lengths, offsets and status out; the pages moved,
        # read once and written once; three words a token
        return {"bytes": int(2 * (20 * case["n"] + 8 * moved) + 12 * sum(_reserve_caps(case))), "flops": 0}
    nh, nkv, hd, e, ce = case["nh"], case["nkv"], case["hd"], SIZE[case["dtype"]], SIZE[case["cache"]]
    if case["family"] == "append":
        t = case["tokens"]
        heads = nh + nkv
        return {"bytes": t * ((nh + 2 * nkv) * hd * e + nh * hd * e + 2 * nkv * hd * ce + 4 * hd + 8),
                "flops": t * heads * hd * (3 + (4 if case["norm"] else 0))}
    lens = _lens(case)
    return {"bytes": sum(lens) * 2 * nkv * hd * ce + 2 * len(lens) * nh * hd * e
            + sum(4 * _blocks(n, page) for n in lens) + 8 * len(lens),
            "flops": 4 * sum(lens) * nh * hd}


# ---- the definitions, in 64 bits ------------------------------------------------------

def _reserve_exact(lens, table, free, count, add, cap, page):
    """One call, request by request, on numpy arrays that it updates."""
    n, width = table.shape
    status, tokens = np.zeros(n, np.int64), []
    back = []
    for i in np.flatnonzero(add < 0):
        new = max(0, int(lens[i] + add[i]))
        a, b = -(-new // page), -(-int(lens[i]) // page)
        back.extend(table[i, a:b].tolist())
        table[i, a:b] = -1
        lens[i] = new
    free[count:count + len(back)] = back[::-1]
    count += len(back)
    avail, asked, room = count, 0, 0
    cu = [0]
    for i in range(n):
        grow = int(add[i])
        if grow >= 0:
            new, have = int(lens[i]) + grow, -(-int(lens[i]) // page)
            if new > width * page:
                status[i] = 2
            else:
                need = -(-new // page) - have
                asked, room = asked + need, room + grow
                if need and asked > avail:
                    status[i] = 1
                elif grow and room > cap:
                    status[i] = 3
                else:
                    table[i, have:have + need] = free[count - need:count][::-1]
                    count -= need
                    p = np.arange(lens[i], new)
                    tokens.append(np.stack([table[i, p // page].astype(np.int64) * page + p % page, p, np.full_like(p, i)]))
                    lens[i] = new
                    cu.append(cu[-1] + grow)
                    continue
        cu.append(cu[-1])
    out = np.full((3, cap), -1, np.int64)
    out[:, :cu[-1]] = np.concatenate([np.zeros((3, 0), np.int64), *tokens], 1)
    return count, [_i32(v) for v in (cu, *out, status)]


def _pages64(pool, table_row, n, page):
    t = table_row[:_blocks(n, page)].long()
    return pool[t].to(F64).transpose(0, 1).reshape(pool.shape[1], -1, pool.shape[3])[:, :n]


def exact(case, seed):
    st = _plain_state(case, seed)
    page = case["page"]
    if case["family"] == "reserve":
        lens, table, free = (st[k].cpu().numpy().astype(np.int64) for k in ("lens", "table", "free"))
        count, maps = int(st["free_count"].item()), []
        for add, cap in ((st["add"], st["caps"][0]), (st["back"], st["caps"][1])):
            count, m = _reserve_exact(lens, table, free, count, add.cpu().numpy().astype(np.int64), cap, page)
            maps += m
        return [*maps, _i32(lens), _i32(table), _i32(free), _i32([count])]
    nh, nkv, hd = case["nh"], case["nkv"], case["hd"]
    if case["family"] == "append":
        n = case["tokens"]
        heads = st["qkv"][:n].to(F64).view(n, nh + 2 * nkv, hd)
        if case["norm"]:
            rms = torch.rsqrt(heads.square().mean(-1, keepdim=True) + EPS)
            w = torch.cat([st["q_norm"].to(F64).expand(nh, hd), st["k_norm"].to(F64).expand(nkv, hd)])
            heads = torch.cat([heads[:, :nh + nkv] * rms[:, :nh + nkv] * w, heads[:, nh + nkv:]], 1)
        # the rotation as a complex product
        turn = torch.complex(st["cos"].to(F64), st["sin"].to(F64))[st["pos"][:n].long()][:, None]
        rot = heads[:, :nh + nkv]
        if case["interleaved"]:
            z = torch.complex(rot[..., 0::2].contiguous(), rot[..., 1::2].contiguous()) * turn
            rot = torch.view_as_real(z).reshape(n, nh + nkv, hd)
        else:
            z = torch.complex(rot[..., :hd // 2].contiguous(), rot[..., hd // 2:].contiguous()) * turn
            rot = torch.cat([z.real, z.imag], -1)
        out, k, v = st["out"].to(F64), st["k"].to(F64), st["v"].to(F64)
        out[:n] = rot[:, :nh].reshape(n, -1)
        flat = (st["slots"][:n].long() // page, slice(None), st["slots"][:n].long() % page)
        k[flat], v[flat] = rot[:, nh:], heads[:, nh + nkv:]
        return [out, k, v]
    out = st["out"].to(F64)
    for i, n in enumerate(_lens(case)):
        if n == 0:
            out[i] = 0
            continue
        k, v = (_pages64(st[name], st["table"][i], n, page) for name in ("k", "v"))
        q = st["q"][i].to(F64).view(nkv, nh // nkv, hd)
        for h in range(nkv):
            p = torch.softmax((q[h] @ k[h].t().contiguous()) / math.sqrt(hd), -1)
            out[i, h * (nh // nkv):(h + 1) * (nh // nkv)] = p @ v[h]
    return [out]


def _plain_state(case, seed):
    """The inputs alone, as ``prepare`` makes them, without a cache object."""
    global own
    kept, own = own, False
    try:
        return prepare(case, seed)
    finally:
        own = kept
