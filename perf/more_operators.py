"""The paged key/value cache held in 8 bits, as a serving loop calls it: int8 or float8 e4m3 codes
with one scale, a power of two, for every block of 16 positions of a KV head.

Four families:

* ``write``   new tokens' fused q|k|v rows into the cache (QK-RMSNorm, RoPE, quantization; a block
  whose scale grows has its earlier codes rescaled) and the touched blocks read back;
* ``read``    ranges of requests' positions as packed bf16, f16 or f32 keys and values;
* ``attend``  attention of one new token per request;
* ``extend``  attention of several new tokens per request, each over its own prefix.

A block's scale is the smallest power of two 2^e, e >= -100, with max|x| <= Q 2^e (Q: 127, or 448
for e4m3), or the block's earlier scale where that is larger; a block whose first position is
written begins anew.  A code is x / scale, rounded to nearest, ties to even.

``run`` computes them in elementary torch operations, 32-bit, or with ``own`` set through
``syrinx_amd.paged``.  ``exact`` states each one again in 64 bits.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEV = "cuda:0"
F64 = torch.float64
DTYPE = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "i8": torch.int8, "e4m3": torch.float8_e4m3fn}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
TOP = {"i8": 127.0, "e4m3": 448.0}
BLOCK = 16
EPS = 1e-6
THETA = 1e6


# ---- the cases ------------------------------------------------------------------------

def listed():
    return [
        # one token of each of the decode engine's 16 Fish streams: latency
        _write("write_step_16", 16, 16, 32, 8, 128, 32, "f32", "e4m3", True, True),
        # ragged Fish prompts of three requests, f32 activations
        _write("write_fish_prompt_1412", 1412, 3, 32, 8, 128, 64, "f32", "e4m3", True, True),
        # an odd head width and group, short prompts that begin inside a block
        _write("write_f16_333", 333, 7, 12, 3, 80, 32, "f16", "i8", True, False),
        # many prompts at once, 16-bit activations
        _write("write_bf16_8192", 8192, 8, 32, 8, 128, 32, "bf16", "i8", True, True),
        # a CosyVoice2 utterance's cache handed to a prompt attention in f32: latency
        _read("read_cv2_500", "500", 2, 64, 16, "e4m3", "f32"),
        # a full batch of long requests moved to 16-bit tensors: bandwidth
        _read("read_64_long", "spread:64:1000:16384", 8, 128, 32, "i8", "bf16"),
        # one CosyVoice2 utterance: latency
        _attend("attend_cv2_1", "500", 0, 14, 2, 64, 16, "f32", "e4m3"),
        # 16 concurrent Fish streams with ragged caches, f32 queries
        _attend("attend_fish_16", "1203,414,1845,980,256,1677,733,2040,1390,577,1121,1958,301,861,1544,1099", 0, 32, 8,
                128, 64, "f32", "e4m3"),
        # a full batch of long requests: bandwidth
        _attend("attend_64_long", "spread:64:1000:16384", 0, 32, 8, 128, 32, "bf16", "i8"),
        # five drafted tokens of each of 16 streams, verified together: latency and bandwidth
        _extend("extend_drafts_16", "spread:16:256:2040", "5", 32, 8, 128, 64, "bf16", "e4m3"),
        # ragged Fish prompts of three requests from empty caches, f32 queries
        _extend("extend_fish_prompt_1412", "0,0,0", "611,417,384", 32, 8, 128, 64, "f32", "e4m3"),
        # a chunk of one long prompt after what is cached of it: the matrix cores
        _extend("extend_chunk_2048", "30720", "2048", 32, 8, 128, 32, "bf16", "i8"),
    ]


def _write(name, tokens, requests, nh, nkv, hd, page, dtype, cache, norm, interleaved):
    return {"name": name, "family": "write", "tokens": tokens, "requests": requests, "nh": nh, "nkv": nkv, "hd": hd,
            "page": page, "dtype": dtype, "cache": cache, "norm": norm, "interleaved": interleaved}


def _read(name, lens, nkv, hd, page, cache, dtype):
    return {"name": name, "family": "read", "lens": lens, "nkv": nkv, "hd": hd, "page": page, "cache": cache, "dtype": dtype}


def _attend(name, lens, idle, nh, nkv, hd, page, dtype, cache):
    return {"name": name, "family": "attend", "lens": lens, "idle": idle, "nh": nh, "nkv": nkv, "hd": hd, "page": page,
            "dtype": dtype, "cache": cache}


def _extend(name, before, new, nh, nkv, hd, page, dtype, cache):
    return {"name": name, "family": "extend", "lens": before, "new": new, "nh": nh, "nkv": nkv, "hd": hd, "page": page,
            "dtype": dtype, "cache": cache}


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    family = rng.choice(["write", "write", "read", "attend", "attend", "extend", "extend"])
    page, cache, dtype = rng.choice([16, 32, 64, 128]), rng.choice(["i8", "e4m3"]), rng.choice(["f32", "bf16", "f16"])
    hd = rng.choice([64, 64, 80, 96, 128, 128, 256])
    nkv, group = rng.randint(1, 8), rng.choice([1, 2, 4, 5, 7, 8, 16])
    nh = nkv * group
    if family == "write":
        top = min(8192, 8192 * 48 * 128 // ((nh + 2 * nkv) * hd) // 2)
        tokens = _log(rng, 1, top)
        requests = rng.randint(1, min(tokens, 16)) if rng.random() < 0.7 else min(tokens, 256)
        case = _write("", tokens, requests, nh, nkv, hd, page, dtype, cache, rng.random() < 0.5, rng.random() < 0.5)
    elif family == "extend":
        # at most half of the largest listed case's scores, padded to the longest of each
        n = _log(rng, 1, 32)
        new = _log(rng, 1, 1500)
        room = 2048 * 32768 * 32 * 128 // 4 // (n * new * nh * hd)
        hi = min(30000, room - new)
        if hi < 16:
            n, new, hi = 1, _log(rng, 1, 200), _log(rng, 16, 8000)
        if n <= 4:
            before = ",".join(str(rng.choice([0, _log(rng, 1, hi)])) for _ in range(n))
            more = ",".join(str(_log(rng, 1, new)) for _ in range(n))
        else:
            before, more = f"spread:{n}:{_log(rng, 1, hi)}:{hi}", f"spread:{n}:{_log(rng, 1, new)}:{new}"
        case = _extend("", before, more, nh, nkv, hd, page, dtype, cache)
    else:
        n = _log(rng, 1, 256)
        # at most half of the positions and heads of the largest listed case
        top = 16384 * 8 * 128 * 8 // (nkv * hd * (max(1, group // 4) if family == "attend" else SIZE[dtype]))
        hi = _log(rng, 32, max(33, min(131072, top // n)))
        if n <= 4:
            lens = ",".join(str(_log(rng, 1, hi)) for _ in range(n))
        else:
            lens = f"spread:{n}:{_log(rng, 1, hi)}:{hi}"
        if family == "attend":
            case = _attend("", lens, rng.choice([0, 0, rng.randint(1, 3)]), nh, nkv, hd, page, dtype, cache)
        else:
            case = _read("", lens, nkv, hd, page, cache, dtype)
    del case["name"]
    return case


def _spread(n, lo, hi):
    """n lengths between lo and hi, even over their logarithm, in a mixed order."""
    return [int(round(lo * (hi / lo) ** ((i * 0.6180339887498949) % 1.0))) for i in range(n)]


def _counts(text):
    if text.startswith("spread:"):
        return _spread(*(int(v) for v in text.split(":")[1:]))
    return [int(v) for v in text.split(",")]


def _new_counts(case):
    before, new = _counts(case["lens"]), _counts(case["new"])
    return before, new * len(before) if len(new) == 1 else new


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
    """A table of random distinct pages holding the lengths."""
    order = rng.permutation(n_pages).astype(np.int32)
    table, at = np.full((len(lens), width), -1, np.int32), 0
    for i, n in enumerate(lens):
        b = _blocks(int(n), page)
        table[i, :b] = order[at:at + b]
        at += b
    return table


def _pow2_scale(amax, top):
    """The smallest power of two 2^e, e >= -100, with amax <= top 2^e (f32, exact)."""
    m, e = torch.frexp(amax)  # amax = m 2^e, 1/2 <= m < 1
    m_top, e_top = math.frexp(top)
    e = torch.where(m <= m_top, e - e_top, e - e_top + 1)
    return torch.ldexp(torch.ones_like(amax), torch.where(amax > 0, e, -100).clamp(min=-100))


def _codes(x, case):
    """Codes of x / scale (already divided)."""
    top = TOP[case["cache"]]
    x = x.clamp(-top, top)
    return x.round().to(torch.int8) if case["cache"] == "i8" else x.to(torch.float8_e4m3fn)


def _fill(codes, scale, case, seed, path):
    """Pages that hold quantized normal values, a few heads' channels larger than the others."""
    n_pages, nkv, page, hd = codes.shape
    spread = torch.exp(_normal((nkv, 1, hd), 0.5, torch.float32, seed, path + 10))
    step = max(1, (1 << 28) // (nkv * page * hd))
    for a in range(0, n_pages, step):
        x = _normal((min(step, n_pages - a), nkv, page, hd), 1.0, torch.float32, seed + a, path).mul_(spread)
        x = x.view(x.shape[0], nkv, page // BLOCK, BLOCK, hd)
        s = _pow2_scale(x.abs().amax((-2, -1)), TOP[case["cache"]])
        scale[a:a + step] = s
        codes[a:a + step] = _codes(x / s[..., None, None], case).view(-1, nkv, page, hd)


def prepare(case, seed):
    st, page, family = dict(case), case["page"], case["family"]
    nkv, hd = case["nkv"], case["hd"]
    rng = np.random.default_rng(seed)
    new = None
    if family == "write":
        new = [case["tokens"] // case["requests"] + (i < case["tokens"] % case["requests"]) for i in range(case["requests"])]
        # (which request begins where goes by the seed, the outputs' size does not)
        before = rng.permutation(np.random.default_rng(case["requests"]).integers(0, 1000, case["requests"]))
        lens, most = before + new, 1000 + np.asarray(new)
    elif family == "extend":
        before, new = _new_counts(case)
        lens = most = np.asarray(before) + new
    else:
        lens = most = np.asarray(_counts(case["lens"]))
    max_len = max(1, int(most.max()))
    n_pages = int(_blocks(most, page).sum()) + 3
    table = _page_tables(lens, page, _blocks(max_len, page), n_pages, rng)
    if own:
        from syrinx_amd.paged import PagedKvCache

        kv = st["kv"] = PagedKvCache(1, nkv, hd, n_pages=n_pages, page_size=page, max_rows=len(lens), max_len=max_len,
                                     dtype=DTYPE[case["cache"]], device=DEV)
        kv.lens.copy_(_i32(lens))
        kv.table.copy_(_i32(table))
        st.update(k=kv.k[0], v=kv.v[0], k_scale=kv.k_scale[0], v_scale=kv.v_scale[0], lens_dev=kv.lens, table=kv.table)
    else:
        shape = (n_pages, nkv, page, hd)
        st.update(k=torch.empty(shape, dtype=DTYPE[case["cache"]], device=DEV),
                  v=torch.empty(shape, dtype=DTYPE[case["cache"]], device=DEV),
                  k_scale=torch.empty((n_pages, nkv, page // BLOCK), device=DEV),
                  v_scale=torch.empty((n_pages, nkv, page // BLOCK), device=DEV), lens_dev=_i32(lens), table=_i32(table))
    _fill(st["k"], st["k_scale"], case, seed, 1)
    _fill(st["v"], st["v_scale"], case, seed, 2)
    if new is not None:
        # the map of the new tokens, as the page allocator makes it
        row = np.repeat(np.arange(len(new)), new)
        pos = np.concatenate([np.arange(b, b + n) for b, n in zip(before, new)])
        slot = table[row, pos // page].astype(np.int64) * page + pos % page
        st.update(rows=_i32(row), pos=_i32(pos), slots=_i32(slot))
    if family in ("write", "read"):
        # the ranges read back: from the first touched block on, or whole requests
        first = np.asarray(before) // BLOCK * BLOCK if family == "write" else np.zeros_like(lens)
        count = lens - first
        cu = np.concatenate([[0], np.cumsum(count)])
        st.update(total=int(cu[-1]), cu=_i32(cu), start=_i32(first))
        if family == "read":
            out = DTYPE[case["dtype"]]
        else:
            out = torch.bfloat16
        st["back"] = tuple(torch.empty((st["total"], nkv, hd), dtype=out, device=DEV) for _ in range(2))
    if family == "write":
        nh, dt = case["nh"], DTYPE[case["dtype"]]
        ang = np.arange(max_len)[:, None] * THETA ** (-2.0 * np.arange(hd // 2) / hd)
        block = np.concatenate([np.arange(b // BLOCK, _blocks(n, BLOCK)) for b, n in zip(before, lens)])
        brow = np.repeat(np.arange(len(lens)), _blocks(lens, BLOCK) - np.asarray(before) // BLOCK)
        st.update(cos=torch.as_tensor(np.cos(ang).astype(np.float32)).to(DEV),
                  sin=torch.as_tensor(np.sin(ang).astype(np.float32)).to(DEV),
                  qkv=_normal((case["tokens"], (nh + 2 * nkv) * hd), 1.5, dt, seed, 3),
                  out=torch.empty((case["tokens"], nh * hd), dtype=dt, device=DEV),
                  touched=torch.as_tensor(table[brow, block * BLOCK // page].astype(np.int64) * (page // BLOCK)
                                          + block % (page // BLOCK)).to(DEV))
        st["q_norm"] = 1.0 + _normal((hd,), 0.1, torch.float32, seed, 4) if case["norm"] else None
        st["k_norm"] = 1.0 + _normal((hd,), 0.1, torch.float32, seed, 5) if case["norm"] else None
        if own:
            from syrinx_amd.paged import SlotMap

            st["map"] = SlotMap(slots=st["slots"], pos=st["pos"], rows=st["rows"])
    elif family == "attend":
        n, idle = len(lens), case["idle"]
        st.update(q=_normal((n + idle, case["nh"], hd), 2.0, DTYPE[case["dtype"]], seed, 3),
                  rows=_i32(list(range(n)) + [-1] * idle), top=max_len, n=n,
                  out=torch.zeros((n + idle, case["nh"], hd), dtype=DTYPE[case["dtype"]], device=DEV))
    elif family == "extend":
        at = np.concatenate([np.arange(n) for n in new])
        st.update(q=_normal((int(sum(new)), case["nh"], hd), 2.0, DTYPE[case["dtype"]], seed, 3), top=max_len, n=len(new),
                  most_new=int(max(new)), at=torch.as_tensor(at).to(DEV),
                  out=torch.empty((int(sum(new)), case["nh"], hd), dtype=DTYPE[case["dtype"]], device=DEV))
    return st


# ---- the plain forms ------------------------------------------------------------------

def _rotate(x, c, s, interleaved):
    if interleaved:
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2)
    a, b = x.chunk(2, -1)
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def _bytes(codes):
    """The codes as bytes, which torch indexes whatever they stand for."""
    return codes.view(torch.uint8)


def _values(st, b):
    return b.view(DTYPE[st["cache"]]).float()


def _store(st, codes, scale, x):
    """The new rows x [tokens, nkv, hd] into one of the two pools."""
    page, hd, nkv = st["page"], st["hd"], st["nkv"]
    per, slot = page // BLOCK, st["slots"].long()
    blk, hit = slot // BLOCK, st["touched"]
    pg, b = hit // per, hit % per
    # what each block needs now, and what it had (nothing, if its first position is among the new)
    need = torch.zeros((scale.shape[0] * per, nkv), device=DEV)
    need.index_reduce_(0, blk, x.abs().amax(-1), "amax")
    begun = torch.zeros(need.shape[0], device=DEV)
    begun.index_reduce_(0, blk, (slot % BLOCK == 0).float(), "amax")
    had, fresh = scale[pg, :, b], begun[hit][:, None] > 0
    s = torch.maximum(_pow2_scale(need[hit], TOP[st["cache"]]), torch.where(fresh, torch.zeros_like(had), had))
    view = _bytes(codes).view(-1, nkv, per, BLOCK, hd)
    ratio = torch.where(fresh, torch.ones_like(had), had / s)
    view[pg, :, b] = _bytes(_codes(_values(st, view[pg, :, b]) * ratio[..., None, None], st))
    scale[pg, :, b] = s
    at = scale[slot // page, :, slot % page // BLOCK]
    _bytes(codes)[slot // page, :, slot % page] = _bytes(_codes(x / at[..., None], st))


def _write_plain(st):
    nh, nkv, hd = st["nh"], st["nkv"], st["hd"]
    x = st["qkv"].float().view(-1, nh + 2 * nkv, hd)
    q, k, v = x.split([nh, nkv, nkv], 1)
    if st["norm"]:
        q = q / torch.sqrt((q * q).mean(-1, keepdim=True) + EPS) * st["q_norm"]
        k = k / torch.sqrt((k * k).mean(-1, keepdim=True) + EPS) * st["k_norm"]
    at = st["pos"].long()
    c, s = st["cos"][at][:, None], st["sin"][at][:, None]
    q, k = _rotate(q, c, s, st["interleaved"]), _rotate(k, c, s, st["interleaved"])
    _store(st, st["k"], st["k_scale"], k)
    _store(st, st["v"], st["v_scale"], v)
    st["out"].copy_(q.reshape(st["out"].shape))


def _read_plain(st):
    page, cu = st["page"], st["cu"].long()
    t = torch.arange(st["total"], device=DEV)
    row = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    pos = st["start"].long()[row] + t - cu[row]
    pg, o = st["table"][row, pos // page].long(), pos % page
    for out, codes, scale in ((st["back"][0], st["k"], st["k_scale"]), (st["back"][1], st["v"], st["v_scale"])):
        out.copy_(_values(st, _bytes(codes)[pg, :, o]) * scale[pg, :, o // BLOCK][..., None])


def _padded(st, codes, scale):
    """[requests, nkv, positions, hd] in f32, as many positions as the longest request has pages for."""
    nkv, hd, page = st["nkv"], st["hd"], st["page"]
    pages = st["table"].long().clamp(min=0)[:st["n"], :_blocks(st["top"], page)]
    x = _values(st, _bytes(codes)[pages]).view(*pages.shape, nkv, page // BLOCK, BLOCK, hd) * scale[pages][..., None, None]
    return x.permute(0, 2, 1, 3, 4, 5).reshape(pages.shape[0], nkv, -1, hd)


def _weighted(st, q, limit):
    """softmax over the first limit positions [n, tokens] of q [n, nkv, group, tokens, hd]."""
    n, nkv, group, tokens, hd = q.shape
    k = _padded(st, st["k"], st["k_scale"]).transpose(2, 3).contiguous()
    s = torch.matmul(q.reshape(n, nkv, group * tokens, hd), k).view(n, nkv, group, tokens, -1) / math.sqrt(hd)
    gone = torch.arange(s.shape[-1], device=DEV) >= limit[..., None]
    s = s.masked_fill_(gone[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    p = s.sub_(torch.where(torch.isinf(top), torch.zeros_like(top), top)).exp_()
    total = p.sum(-1, keepdim=True)
    v = _padded(st, st["v"], st["v_scale"])
    o = torch.matmul(p.view(n, nkv, group * tokens, -1), v).view(q.shape)
    return o / torch.where(total == 0, torch.ones_like(total), total)


def _attend_plain(st):
    nh, nkv, hd, n = st["nh"], st["nkv"], st["hd"], st["n"]
    q = st["q"][:n].float().view(n, nkv, nh // nkv, 1, hd)
    st["out"][:n] = _weighted(st, q, st["lens_dev"].long()[:, None]).view(n, nh, hd)


def _extend_plain(st):
    nh, nkv, hd, n = st["nh"], st["nkv"], st["hd"], st["n"]
    q = torch.zeros((n, st["most_new"], nkv, nh // nkv, hd), device=DEV)
    limit = torch.zeros((n, st["most_new"]), dtype=torch.long, device=DEV)
    row = st["rows"].long()
    q[row, st["at"]] = st["q"].float().view(-1, nkv, nh // nkv, hd)
    limit[row, st["at"]] = st["pos"].long() + 1
    o = _weighted(st, q.permute(0, 2, 3, 1, 4).contiguous(), limit)
    st["out"].copy_(o.permute(0, 3, 1, 2, 4)[row, st["at"]].reshape(-1, nh, hd))


def run(st):
    family = st["family"]
    if family == "write":
        if own:
            st["kv"].append(0, st["qkv"], st["map"], n_heads=st["nh"], q_norm=st["q_norm"], k_norm=st["k_norm"], eps=EPS,
                            rope=(st["cos"], st["sin"]), interleaved=st["interleaved"], out=st["out"])
            st["kv"].read(0, st["cu"], st["total"], start=st["start"], out=st["back"])
        else:
            _write_plain(st)
            _read_plain(st)
        return [st["out"], *st["back"]]
    if family == "read":
        if own:
            st["kv"].read(0, st["cu"], st["total"], start=st["start"], out=st["back"])
        else:
            _read_plain(st)
        return [*st["back"]]
    if family == "attend":
        if own:
            st["kv"].attend(0, st["q"], rows=st["rows"], out=st["out"])
        else:
            _attend_plain(st)
        return [st["out"]]
    if own:
        st["kv"].attend(0, st["q"], rows=st["rows"], pos=st["pos"], out=st["out"])
    else:
        _extend_plain(st)
    return [st["out"]]


# ---- what a pass cannot do without ----------------------------------------------------

def work(case):
    page, family, nkv, hd = case["page"], case["family"], case["nkv"], case["hd"]
    held = nkv * (hd + 4 / BLOCK)  # bytes of a position's keys or values
    if family == "write":
        t, nh, e = case["tokens"], case["nh"], SIZE[case["dtype"]]
        return {"bytes": int(t * ((2 * nh + 2 * nkv) * hd * e + 4 * hd + 8 + 4 * held + 4 * nkv * hd)),
                "flops": t * (nh + 2 * nkv) * hd * (3 + (4 if case["norm"] else 0))}
    if family == "read":
        lens = _counts(case["lens"])
        return {"bytes": int(sum(lens) * 2 * (held + nkv * hd * SIZE[case["dtype"]]) + sum(4 * _blocks(n, page) for n in lens)),
                "flops": 2 * sum(lens) * nkv * hd}
    nh, e = case["nh"], SIZE[case["dtype"]]
    if family == "attend":
        lens = _counts(case["lens"])
        queries, pairs = len(lens), sum(lens)
    else:
        before, new = _new_counts(case)
        lens, queries = [b + n for b, n in zip(before, new)], sum(new)
        pairs = sum(b * n + n * (n + 1) // 2 for b, n in zip(before, new))
    return {"bytes": int(sum(lens) * 2 * held + 2 * queries * nh * hd * e + sum(4 * _blocks(n, page) for n in lens) + 8 * queries),
            "flops": 4 * pairs * nh * hd}


# ---- the definitions, in 64 bits ------------------------------------------------------

def _round8(x, kind):
    """x (64 bits) to the nearest value that a code can stand for, ties to even, ends kept."""
    top = TOP[kind]
    x = np.clip(x, -top, top)
    if kind == "i8":
        return np.rint(x)
    step = np.exp2(np.maximum(np.floor(np.log2(np.maximum(np.abs(x), 2.0 ** -30))), -6) - 3)
    return np.clip(np.rint(x / step) * step, -top, top)


def _held(st, codes, scale, i, n):
    """Request i's first n positions, [nkv, n, hd], on the host."""
    pages = st["table"][i, :_blocks(n, st["page"])].long()
    c, s = _values(st, _bytes(codes)[pages]).double(), scale[pages].double()
    x = c * s.repeat_interleave(BLOCK, -1)[..., None]
    return x.transpose(0, 1).reshape(c.shape[1], -1, c.shape[3])[:, :n]


def _write_exact(case, st):
    nh, nkv, hd, page, kind = case["nh"], case["nkv"], case["hd"], case["page"], case["cache"]
    heads = st["qkv"].to(F64).view(-1, nh + 2 * nkv, hd)
    if case["norm"]:
        rms = torch.rsqrt(heads.square().mean(-1, keepdim=True) + EPS)
        w = torch.cat([st["q_norm"].to(F64).expand(nh, hd), st["k_norm"].to(F64).expand(nkv, hd)])
        heads = torch.cat([heads[:, :nh + nkv] * rms[:, :nh + nkv] * w, heads[:, nh + nkv:]], 1)
    # the rotation as a complex product
    turn = torch.complex(st["cos"].to(F64), st["sin"].to(F64))[st["pos"].long()][:, None]
    rot = heads[:, :nh + nkv]
    if case["interleaved"]:
        z = torch.complex(rot[..., 0::2].contiguous(), rot[..., 1::2].contiguous()) * turn
        rot = torch.view_as_real(z).reshape(-1, nh + nkv, hd)
    else:
        z = torch.complex(rot[..., :hd // 2].contiguous(), rot[..., hd // 2:].contiguous()) * turn
        rot = torch.cat([z.real, z.imag], -1)
    rows, pos, lens = (st[k].cpu().numpy().astype(np.int64) for k in ("rows", "pos", "lens_dev"))
    back = []
    for codes, scale, x in ((st["k"], st["k_scale"], rot[:, nh:]), (st["v"], st["v_scale"], heads[:, nh + nkv:])):
        x, parts = x.cpu().numpy(), []
        for i, n in enumerate(lens):
            mine = rows == i
            first = int(pos[mine][0])
            lo = first // BLOCK * BLOCK
            held = _held(st, codes, scale, i, int(n))[:, lo:].cpu().numpy()
            held[:, first - lo:] = x[mine].transpose(1, 0, 2)
            for a in range(0, held.shape[1], BLOCK):
                block, fresh = held[:, a:a + BLOCK], lo + a >= first
                added = block if fresh else block[:, first - lo:]
                amax = np.abs(added).max((1, 2))
                e = np.maximum(np.ceil(np.log2(np.maximum(amax, 2.0 ** -120) / TOP[kind]) - 1e-13), -100)
                e = np.where(amax > TOP[kind] * np.exp2(e), e + 1, e)
                if not fresh:
                    at = int(st["table"][i, (lo + a) // page])
                    e = np.maximum(e, np.log2(scale[at, :, (lo + a) % page // BLOCK].double().cpu().numpy()))
                s = np.exp2(e)[:, None, None]
                block[:] = _round8(block / s, kind) * s
            parts.append(held)
        back.append(torch.as_tensor(np.concatenate(parts, 1).transpose(1, 0, 2)))
    return [rot[:, :nh].reshape(rot.shape[0], -1), *back]


def exact(case, seed):
    st = _plain_state(case, seed)
    nkv, hd, family = case["nkv"], case["hd"], case["family"]
    if family == "write":
        return _write_exact(case, st)
    if family == "read":
        lens = _counts(case["lens"])
        return [torch.cat([_held(st, c, s, i, n).transpose(0, 1) for i, n in enumerate(lens)])
                for c, s in ((st["k"], st["k_scale"]), (st["v"], st["v_scale"]))]
    nh = case["nh"]
    group, out = nh // nkv, st["out"].to(F64)
    if family == "attend":
        before, new = [n - 1 for n in _counts(case["lens"])], [1] * st["n"]
    else:
        before, new = _new_counts(case)
    at = 0
    for i, (b, m) in enumerate(zip(before, new)):
        k, v = (_held(st, st[name], st[name + "_scale"], i, b + m) for name in ("k", "v"))
        q = st["q"][at:at + m].to(F64).view(m, nkv, group, hd)
        seen = torch.arange(b + m, device=DEV)[None, :] <= torch.arange(b, b + m, device=DEV)[:, None]
        for h in range(nkv):
            s = (q[:, h].reshape(m * group, hd) @ k[h].t().contiguous()).view(m, group, -1) / math.sqrt(hd)
            p = torch.softmax(s.masked_fill(~seen[:, None], -math.inf), -1)
            out[at:at + m, h * group:(h + 1) * group] = (p.view(m * group, -1) @ v[h]).view(m, group, hd)
        at += m
    return [out]


def _plain_state(case, seed):
    """The inputs alone, as ``prepare`` makes them, without a cache object."""
    global own
    kept, own = own, False
    try:
        return prepare(case, seed)
    finally:
        own = kept
