"""The 8-bit paged cache on the GPU where it can go wrong beside test_gpu_paged8's cases: threads, maps
of more entries than tokens, value scales far from one, pools of other strides under many rows."""
import ctypes
import math
import threading

import numpy as np
import pytest
import torch

from test_gpu_paged import DT, F64, U32, _close
from test_gpu_paged8 import CT, PREFIX_SPLIT, B, _attend, _cache, _code_values, _filled, _queries, _reference, cuda  # noqa: F401

pytestmark = pytest.mark.gpu


def _i32(cuda, v):
    return torch.tensor(v, dtype=torch.int32, device=cuda)


def test_threads_attend_on_one_stream_at_once(cuda):
    """Two threads, calls of unlike sizes, both on the default stream: each call's outputs are its own."""
    cache, g = _filled(cuda, 2, 64, 16, [5000, 300], "i8", 2)
    calls = []
    for n in (3, 700):
        q = _queries(g, cuda, n, 8, 64, "bf16")
        rows, pos = _i32(cuda, [i % 2 for i in range(n)]), _i32(cuda, [299 - i % 290 for i in range(n)])
        calls.append((q, rows, pos, cache.attend(0, q, rows=rows, pos=pos), cache.attend(0, q, rows=rows)))
    torch.cuda.synchronize()
    got = [[], []]

    def work(i):
        q, rows, pos = calls[i][:3]
        for _ in range(50):
            got[i].append((cache.attend(0, q, rows=rows, pos=pos), cache.attend(0, q, rows=rows)))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for i in range(2):
        assert len(got[i]) == 50
        assert all(torch.equal(x, calls[i][3]) and torch.equal(y, calls[i][4]) for x, y in got[i])


@pytest.mark.parametrize("form", [False, True, "wide"])
@pytest.mark.parametrize("ct", ["i8", "e4m3"])
def test_scores_of_rows_and_scales_far_apart(cuda, ct, form):
    """f32 queries whose power of two and the keys' scale pass f32's range together.  A huge element
    that meets zeros in every key has scores of zero: even weights.  An infinite one that meets
    negative codes alone has scores of -inf: no weights, zeros."""
    L, hd = 300, 64
    cache, g = _filled(cuda, 1, hd, 16, [L], ct, 4)
    held = cache.table[0, :-(-L // 16)].long()
    values = (cache.v[0, held, 0].float() * cache.v_scale[0, held, 0, 0][:, None, None]).to(F64).view(-1, hd)[:L]
    rows, pos = _i32(cuda, [0]), _i32(cuda, [L - 1]) if form else None
    codes = cache.k[0].float().nan_to_num(3.0)
    q = torch.zeros((1, 2, hd), device=cuda)
    for first, scale, by in ((0.0, 2.0 ** 60, 2.0 ** 100), (0.0, 2.0 ** 100, -2.0 ** 127), (-1.0, 2.0 ** -30, math.inf),
                             (-2.0, 2.0 ** -100, math.inf)):
        codes[..., 0] = first
        cache.k[0] = codes.to(cache.k.dtype)
        cache.k_scale[0, held] = scale
        q[:] = 0
        q[..., 0] = by
        got = _attend(cache, q, rows, pos, form)
        if first:
            assert not bool(got.any()), (first, scale, by)
        else:
            # even weights, each 1 / L within 2^-16 (parts, exponential, a sum of L terms), a value off by nothing
            off = (got[0, 0].to(F64) - values.mean(0)).abs()
            assert bool((off <= 2.0 ** -16 * values.abs().mean(0)).all()), (first, scale, by)


@pytest.mark.parametrize("qt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("form", [False, True, "wide"])
@pytest.mark.parametrize("ct", ["i8", "e4m3"])
def test_weights_beside_value_scales(cuda, ct, form, qt):
    """Keys whose scores are all one power of two times the factor, so that each weight is exp(0) = 1 and
    every sum exact: the half of the positions whose values are ones is a half, whatever the scales of
    the other half's values (zeros), and whatever the scores."""
    hd, L = 64, 32
    cache, _ = _filled(cuda, 1, hd, 16, [L], ct, 5)
    one, other = cache.table[0, :2].long().tolist()
    cache.k[0] = torch.ones_like(cache.k[0].float()).to(cache.k.dtype)
    cache.k_scale[0] = 0.5
    cache.v[0] = torch.zeros_like(cache.v[0].float()).to(cache.v.dtype)
    cache.v[0, one] = torch.ones_like(cache.v[0, one].float()).to(cache.v.dtype)
    cache.v_scale[0, one] = 1.0
    q = torch.zeros((1, 2, hd), dtype=DT[qt], device=cuda)
    q[0, 0, 3], q[0, 1, 40] = 4.0, -8.0
    rows, pos = _i32(cuda, [0]), _i32(cuda, [L - 1]) if form else None
    for e in (0, -3, -9, -20, -33, -50, -60, -61, -100, 17, 99):
        cache.v_scale[0, other] = 2.0 ** e
        for scale in (0.125, 0.3, 0.7071, 1.1, 1.7):
            n, more = 1, 32768 // 2 + 1
            if form == "wide":
                none = torch.full((more,), -1, dtype=torch.int32, device=cuda)
                qq = torch.cat([q, torch.zeros((more, 2, hd), dtype=q.dtype, device=cuda)])
                got = cache.attend(0, qq, rows=torch.cat([rows, none]), pos=torch.cat([pos, none]), scale=scale)[:n]
            else:
                got = cache.attend(0, q, rows=rows, pos=pos, scale=scale)
            assert bool((got == 0.5).all()), (e, scale, float((got.float() - 0.5).abs().max()))


@pytest.mark.parametrize("ct", ["i8", "e4m3"])
@pytest.mark.parametrize("nh,nkv,hd", [(8, 2, 64), (32, 8, 128), (4, 2, 256)])
def test_drafts_keep_the_precision_of_one_token(cuda, ct, nh, nkv, hd):
    """Positions in a call of few rows take nothing from its weights: bf16 queries too carry them in two
    parts, as without positions (the bound that one part passes where values of both signs cancel)."""
    lens = [40, 300, 1000, 7]
    cache, g = _filled(cuda, nkv, hd, 32, lens, ct, hd)
    rows = [r for r in range(4) for _ in range(5)]
    pos = [lens[r] - 5 + j for r in range(4) for j in range(5)]
    q = _queries(g, cuda, 20, nh, hd, "bf16")
    got = cache.attend(0, q, rows=_i32(cuda, rows), pos=_i32(cuda, pos))
    want, bound = _reference(q, cache, rows, [p + 1 for p in pos], hd ** -0.5, split=2.0 ** -17)
    _close(got, want, bound, torch.bfloat16)


def _prefix_with_plan(cache, q, rows, pos, out=None):
    """attend over prefixes, and what its plan says (the workspace begins with it): items, tiles that are
    cut, their pieces."""
    ws = cache.workspace(q.shape[0], q.shape[1], prefix=True)
    got = cache.attend(0, q, rows=rows, pos=pos, out=out, workspace=ws)
    return got, ws[:12].view(torch.int32).tolist()


@pytest.mark.parametrize("qt", ["f32", "bf16"])
@pytest.mark.parametrize("entries", [600, 8192])
def test_padded_maps_are_cut_as_their_live_tokens_ask(cuda, entries, qt):
    """A map of a captured step's fixed capacity, few of whose entries have tokens: what few tokens see of
    a long request is divided over the card as in a call of these tokens alone."""
    lens, nh, nkv, hd = [30000, 50], 32, 8, 128
    cache, g = _filled(cuda, nkv, hd, 32, lens, "i8", 6)
    at = [0, 1, 2, 3, 40, entries - 1]
    rows, pos = [-1] * entries, [-1] * entries
    for i, (r, p) in zip(at, [(0, 29996), (0, 29997), (0, 29998), (0, 29999), (1, 20), (0, 15000)]):
        rows[i], pos[i] = r, p
    q = _queries(g, cuda, entries, nh, hd, qt)
    out = torch.full_like(q, 7.0)
    got, (items, cut, pieces) = _prefix_with_plan(cache, q, _i32(cuda, rows), _i32(cuda, pos), out)
    some, (items1, cut1, pieces1) = _prefix_with_plan(cache, q[at], _i32(cuda, [rows[i] for i in at]), _i32(cuda, [pos[i] for i in at]))
    assert cut >= 2 and cut1 >= 2 and pieces > 20 and items == pieces + (3 - cut)
    want, bound = _reference(q[at], cache, [rows[i] for i in at], [pos[i] + 1 for i in at], hd ** -0.5, split=PREFIX_SPLIT[qt])
    _close(got[at], want, bound, DT[qt])
    _close(some, want, bound, DT[qt])
    rest = torch.ones(entries, dtype=torch.bool, device=cuda)
    rest[at] = False
    assert bool((got[rest] == 7).all())


@pytest.mark.parametrize("short,nh,nkv,hd,qt", [(1100, 4, 1, 64, "bf16"), (300, 32, 8, 64, "f16"), (300, 32, 8, 128, "bf16"),
                                                (3000, 8, 2, 32, "f32"), (2048, 2, 1, 256, "bf16"), (1023, 1, 1, 128, "f32")])
def test_one_long_request_beside_many_short_ones_is_cut(cuda, short, nh, nkv, hd, qt):
    """However many tiles there are, before and after it."""
    rng = np.random.default_rng(short)
    long = short // 3
    lens = [int(v) for v in rng.integers(1, 40, short)]
    lens.insert(long, 20000)
    cache, g = _filled(cuda, nkv, hd, 16, lens, "e4m3", short)
    rows, pos = [], []
    for r, n in enumerate(lens):
        for p in ([n - 1] if r != long else [17000, 19998, 19999]):
            rows.append(r)
            pos.append(p)
    q = _queries(g, cuda, len(rows), nh, hd, qt)
    got, (items, cut, pieces) = _prefix_with_plan(cache, q, _i32(cuda, rows), _i32(cuda, pos))
    assert cut == 1 and pieces > 10 and items == short + pieces
    some = [0, 1, long, long + 1, long + 2, long + 3, len(rows) - 1, len(rows) - 2] + rng.permutation(len(rows))[:80].tolist()
    want, bound = _reference(q[some], cache, [rows[i] for i in some], [pos[i] + 1 for i in some], hd ** -0.5, split=PREFIX_SPLIT[qt])
    _close(got[some], want, bound, DT[qt])


def test_many_tiles_of_which_none_is_cut(cuda):
    """More tiles than stay in LDS, alike in length: they go as they are, every query's result there."""
    n, nh = 2600, 2
    cache, g = _filled(cuda, 1, 32, 16, [int(v) for v in np.random.default_rng(1).integers(0, 60, n)], "i8", 9)
    rows = list(range(n))
    q = _queries(g, cuda, n, nh, 32, "f16")
    got, (items, cut, pieces) = _prefix_with_plan(cache, q, _i32(cuda, rows), _i32(cuda, [1 << 30] * n))
    assert (items, cut, pieces) == (n, 0, 0)
    want, bound = _reference(q, cache, rows, [1 << 30] * n, 32 ** -0.5)
    _close(got, want, bound, torch.float16)


@pytest.mark.parametrize("it", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("ct", ["i8", "e4m3"])
def test_append_of_rows_whose_norm_is_exact(cuda, ct, it):
    """Rows of elements +-n: the root mean square is n, a row over it +-1 and times the weight the weight,
    all exact, so that weights half way between two codes go to the even one, and queries are the
    weights.  (n times the rounded inverse of these n is not 1.)"""
    nh, nkv, hd = 2, 1, 64
    ns = [41, 47, 55, 61, 82, 83, 94, 97, 107, 109]
    cache = _cache(cuda, nkv, hd, ct, n_pages=10, page=16, rows=10, max_len=16)
    sign = torch.where(torch.arange(hd, device=cuda) % 3 == 1, -1.0, 1.0)
    qkv = (torch.tensor(ns, device=cuda, dtype=torch.float32)[:, None] * sign).repeat(1, nh + 2 * nkv).to(DT[it])
    if ct == "i8":
        w = (torch.arange(hd, device=cuda) + 63.5) * 2.0 ** -6  # codes of a scale of 2^-6
    else:
        w = (2 * torch.arange(hd, device=cuda) % 16 + 17) * 2.0 ** -4  # between two of eight codes
    m = cache.reserve([1] * 10)
    q = cache.append(0, qkv, m, n_heads=nh, q_norm=w, k_norm=w, eps=0.0).view(10, nh, hd)
    assert torch.equal(q, (w * sign).to(DT[it]).expand(10, nh, hd))
    s = cache.k_scale[0, m.slots.long() // 16, 0, 0].to(F64)
    assert bool((s == (2.0 ** -6 if ct == "i8" else 2.0 ** -7)).all())
    want = _code_values((w * sign).to(F64) / s[:, None], ct)
    got = cache.k[0, m.slots.long() // 16, 0, m.slots.long() % 16]
    assert torch.equal(got.float().to(F64), want)


@pytest.mark.parametrize("ct", ["i8", "e4m3"])
def test_append_of_rows_whose_norm_passes_the_range(cuda, ct):
    """Rows whose mean square is infinite in f32 become zeros, but for what is infinite itself (NaN, not a
    number's code); rows of zeros without an eps NaN; rows of the smallest and largest squares ordinary."""
    hd = 32
    cache = _cache(cuda, 1, hd, ct, n_pages=6, page=16, rows=6, max_len=16)
    x = torch.ones((6, hd), device=cuda)
    x[0] = 1e30
    x[1, 3] = math.inf
    x[2] = 0.0
    x[3] = 2e-19
    x[4] = 1e18
    x[5] *= torch.where(torch.arange(hd, device=cuda) % 2 == 0, 1.0, -1.0)
    w = torch.full((hd,), 2.0, device=cuda)
    q = cache.append(0, x.repeat(1, 3), cache.reserve([1] * 6), n_heads=1, q_norm=w, k_norm=w, eps=0.0)
    k, _ = cache.read(0, torch.arange(7, dtype=torch.int32, device=cuda), 6, dtype=torch.float32)
    nan = torch.tensor(math.nan, device=cuda) if ct == "e4m3" else torch.tensor(0.0, device=cuda)
    want = torch.full((6, hd), 2.0, device=cuda)
    want[0] = 0.0
    want[1] = 0.0
    want[5] *= x[5]
    got, one = q.clone(), torch.full((), math.nan, device=cuda)
    want[1, 3], want[2] = one, one
    assert torch.allclose(got, want, rtol=2.0 ** -20, atol=0, equal_nan=True)
    want[1, 3], want[2] = nan, nan
    # (codes: 2 is one of both kinds; within half a step where the norm rounds)
    assert torch.allclose(k[:, 0], want, rtol=2.0 ** -4, atol=0, equal_nan=True)


@pytest.mark.parametrize("ct,code", [("i8", 24), ("e4m3", 0x101)])
@pytest.mark.parametrize("hd", [64, 80, 128, 256])
def test_many_rows_over_pools_of_other_strides(cuda, ct, code, hd):
    """Tiles of many rows over position-major pages, keys and values of one tensor, scales of one tensor,
    queries and outputs as columns of wider rows: the bits of the same call over pages of their own."""
    from syrinx_amd import lib
    from syrinx_amd._lib import check
    from syrinx_amd.paged import KvPages

    nh, nkv, page, lens = 6, 2, 32, [5, 100, 33, 400]
    plain, g = _filled(cuda, nkv, hd, page, lens, ct, hd)
    n_pages = plain.n_pages
    both = torch.full((n_pages, page, 2, nkv, hd + 16), 0x7F, dtype=torch.uint8, device=cuda)
    sc = torch.full((n_pages, 2, nkv, page // B + 1), math.nan, device=cuda)
    k, v = both[:, :, 0, :, :hd], both[:, :, 1, :, :hd]
    for mine, scale, codes, scales in ((k, sc[:, 0], plain.k[0], plain.k_scale[0]), (v, sc[:, 1], plain.v[0], plain.v_scale[0])):
        mine.copy_(codes.view(torch.uint8).transpose(1, 2))
        scale[..., :page // B] = scales
    pages = KvPages(code, nkv, hd, page, n_pages, k.data_ptr(), v.data_ptr(), k.stride(0), k.stride(2), k.stride(1),
                    sc[:, 0].data_ptr(), sc[:, 1].data_ptr(), sc.stride(0), sc.stride(2))
    live = [(r, p) for r, n in enumerate(lens) for p in range(max(0, n - 150), n)]
    n = 32768 // nh + 1 + len(live)
    rows = _i32(cuda, [r for r, _ in live] + [-1] * (n - len(live)))
    pos = _i32(cuda, [p for _, p in live] + [-1] * (n - len(live)))
    for qt in ("f32", "bf16", "f16"):
        qw = (2 * torch.randn((n, (nh + 4) * hd), generator=g, device=cuda)).to(DT[qt])
        q = qw.as_strided((n, nh, hd), (qw.stride(0), hd, 1))
        buf = torch.full((n, (nh + 1) * hd), 3.0, device=cuda, dtype=DT[qt])
        size = ctypes.c_size_t()
        check(lib().sxq_kv_prefix_attention_workspace(ctypes.byref(pages), n, nh, ctypes.byref(size)))
        ws = torch.full((size.value,), 0xA5, dtype=torch.uint8, device=cuda)
        check(lib().sxq_kv_prefix_attention(0, ctypes.byref(pages), {"f32": 0, "f16": 1, "bf16": 30}[qt], q.data_ptr(), q.stride(0), n, nh,
                                            rows.data_ptr(), pos.data_ptr(), plain.lens.data_ptr(), len(lens), plain.table.data_ptr(),
                                            plain.max_blocks, plain.max_blocks, 0.1, buf.data_ptr(), buf.stride(0), ws.data_ptr(),
                                            size.value, torch.cuda.current_stream().cuda_stream))
        out = torch.full((n, nh, hd), 3.0, device=cuda, dtype=DT[qt])
        want = plain.attend(0, q.contiguous(), rows=rows, pos=pos, scale=0.1, out=out)
        assert bool(want[:len(live)].isfinite().all()) and bool((want[len(live):] == 3).all())
        assert torch.equal(buf[:, :nh * hd].reshape(n, nh, hd), want) and bool((buf[:, nh * hd:] == 3).all())
        some = [0, 4, 5, 104, 137, 138, len(live) - 1]
        ref, bound = _reference(q[some].contiguous(), plain, [live[i][0] for i in some], [live[i][1] + 1 for i in some], 0.1,
                                split=PREFIX_SPLIT[qt])
        _close(want[some], ref, bound, DT[qt])


@pytest.mark.parametrize("form", [True, "wide"])
@pytest.mark.parametrize("hd,n_pages", [(64, 600000), (128, 300000), (256, 150000)])
def test_prefixes_past_32_bits(cuda, hd, n_pages, form):
    """Pages whose byte offsets pass 2^32: the bits of the same requests in a small cache's pages."""
    nkv, nh, lens = 8, 32, [90, 20]
    big = _cache(cuda, nkv, hd, "e4m3", n_pages=n_pages, page=16, rows=2, max_len=128)  # 4.9e9 bytes a pool
    small = _cache(cuda, nkv, hd, "e4m3", n_pages=20, page=16, rows=2, max_len=128)
    big.free.copy_(torch.arange(n_pages, dtype=torch.int32))  # the last page on top
    x = torch.randn((110, 48 * hd), generator=torch.Generator(device=cuda).manual_seed(1), device=cuda).bfloat16()
    outs = []
    for cache in (big, small):
        m = cache.reserve(lens)
        q = cache.append(0, x, m, n_heads=nh).view(110, nh, hd)
        outs.append((_attend(cache, q, m.rows, m.pos, form), m))
    assert int(outs[0][1].slots.min()) > (n_pages - 10) * 16 and bool(outs[0][0].isfinite().all())
    assert torch.equal(outs[0][0], outs[1][0])


@pytest.mark.parametrize("form", [False, True, "wide"])
@pytest.mark.parametrize("ct", ["i8", "e4m3"])
@pytest.mark.parametrize("hd", [64, 128])
def test_small_query_elements_beside_an_outlier(cuda, ct, form, hd):
    """f32 queries, one element of which is 2^18 times the others and meets zeros in every key, so that
    the scores are the small ones' alone: an element is off by 2^-22 of itself or 2^-39 of the largest,
    a score by that times its keys, scaled (and (hd + 10) 2^-24 of the sum of its products' sizes)."""
    L, nkv, nh = 200, 2, 8
    cache, g = _filled(cuda, nkv, hd, 16, [L], ct, hd)
    codes = cache.k[0].float()
    codes[..., 5] = 0
    cache.k[0] = codes.to(cache.k.dtype)
    scale = 2.0 ** 18 * hd ** -0.5
    q = 2.0 ** -18 * torch.randn((1, nh, hd), generator=g, device=cuda)
    q[..., 5] = 1.7
    if form:
        more = 32768 // nh + 1 if form == "wide" else 0
        rows, pos = _i32(cuda, [0] + [-1] * more), _i32(cuda, [L - 1] + [-1] * more)
        got = cache.attend(0, torch.cat([q, torch.zeros((more, nh, hd), device=cuda)]), rows=rows, pos=pos, scale=scale)[:1]
    else:
        got = cache.attend(0, q, scale=scale)
    p = torch.arange(L, device=cuda)
    ids, at = cache.table[0].long()[p // 16], p % 16
    k, v = ((c[0].float().to(F64) * s[0].to(F64).repeat_interleave(B, -1)[..., None])[ids, :, at].transpose(0, 1).contiguous()
            for c, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)))
    qq = q.to(F64).view(nkv, nh // nkv, hd)
    kt = k.transpose(1, 2).contiguous()
    w = torch.softmax(qq @ kt * scale, -1)
    off = torch.maximum(2.0 ** -22 * qq.abs(), torch.full_like(qq, 2.0 ** -39 * 1.7))
    delta = ((off + (hd + 10) * U32 * qq.abs()) @ kt.abs() * scale).amax(-1, keepdim=True)
    bound = 2 * (2 * delta + (8 + 4 * (L / 16 + 2) + 2 * L) * U32) * (w @ v.abs())
    assert float(delta.max()) < 2.0 ** -9  # (a part that is lost would be 2^-5 and more)
    _close(got, (w @ v).reshape(1, nh, hd), bound.reshape(1, nh, hd), torch.float32)


def _forms(cache, q, rows, pos, form, scale):
    """attend as one token's, or over prefixes in tiles of few or many rows."""
    if not form:
        return cache.attend(0, q, rows=rows, scale=scale)
    more = 32768 // q.shape[1] + 1 if form == "wide" else 0
    none = torch.full((more,), -1, dtype=torch.int32, device=q.device)
    qq = torch.cat([q, torch.zeros((more, *q.shape[1:]), dtype=q.dtype, device=q.device)])
    return cache.attend(0, qq, rows=torch.cat([rows, none]), pos=torch.cat([pos, none]), scale=scale)[:q.shape[0]]


@pytest.mark.parametrize("qt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("form", [False, True, "wide"])
@pytest.mark.parametrize("scale", [-0.3, 0.0, -2.5, 1e-30, 4.0])
def test_scales_of_either_sign(cuda, form, qt, scale):
    lens = [300, 17, 1, 64]
    cache, g = _filled(cuda, 2, 64, 16, lens, "e4m3", 12)
    q = _queries(g, cuda, 4, 6, 64, qt)
    got = _forms(cache, q, _i32(cuda, range(4)), _i32(cuda, [n - 1 for n in lens]), form, scale)
    want, bound = _reference(q, cache, range(4), lens, scale, split=PREFIX_SPLIT[qt] if form else None)
    _close(got, want, bound, DT[qt])


@pytest.mark.parametrize("qt,ct", [("f32", "e4m3"), ("bf16", "i8"), ("f16", "e4m3")])
@pytest.mark.parametrize("nh,nkv,hd", [(300, 2, 64), (130, 1, 128), (257, 1, 32), (129, 1, 256)])
def test_prefix_of_groups_wider_than_a_tile(cuda, qt, ct, nh, nkv, hd):
    """More query heads a KV head than a tile has rows, the last part of a group small."""
    lens = [150, 9, 33]
    cache, g = _filled(cuda, nkv, hd, 32, lens, ct, nh)
    rows, pos = [0] * 40 + [1] * 3 + [2] * 33, list(range(110, 150)) + [6, 7, 8] + list(range(33))
    for n in (76, 3):
        q = _queries(g, cuda, n, nh, hd, qt)
        got = _forms(cache, q, _i32(cuda, rows[:n]), _i32(cuda, pos[:n]), "wide" if n == 76 else True, hd ** -0.5)
        want, bound = _reference(q, cache, rows[:n], [p + 1 for p in pos[:n]], hd ** -0.5, split=PREFIX_SPLIT[qt])
        _close(got, want, bound, DT[qt])


def test_prefix_of_two_hundred_thousand_tiles(cuda):
    """Queries of alternating requests, one of a long one among them, which alone is cut."""
    n, at, hd = 200000, 77777, 16
    lens = [30, 60, 45, 40000]
    cache, g = _filled(cuda, 1, hd, 16, lens, "i8", 3)
    rows = np.arange(n) % 3
    pos = np.random.default_rng(2).integers(0, 60, n)
    rows[at], pos[at] = 3, 39999
    q = _queries(g, cuda, n, 1, hd, "bf16")
    got, (items, cut, pieces) = _prefix_with_plan(cache, q, _i32(cuda, rows.tolist()), _i32(cuda, pos.tolist()))
    assert cut == 1 and pieces >= 2 and items == n - 1 + pieces
    some = [0, 1, 1023, 1024, at - 1, at, at + 1, n - 1] + np.random.default_rng(1).integers(0, n, 300).tolist()
    want, bound = _reference(q[some], cache, rows[some].tolist(), (pos[some] + 1).tolist(), hd ** -0.5, split=PREFIX_SPLIT["bf16"])
    _close(got[some], want, bound, torch.bfloat16)
    assert bool(got.isfinite().all())


@pytest.mark.parametrize("it", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("hd,inter", [(64, False), (80, True), (256, False)])
def test_append_of_rows_at_odd_strides(cuda, it, hd, inter):
    """Rows that begin at any element: the bits of the same rows packed."""
    nh, nkv, T = 3, 2, 70
    width = (nh + 2 * nkv) * hd
    g = torch.Generator(device=cuda).manual_seed(hd)
    wide = torch.randn((T, width + 7), generator=g, device=cuda).to(DT[it])
    rope = tuple(torch.randn((90, hd // 2), generator=g, device=cuda) for _ in range(2))
    w = torch.randn(hd, generator=g, device=cuda)
    outs = []
    for qkv in (wide[:, 3:3 + width], wide[:, 3:3 + width].contiguous()):
        cache = _cache(cuda, nkv, hd, "e4m3", n_pages=8, page=16, rows=1, max_len=90)
        m = cache.reserve([T])
        q = cache.append(0, qkv, m, n_heads=nh, q_norm=w, k_norm=w, rope=rope, interleaved=inter)
        outs.append((q, *cache.read(0, _i32(cuda, [0, T]), T, dtype=torch.float32)))
    assert all(torch.equal(a, b) for a, b in zip(*outs))


@pytest.mark.parametrize("entries,nh", [(3000, 8), (40, 8)])
def test_a_captured_map_whose_tokens_change(cuda, entries, nh):
    """One graph, its map's entries nobody's, one long request's, everybody's in turn: what is cut is
    decided at each replay, and each is the eager call."""
    lens = [9000, 40, 300, 1]
    cache, g = _filled(cuda, 2, 64, 16, lens, "i8", 8)
    rows, pos = _i32(cuda, [-1] * entries), _i32(cuda, [-1] * entries)
    q = _queries(g, cuda, entries, nh, 64, "bf16")
    out = torch.zeros_like(q)
    ws = cache.workspace(entries, nh, prefix=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cache.attend(0, q, rows=rows, pos=pos, out=out, workspace=ws)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.attend(0, q, rows=rows, pos=pos, out=out, workspace=ws)
    rng = np.random.default_rng(entries)
    maps = [([-1] * entries, [-1] * entries), ([0] * 3 + [-1] * (entries - 3), [8997, 8998, 8999] + [-1] * (entries - 3)),
            (rng.integers(-1, 5, entries).tolist(), rng.integers(-1, 9000, entries).tolist()),
            ([2] * entries, (np.arange(entries) % 300).tolist()), ([-1] * (entries - 1) + [0], [0] * (entries - 1) + [8999])]
    for turn, (r, p) in enumerate(maps + maps):
        rows.copy_(_i32(cuda, r))
        pos.copy_(_i32(cuda, p))
        out.fill_(7.0)
        graph.replay()
        if turn % 2:
            torch.cuda.synchronize()
        want = cache.attend(0, q, rows=rows, pos=pos, out=torch.full_like(q, 7.0))
        assert torch.equal(out, want), turn
