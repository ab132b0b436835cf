"""The 8-bit paged cache on the GPU against 64-bit statements of its operators: append (scales and
rescaled codes equal, new codes within half a step), read (equal), attention of one token and over
prefixes (bounds derived from the arithmetic), their edges, and the operators together."""
import math

import numpy as np
import pytest
import torch

from syrinx_amd import SxqError
from syrinx_amd.paged import RELEASE, SCALE_BLOCK, PagedKvCache, SlotMap
from test_gpu_paged import DT, F64, U32, _append_reference, _close, _half_step, _tables

pytestmark = pytest.mark.gpu

CT = {"i8": torch.int8, "e4m3": torch.float8_e4m3fn}
TOP = {"i8": 127.0, "e4m3": 448.0}
B = SCALE_BLOCK


@pytest.fixture(scope="module")
def cuda():
    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a ROCm GPU")
    return torch.device("cuda:0")


# ---- 64-bit statements ----------------------------------------------------------------

def _need(amax, ct):
    """The smallest 2^e, e >= -100, with amax <= TOP 2^e, of f64 amax (exact: powers of two by search)."""
    e = torch.floor(torch.log2(amax.clamp(min=2.0 ** -140) / TOP[ct])) - 1
    for _ in range(4):
        e = torch.where(amax > TOP[ct] * torch.exp2(e), e + 1, e)
    return torch.exp2(e.clamp(min=-100))


def _code_values(x, ct):
    """The nearest values that codes stand for (ties to even, the ends kept) of f64 x."""
    top = TOP[ct]
    x = x.clamp(-top, top)
    if ct == "i8":
        return x.round()
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -30))).clamp(min=-6) - 3)
    return (x / step).round() * step


def _step(x, ct):
    """The distance of codes at the values x (in units of the scale)."""
    if ct == "i8":
        return torch.ones_like(x)
    return torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -30))).clamp(min=-6) - 3)


def _deq(codes, scale):
    """Pages [n_pages, nkv, page, hd] as f64 values."""
    return codes.float().to(F64) * scale.to(F64).repeat_interleave(B, -1)[..., None]


def _cache(cuda, nkv, hd, ct, *, n_pages, page, rows, max_len, layers=1):
    return PagedKvCache(layers, nkv, hd, n_pages=n_pages, page_size=page, max_rows=rows, max_len=max_len, dtype=CT[ct], device=cuda)


def _junk(cache, seed):
    """Codes, and scales that are powers of two, everywhere: a cache in use."""
    g = torch.Generator(device=cache.device).manual_seed(seed)
    for codes, scale in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        x = torch.randn(codes.shape, generator=g, device=cache.device) * (40 if codes.dtype is torch.int8 else 100)
        codes.copy_(x.clamp(-120, 120).round().to(codes.dtype) if codes.dtype is torch.int8 else x.clamp(-440, 440).to(codes.dtype))
        scale.copy_(torch.exp2(torch.randint(-9, -2, scale.shape, generator=g, device=cache.device).float()))


# ---- append ---------------------------------------------------------------------------

def _rows64(qkv, nh, nkv, hd, qn, kn, eps, rope, pos, inter):
    """Normalised and rotated heads in 64 bits, and what f32 arithmetic may be off: a norm's hd products
    summed (halved by the root), the division, + eps, the root, the division and the weight, then two
    products and their sum."""
    want, mag = _append_reference(qkv.contiguous(), nh, nkv, hd, qn, kn, eps, rope, pos, inter)
    return want, (hd / 2 + 9) * U32 * mag


def _check_append(cache, ct, before, x, err, slots, what=""):
    """The pools after an append of the f64 rows x [T, 2 nkv, hd] (each off by at most err) at the
    slots, from the pools `before`: scales, the rescaled earlier codes and everything that no
    token touches equal; new codes within half a step of the value."""
    nkv, page = cache.n_kv_heads, cache.page_size
    slots = [int(s) for s in slots]
    runs, at = [], 0
    while at < len(slots):
        n = 1
        while at + n < len(slots) and slots[at + n] == slots[at] + n and slots[at + n] % B:
            n += 1
        if 0 <= slots[at] < cache.n_pages * page:
            runs.append((at, n))
            at += n
        else:
            at += 1
    for which, codes, scale, (old_c, old_s) in ((0, cache.k[0], cache.k_scale[0], before[0]), (nkv, cache.v[0], cache.v_scale[0], before[1])):
        want_s, keep = old_s.clone(), torch.ones(codes.shape[:3], dtype=torch.bool, device=codes.device)
        got = _deq(codes, scale)
        for t, n in runs:
            pg, o = slots[t] // page, slots[t] % page
            b, k = o // B, o % B
            new, off = x[t:t + n, which:which + nkv].transpose(0, 1), err[t:t + n, which:which + nkv].transpose(0, 1)
            amax, slack = new.abs().amax((1, 2)), off.amax((1, 2))
            lo, hi = _need((amax - slack).clamp(min=0), ct), _need(amax + slack, ct)
            had = old_s[pg, :, b].to(F64)
            if k:
                lo, hi = torch.maximum(lo, had), torch.maximum(hi, had)
            s = scale[pg, :, b].to(F64)
            assert bool(((s == lo) | (s == hi)).all()), f"{what} scales of token {t}: {s} not {lo}"
            want_s[pg, :, b] = scale[pg, :, b]
            # the codes before the run: as they were, times had / s, rounded
            a = b * B
            if k:
                was = _code_values(old_c[pg, :, a:a + k].float().to(F64) * (had / s)[:, None, None], ct)
                assert torch.equal(codes[pg, :, a:a + k].float().to(F64), was), f"{what} earlier codes of token {t}"
            d = (got[pg, :, o:o + n] - new).abs()
            tol = _step((new.abs() + off) / s[:, None, None], ct) / 2 * s[:, None, None] + off
            assert bool((d <= tol).all()), f"{what} token {t}: {float((d / tol).max()):.2f} of the bound"
            keep[pg, :, a:o + n] = False
        assert torch.equal(scale, want_s), what + " other scales"
        assert torch.equal(codes.view(torch.uint8)[keep], old_c.view(torch.uint8)[keep]), what + " other codes"


def _state(cache):
    return [(c[0].clone(), s[0].clone()) for c, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale))]


@pytest.mark.parametrize("it", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("ct", ["i8", "e4m3"])
@pytest.mark.parametrize("nh,nkv,hd,page,norm,inter", [
    (8, 2, 64, 16, True, False), (32, 8, 128, 64, True, True), (3, 1, 16, 32, False, False), (6, 3, 80, 32, True, False),
    (2, 2, 256, 16, False, True), (5, 1, 144, 128, True, False), (4, 4, 32, 16, False, True), (9, 3, 48, 1024, True, True)])
def test_append_codes_scales_and_queries(cuda, it, ct, nh, nkv, hd, page, norm, inter):
    """Prompts from empty, blocks begun in the middle, single tokens, requests that wait, a map longer
    than its tokens; over a cache full of other requests' codes."""
    lens, max_len = [0, 5, 16, 31, 17, 47, 40, 3], 160
    add = [33, 1, 1, 40, 16, 0, 100, 2]
    cache = _cache(cuda, nkv, hd, ct, n_pages=90, page=page, rows=8, max_len=max_len)
    _junk(cache, hd)
    cache.reserve(lens)
    m = cache.reserve(torch.tensor(add, dtype=torch.int32, device=cuda), sum(add) + 3)
    T = sum(add) + 3
    g = torch.Generator(device=cuda).manual_seed(nh + hd)
    wide = torch.randn((T, (nh + 2 * nkv) * hd + 16), generator=g, device=cuda)
    wide *= torch.exp(2 * torch.randn((T, 1), generator=g, device=cuda))  # tokens of unlike sizes
    qkv = wide.to(DT[it])[:, :(nh + 2 * nkv) * hd]
    w = (1 + 0.1 * torch.randn(hd, generator=g, device=cuda)) if norm else None
    tables = _tables(max_len, hd, cuda)
    before = _state(cache)
    out = torch.full((T, nh * hd), 55.0, dtype=DT[it], device=cuda)
    q = cache.append(0, qkv, m, n_heads=nh, q_norm=w, k_norm=w, rope=tables, interleaved=inter, out=out)
    want, err = _rows64(qkv, nh, nkv, hd, w, w, 1e-6, tables, m.pos.long(), inter)
    live = m.slots >= 0
    _close(q.view(T, nh, hd)[live], want[live][:, :nh], err[live][:, :nh], DT[it], "queries")
    assert bool((q[~live] == 55).all())
    _check_append(cache, ct, before, want[:, nh:], err[:, nh:], m.slots.tolist())


@pytest.mark.parametrize("ct", ["i8", "e4m3"])
@pytest.mark.parametrize("T", [1, 2, 5, 47, 600, 2500])
def test_append_of_any_number_of_tokens(cuda, ct, T):
    """Token counts beside the chunks that the work is divided by, blocks begun anywhere."""
    rows = 7
    cache = _cache(cuda, 2, 64, ct, n_pages=260, page=16, rows=rows, max_len=600)
    _junk(cache, T)
    cache.reserve([3, 0, 15, 16, 100, 1, 30])
    add = [T // rows + (r < T % rows) for r in range(rows)]
    m = cache.reserve(add)
    g = torch.Generator(device=cuda).manual_seed(T)
    qkv = torch.randn((T, 8 * 64), generator=g, device=cuda)
    before = _state(cache)
    cache.append(0, qkv, m, n_heads=4)
    want, err = _rows64(qkv, 4, 2, 64, None, None, 1e-6, None, m.pos.long(), False)
    _check_append(cache, ct, before, want[:, 4:], err[:, 4:], m.slots.tolist())


@pytest.mark.parametrize("ct", ["i8", "e4m3"])
def test_append_token_by_token(cuda, ct):
    """Sixteen tokens one at a time, each larger than the last: a block's scale follows, its codes are
    rescaled at each step; for e4m3 what comes of it is what one call gives, but for values that are
    subnormal at the last scale."""
    nkv, hd = 2, 64
    one, many = (_cache(cuda, nkv, hd, ct, n_pages=4, page=32, rows=1, max_len=64) for _ in range(2))
    g = torch.Generator(device=cuda).manual_seed(2)
    x = torch.randn((20, 6 * hd), generator=g, device=cuda) * torch.exp2(torch.arange(20, device=cuda) * 0.7)[:, None]
    one.append(0, x, one.reserve([20]), n_heads=2)
    for t in range(20):
        before, m = _state(many), many.reserve([1])
        many.append(0, x[t:t + 1], m, n_heads=2)
        want, err = _rows64(x[t:t + 1], 2, nkv, hd, None, None, 1e-6, None, m.pos.long(), False)
        _check_append(many, ct, before, want[:, 2:], err[:, 2:], m.slots.tolist(), f"step {t}")
    assert torch.equal(one.k_scale, many.k_scale) and torch.equal(one.v_scale, many.v_scale)
    if ct == "e4m3":
        for a, b, s in ((one.k, many.k, one.k_scale), (one.v, many.v, one.v_scale)):
            a, b = (_deq(c[0], s[0])[:, :, :20] for c in (a, b))
            big = a.abs() >= 2.0 ** -6 * s[0].to(F64).repeat_interleave(B, -1)[:, :, :20, None]
            assert torch.equal(a[big], b[big])


@pytest.mark.parametrize("ct", ["i8", "e4m3"])
@pytest.mark.parametrize("it", ["f32", "bf16", "f16"])
def test_append_again_changes_nothing(cuda, ct, it):
    cache = _cache(cuda, 2, 64, ct, n_pages=20, page=16, rows=3, max_len=90)
    _junk(cache, 1)
    cache.reserve([5, 16, 33])
    m = cache.reserve([20, 1, 7])
    qkv = (3 * torch.randn((28, 8 * 64), generator=torch.Generator(device=cuda).manual_seed(4), device=cuda)).to(DT[it])
    cache.append(0, qkv, m, n_heads=4)
    first = _state(cache)
    cache.append(0, qkv, m, n_heads=4)
    for (c, s), (c1, s1) in zip(_state(cache), first):
        assert torch.equal(c.view(torch.uint8), c1.view(torch.uint8)) and torch.equal(s, s1)


@pytest.mark.parametrize("ct", ["i8", "e4m3"])
def test_append_values_at_the_ends(cuda, ct):
    """Zeros, the largest and smallest f32, subnormals, infinities and NaN, values on a scale's border."""
    nkv, hd, top = 1, 16, TOP[ct]
    cache = _cache(cuda, nkv, hd, ct, n_pages=12, page=16, rows=12, max_len=16)
    inf, nan, big = float("inf"), float("nan"), 3e38  # (beyond 2^128 (1 - 2^-7) a code may stand for infinity in f32)
    rows = [[0.0] * 16, [-0.0] * 16, [1e-40] * 16, [big, -big, 1.0] + [0.0] * 13, [inf, -inf, 2.0, nan] + [-1.0] * 12,
            [nan] * 16, [inf] * 16, [top] + [1.0] * 15, [math.nextafter(top, 1e9) * (1 + 2 ** -20)] + [1.0] * 15,
            [top * 2.0 ** -100, 2.0 ** -101, 3 * 2.0 ** -101] + [0.0] * 13, [-top * 0.5, 0.25, 0.75] + [2.5] * 13, [1.0] * 16]
    k = torch.tensor(rows, device=cuda, dtype=torch.float32)
    m = cache.reserve([1] * 12)
    cache.append(0, torch.cat([k, k, -k], 1), m, n_heads=1)
    got_k, got_v = cache.read(0, torch.arange(13, device=cuda, dtype=torch.int32), 12, dtype=torch.float32)
    got_k, got_v = got_k[:, 0], got_v[:, 0]
    s = cache.k_scale[0, m.slots.long() // 16, 0, 0].tolist()
    e = lambda v: math.frexp(v)[1] - 1  # noqa: E731
    t = 6 if ct == "i8" else 8  # top = (1 + f) 2^t
    assert s[0] == s[1] == s[2] == s[5] == s[6] == 2.0 ** -100
    assert s[3] == 2.0 ** (127 - t + (ct == "e4m3")) and s[4] == 2.0 ** (1 - t) and s[7] == 1.0 and s[8] == 2.0 and s[9] == 2.0 ** -100 and s[10] == 0.5
    assert e(s[11]) == -t
    for got, sign in ((got_k, 1.0), (got_v, -1.0)):
        assert not bool(got[:3].any())
        assert abs(float(got[3, 0]) / (sign * big) - 1) <= 2.0 ** -4 and float(got[3, 2]) == 0
        assert float(got[4, 0]) == sign * top * s[4] and float(got[4, 1]) == -sign * top * s[4] and float(got[4, 2]) == sign * 2.0
        nans = got[5].isnan().all() and got[4, 3].isnan()
        assert bool(nans) if ct == "e4m3" else (not bool(got[5].any()) and float(got[4, 3]) == 0)
        assert bool((got[4, 4:] == -sign).all())
        assert bool((got[6] == sign * top * 2.0 ** -100).all())
        assert float(got[7, 0]) == sign * top and float(got[9, 0]) == sign * top * 2.0 ** -100
        want = _code_values(torch.tensor([0.5, 1.5], dtype=F64), ct) * 2.0 ** -100 * sign  # int8: ties to even
        assert torch.equal(got[9, 1:3].cpu().to(F64), want)
        assert bool((got[11] == sign).all())


def test_append_slots_outside_the_pool_and_runs(cuda):
    """Tokens without a slot between others', a run cut by the page's end, neighbouring slots of two
    requests (one block ends where the other begins)."""
    for ct in ("i8", "e4m3"):
        cache = _cache(cuda, 2, 32, ct, n_pages=6, page=16, rows=1, max_len=16)
        _junk(cache, 9)
        slots = [-1, 14, 15, 16, 17, 2**31 - 1, 34, -2**31, 35, 96, 50, 51, 52, -7]
        qkv = torch.randn((len(slots), 6 * 32), generator=torch.Generator(device=cuda).manual_seed(3), device=cuda)
        sl = torch.tensor(slots, dtype=torch.int32, device=cuda)
        before = _state(cache)
        cache.append(0, qkv, SlotMap(sl, torch.zeros_like(sl), None), n_heads=2)
        want, err = _rows64(qkv, 2, 2, 32, None, None, 1e-6, None, torch.zeros(len(slots), dtype=torch.long, device=cuda), False)
        # (34 and 35 have a token without a slot between them: two runs of one block, which the
        # documentation leaves open; their block is not looked at)
        keep = [s if s not in (34, 35) else -1 for s in slots]
        for (c, s), (bc, bs) in zip(((cache.k[0], cache.k_scale[0]), (cache.v[0], cache.v_scale[0])), before):
            c[2], s[2] = bc[2], bs[2]
        _check_append(cache, ct, before, want[:, 2:], err[:, 2:], keep)


# ---- read -----------------------------------------------------------------------------

@pytest.mark.parametrize("ot", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("ct", ["i8", "e4m3", "f32", "bf16", "f16"])
@pytest.mark.parametrize("nkv,hd,page", [(2, 64, 16), (8, 128, 64), (3, 80, 32), (1, 16, 1024), (5, 256, 16)])
def test_read_ranges(cuda, ot, ct, nkv, hd, page):
    """Ranges in any order, repeated, empty, beyond a request's end and before its first position, of
    requests and pages that are not there; entries behind the last range left alone."""
    lens = [70, 0, 33, 200]
    dt = CT.get(ct, DT.get(ct))
    cache = PagedKvCache(2, nkv, hd, n_pages=60, page_size=page, max_rows=4, max_len=256, dtype=dt, device=cuda)
    cache.reserve(lens)
    g = torch.Generator(device=cuda).manual_seed(hd)
    if ct in CT:
        _junk(cache, 5)
        pools = [_deq(cache.k[1], cache.k_scale[1]), _deq(cache.v[1], cache.v_scale[1])]
    else:
        for p in (cache.k, cache.v):
            p.copy_(torch.randn(p.shape, generator=g, device=cuda))
        pools = [cache.k[1].to(F64), cache.v[1].to(F64)]
    if page == 16:
        cache.table[3, 2], cache.table[3, 3] = -1, cache.n_pages
    rows, start, count = [3, 0, 2, 2, 1, 9, -1, 0, 3, 3], [190, 0, 30, 0, 0, 0, 0, -3, 5, 1 << 30], [30, 70, 10, 0, 2, 3, 1, 5, 100, 2]
    cu = np.concatenate([[0], np.cumsum(count)])
    total = int(cu[-1]) + 5
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda)  # noqa: E731
    buf = [torch.full((total, nkv * hd + 16), 3.0, dtype=DT[ot], device=cuda) for _ in range(2)]
    out = tuple(b.as_strided((total, nkv, hd), (b.stride(0), hd, 1)) for b in buf)
    got = cache.read(1, i32(cu), total, rows=i32(rows), start=i32(start), out=out)
    for t, pool, b in zip(got, pools, buf):
        want = torch.zeros((total, nkv, hd), dtype=F64, device=cuda)
        want[int(cu[-1]):] = 3.0
        for r, s, n, at in zip(rows, start, count, cu):
            for j in range(n):
                p = s + j
                if 0 <= r < 4 and 0 <= p < lens[r]:
                    pg = int(cache.table[r, p // page])
                    if 0 <= pg < cache.n_pages:
                        want[at + j] = pool[pg, :, p % page]
        # equal but for the output's one rounding; codes times powers of two are exact in f32
        assert torch.equal(t, want.to(torch.float32).to(DT[ot]))
        assert bool((b[:, nkv * hd:] == 3).all())
    # fewer entries than the ranges have: the first of them
    k, v = cache.read(1, i32(cu), 17, rows=i32(rows), start=i32(start), dtype=DT[ot])
    assert torch.equal(k, got[0][:17]) and torch.equal(v, got[1][:17])
    # whole requests by default
    k, v = cache.read(1, i32([0, 70, 70, 103]), 103, dtype=DT[ot])
    assert torch.equal(k[:70], got[0][30:100]) and k.shape == (103, nkv, hd)
    assert cache.read(1, i32([0]), 0)[0].shape == (0, nkv, hd)


def test_read_many_ranges(cuda):
    rng = np.random.default_rng(0)
    cache = _cache(cuda, 1, 16, "i8", n_pages=400, page=16, rows=300, max_len=200)
    _junk(cache, 3)
    lens = rng.integers(0, 20, 300)
    cache.reserve([int(n) for n in lens])
    order = rng.permutation(300)
    cu = torch.tensor(np.concatenate([[0], np.cumsum(lens[order])]), dtype=torch.int32, device=cuda)
    rows = torch.tensor(order, dtype=torch.int32, device=cuda)
    k, v = cache.read(0, cu, int(cu[-1]), rows=rows, dtype=torch.float32)
    pool, table = _deq(cache.k[0], cache.k_scale[0]), cache.table.cpu().numpy()
    where = [(r, p) for r in order for p in range(lens[r])]
    ids = torch.tensor([table[r, p // 16] for r, p in where], device=cuda).long()
    off = torch.tensor([p % 16 for _, p in where], device=cuda)
    assert torch.equal(k.to(F64), pool[ids, :, off])


# ---- attention ------------------------------------------------------------------------

def _reference(q, cache, rows, seen, scale, layer=0, split=None):
    """Outputs [n, nh, hd] in 64 bits over positions 0 .. seen[i] - 1 of request rows[i], and each
    element's error bound before the output's rounding, u = 2^-24, S the largest scale sum |q_d k_d| of
    a head: a score is off by (hd + 4) u S (hd products and sums, the scales, which are exact powers
    of two but for `scale` itself), an f32 query's two f16 parts leave out 2^-22 = 4 u of an element (and
    2^-39 of the row's largest, far below that for these queries), a weight is off by twice that
    relative, by |s - m| u <= 2 S u for its argument, 4 u for exp and 4 u for each rescaling; `split`
    is what the weights' parts leave out; sums of len terms len u each."""
    n, nh, hd = q.shape
    nkv, page = cache.n_kv_heads, cache.page_size
    G = nh // nkv
    kp, vp = _deq(cache.k[layer], cache.k_scale[layer]), _deq(cache.v[layer], cache.v_scale[layer])
    out, bound = torch.zeros((n, nh, hd), dtype=F64, device=q.device), torch.zeros((n, nh, hd), dtype=F64, device=q.device)
    table, lens, cells = cache.table.cpu(), cache.lens.tolist(), {}
    if split is None:
        split = 4 * U32 if q.dtype is torch.float32 else 2.0 ** -17  # three bf16 parts, or two
    parts = 4 if q.dtype is torch.float32 else 0
    for i in range(n):
        r = int(rows[i])
        if not 0 <= r < cache.max_rows:
            continue
        if r not in cells:
            p = torch.arange(min(max(lens[r], 0), table.shape[1] * page))
            ids = table[r].long()[p // page]
            ok = (ids >= 0) & (ids < cache.n_pages)
            p, ids = p[ok].to(q.device), ids[ok].to(q.device)
            cells[r] = p, kp[ids, :, p % page].transpose(0, 1).contiguous(), vp[ids, :, p % page].transpose(0, 1).contiguous()
        p, k, v = cells[r]
        L = int((p < seen[i]).sum())
        if L == 0:
            continue
        k, v = k[:, :L], v[:, :L]
        qq = q[i].to(F64).view(nkv, G, hd)
        kt = k.transpose(1, 2).contiguous()
        w = torch.softmax(qq @ kt * scale, -1)
        S = (qq.abs() @ kt.abs() * abs(scale)).amax(-1, keepdim=True)
        rel = 2 * (hd + 4 + parts) * U32 * S + 2 * S * U32 + split + (4 + 4 * (L / 16 + 2) + 2 * L) * U32
        out[i] = (w @ v).reshape(nh, hd)
        bound[i] = (2 * rel * (w @ v.abs())).reshape(nh, hd)
    return out, bound


def _filled(cuda, nkv, hd, page, lens, ct, seed, extra=3, max_len=None):
    """Requests of these lengths in scattered pages; what none holds is NaN where a type has it (scales
    of blocks that no request reaches, e4m3 codes)."""
    g = torch.Generator(device=cuda).manual_seed(seed)
    n_pages = sum(-(-n // page) for n in lens) + extra
    cache = _cache(cuda, nkv, hd, ct, n_pages=n_pages, page=page, rows=len(lens), max_len=max_len or max(1, max(lens)))
    cache.reserve(lens)
    order = torch.randperm(n_pages, generator=g, device=cuda).int()
    cache.table.copy_(torch.where(cache.table >= 0, order[cache.table.clamp(min=0).long()], cache.table))
    held = torch.zeros((n_pages, page), dtype=torch.bool)
    table = cache.table.cpu()
    for r, n in enumerate(lens):
        for b in range(-(-n // page)):
            held[int(table[r, b]), :min(page, n - b * page)] = True
    held = held.to(cuda)
    for codes, scale in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        x = torch.randn(codes.shape[1:], generator=g, device=cuda) * torch.exp(torch.randn((1, nkv, 1, hd), generator=g, device=cuda) / 2)
        x = x.to(F64).view(n_pages, nkv, page // B, B, hd)
        s = _need(x.abs().amax((-2, -1)), ct)
        c = _code_values(x / s[..., None, None], ct).view(n_pages, nkv, page, hd)
        junk = 113.0 if ct == "i8" else float("nan")
        c = torch.where(held[:, None, :, None], c, torch.full_like(c, junk))
        codes[0] = c.float().to(codes.dtype)
        scale[0] = torch.where(held.view(n_pages, 1, page // B, B).any(-1), s.float(), torch.full_like(s.float(), float("nan")))
    return cache, g


TYPES = [(qt, ct) for qt in ("f32", "bf16", "f16") for ct in ("i8", "e4m3")]
EDGES = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 300, 511, 513, 1000]
SHAPES = [(8, 2, 64, 16), (32, 8, 128, 32), (7, 1, 128, 64), (16, 1, 256, 16), (5, 5, 80, 32), (6, 3, 96, 128), (40, 2, 64, 32),
          (3, 1, 16, 16), (33, 1, 48, 1024), (2, 2, 144, 16)]


def _queries(g, cuda, n, nh, hd, qt):
    return (2 * torch.randn((n, nh, hd), generator=g, device=cuda)).to(DT[qt])


@pytest.mark.parametrize("qt,ct", TYPES)
@pytest.mark.parametrize("nh,nkv,hd,page", SHAPES)
def test_attend_lengths_beside_tiles_and_pages(cuda, qt, ct, nh, nkv, hd, page):
    cache, g = _filled(cuda, nkv, hd, page, EDGES, ct, nh * 1000 + hd)
    q = _queries(g, cuda, len(EDGES), nh, hd, qt)
    got = cache.attend(0, q)
    want, bound = _reference(q, cache, range(len(EDGES)), EDGES, hd ** -0.5)
    _close(got, want, bound, DT[qt], f"{nh}/{nkv}x{hd}")
    assert not bool(got[0].any())
    assert torch.equal(cache.attend(0, q), got)  # the same call, the same bits


@pytest.mark.parametrize("qt,ct", TYPES)
@pytest.mark.parametrize("lens,nh,nkv,hd,page", [
    ([9001], 14, 2, 64, 16), ([20000, 3, 0, 777], 32, 8, 128, 32), ([70001], 4, 1, 128, 16), ([4096, 4097], 16, 16, 64, 256),
    ([12345], 48, 2, 96, 64)])
def test_attend_long_caches(cuda, qt, ct, lens, nh, nkv, hd, page):
    cache, g = _filled(cuda, nkv, hd, page, lens, ct, sum(lens))
    q = _queries(g, cuda, len(lens), nh, hd, qt)
    want, bound = _reference(q, cache, range(len(lens)), lens, hd ** -0.5)
    _close(cache.attend(0, q), want, bound, DT[qt])


@pytest.mark.parametrize("ct", ["i8", "e4m3"])
@pytest.mark.parametrize("n,long", [(100, 0), (1300, 20000)])
def test_attend_many_requests(cuda, ct, n, long):
    """Idle, repeated and reordered rows, more of them than a workgroup walks over by itself."""
    rng = np.random.default_rng(n)
    lens = [int(v) for v in np.exp(rng.uniform(0, math.log(300), n))]
    lens[n // 3], lens[n // 2] = max(long, 1), 0
    cache, g = _filled(cuda, 2, 32, 16, lens, ct, n)
    rows = torch.tensor(rng.integers(-1, n, 2 * n), dtype=torch.int32, device=cuda)
    rows[7], rows[11], rows[12] = n // 3, n + 5, n // 2
    q = _queries(g, cuda, 2 * n, 6, 32, "bf16")
    out = torch.full_like(q, 9.0)
    got = cache.attend(0, q, rows=rows, out=out)
    live = (rows >= 0) & (rows < n)
    assert bool((got[~live] == 9).all())
    some = [i for i in [7, 12] + rng.permutation(2 * n)[:300].tolist() if bool(live[i])]
    want, bound = _reference(q[some], cache, rows[some].tolist(), [1 << 30] * len(some), 32 ** -0.5)
    _close(got[some], want, bound, torch.bfloat16)


# Prefix attention: with 16-bit queries a weight is rounded once where its type's output is as coarse
# (bf16: half a step, 2^-8 relative), in two parts for f16.
PREFIX_SPLIT = {"f32": 4 * U32, "f16": 2.0 ** -17, "bf16": 2.0 ** -8}


def _attend(cache, q, rows, pos, form):
    """attend, as one token's (form False), or over prefixes by tiles of few rows (True) or of many, as
    calls of more than 32768 rows of heads take them: entries of no request fill it up."""
    if form != "wide":
        return cache.attend(0, q, rows=rows, pos=pos)
    n, more = q.shape[0], 32768 // q.shape[1] + 1
    none = torch.full((more,), -1, dtype=torch.int32, device=q.device)
    out = torch.full((n + more, *q.shape[1:]), 7.0, dtype=q.dtype, device=q.device)
    cache.attend(0, torch.cat([q, torch.zeros_like(out[n:])]), rows=torch.cat([rows, none]), pos=torch.cat([pos, none]), out=out)
    assert bool((out[n:] == 7).all())
    return out[:n]


def _check_prefix(cache, g, cuda, rows, pos, nh, qt, scale=None, some=None):
    hd, n = cache.head_dim, len(rows)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda)  # noqa: E731
    q = _queries(g, cuda, n, nh, hd, qt)
    out = torch.full_like(q, 7.0)
    got = cache.attend(0, q, rows=i32(rows), pos=i32(pos), scale=scale, out=out)
    some = list(range(n)) if some is None else some
    want, bound = _reference(q[some], cache, [rows[i] for i in some], [max(0, pos[i] + 1) for i in some], scale or hd ** -0.5,
                             split=PREFIX_SPLIT[qt])
    live = torch.tensor([0 <= rows[i] < cache.max_rows for i in some], device=cuda)
    _close(got[some][live], want[live], bound[live], DT[qt], f"{nh}/{cache.n_kv_heads}x{hd}")
    assert bool((got[some][~live] == 7).all())
    assert torch.equal(cache.attend(0, q, rows=i32(rows), pos=i32(pos), scale=scale, out=torch.full_like(q, 7.0)), got)
    if scale is None:
        wide = _attend(cache, q, i32(rows), i32(pos), "wide")
        _close(wide[some][live], want[live], bound[live], DT[qt], f"{nh}/{cache.n_kv_heads}x{hd}, many rows a tile")
    return q, got


@pytest.mark.parametrize("qt,ct", TYPES)
@pytest.mark.parametrize("nh,nkv,hd,page", SHAPES)
def test_prefix_of_maps_as_reserved(cuda, qt, ct, nh, nkv, hd, page):
    """Chunks of several requests after what they hold: none, one token, drafted tokens, lengths beside
    the tiles of queries and of keys; padded entries of the map left alone."""
    before, new = [0, 0, 1, 15, 40, 63, 100, 300, 7], [1, 70, 5, 0, 16, 33, 130, 2, 64]
    cache, g = _filled(cuda, nkv, hd, page, [b + n for b, n in zip(before, new)], ct, hd + nh)
    rows = [r for r, n in enumerate(new) for _ in range(n)] + [-1] * 5
    pos = [b + j for b, n in zip(before, new) for j in range(n)] + [-1] * 5
    _check_prefix(cache, g, cuda, rows, pos, nh, qt)


@pytest.mark.parametrize("qt,ct", TYPES)
def test_prefix_long_chunks_and_few_queries(cuda, qt, ct):
    """One chunk after a long prefix, and single queries and drafts over long caches (split along the
    positions and joined)."""
    rng = np.random.default_rng(5)
    cache, g = _filled(cuda, 2, 64, 32, [5300, 9000, 40], ct, 11)
    rows, pos = [0] * 300 + [1] * 4 + [2] * 2, list(range(5000, 5300)) + [8996, 8997, 8998, 8999] + [3, 39]
    some = [0, 1, 150, 298, 299, 300, 301, 302, 303, 304, 305] + rng.integers(0, 300, 30).tolist()
    _check_prefix(cache, g, cuda, rows, pos, 14, qt, some=some)
    _check_prefix(cache, g, cuda, [1], [8999], 14, qt)
    _check_prefix(cache, g, cuda, [1, 0, 2], [8999, 5299, 39], 6, qt)


@pytest.mark.parametrize("ct", ["i8", "e4m3"])
def test_prefix_maps_in_any_order(cuda, ct):
    """Requests whose queries alternate, positions that fall, repeat, pass the request's length or are
    negative, rows outside the table, a request without positions: each query by itself."""
    rng = np.random.default_rng(6)
    lens = [90, 0, 33, 257]
    cache, g = _filled(cuda, 2, 64, 16, lens, ct, 3)
    rows = [0, 2, 0, 2, 3, 3, 3, 1, -1, 4, 3, 0] + rng.integers(-1, 5, 150).tolist()
    pos = [89, 3, 0, 500, 256, 0, 256, 5, 3, 3, -1, 1 << 30] + rng.integers(-2, 300, 150).tolist()
    _check_prefix(cache, g, cuda, rows, pos, 8, "bf16")
    _check_prefix(cache, g, cuda, sorted(rows), pos, 8, "f32")


@pytest.mark.parametrize("ct", ["i8", "e4m3"])
def test_prefix_of_the_last_token_is_attend(cuda, ct):
    """At the last position both attentions are the same operator, whose arithmetic differs in order only."""
    lens = [1, 17, 64, 200, 1000, 3]
    cache, g = _filled(cuda, 4, 128, 32, lens, ct, 8)
    q, got = _check_prefix(cache, g, cuda, list(range(6)), [n - 1 for n in lens], 16, "f32")
    want, bound = _reference(q, cache, range(6), lens, 128 ** -0.5)
    one = cache.attend(0, q)
    _close(one, want, bound, torch.float32)
    assert float(((one - got).abs().to(F64) - 2 * (bound + U32 * want.abs())).max()) <= 0


@pytest.mark.parametrize("n,nh,nkv,hd", [(2500, 1, 1, 16), (1500, 64, 64, 16), (1100, 16, 16, 128), (2048, 2, 1, 128)])
def test_prefix_of_many_tiles(cuda, n, nh, nkv, hd):
    """Requests that take turns, so that each query is a tile: more of them than stay in LDS, or than are
    cut; one run over a thousand queries among them."""
    lens = [40, 25, 2000]
    cache, g = _filled(cuda, nkv, hd, 16, lens, "e4m3", n)
    rng = np.random.default_rng(n)
    rows, pos = [i % 2 for i in range(n)], rng.integers(0, 40, n).tolist()
    at = n // 2 - 20
    rows[at:at + 40], pos[at:at + 40] = [2] * 40, list(range(1900, 1940))
    some = rng.permutation(n)[:60].tolist() + [0, n - 1, at, at + 39]
    _check_prefix(cache, g, cuda, rows, pos, nh, "bf16", some=some)


@pytest.mark.parametrize("qt,ct", TYPES)
@pytest.mark.parametrize("nh,nkv,hd", [(14, 2, 64), (6, 2, 48), (4, 1, 256)])
def test_prefix_of_few_tiles_in_many_pieces(cuda, qt, ct, nh, nkv, hd):
    """A few queries after a long prefix: a row's pieces are joined by several threads."""
    cache, g = _filled(cuda, nkv, hd, 64, [20000, 50], ct, hd)
    _check_prefix(cache, g, cuda, [0] * 5, list(range(19995, 20000)), nh, qt)
    _check_prefix(cache, g, cuda, [0, 1], [12345, 49], nh, qt)


@pytest.mark.parametrize("n", [3000])
def test_prefix_many_requests(cuda, n):
    rng = np.random.default_rng(n)
    new = rng.integers(0, 4, n)
    before = np.exp(rng.uniform(0, math.log(60), n)).astype(int)
    cache, g = _filled(cuda, 1, 16, 16, [int(v) for v in before + new], "i8", n)
    rows = np.repeat(np.arange(n), new)
    pos = np.concatenate([np.arange(b, b + k) for b, k in zip(before, new)])
    _check_prefix(cache, g, cuda, rows.tolist(), pos.tolist(), 3, "f16", some=rng.permutation(len(rows))[:300].tolist())


@pytest.mark.parametrize("qt,ct", TYPES)
@pytest.mark.parametrize("prefix", [False, True, "wide"])
def test_attention_of_unlike_scales(cuda, qt, ct, prefix):
    """Blocks whose scales lie many powers of two apart, keys and values both; peaked, flat and equal
    scores; a scale near the smallest."""
    L, hd = 700, 64
    cache, g = _filled(cuda, 2, hd, 32, [L, L], ct, 21)
    for scale, lo, hi in ((cache.k_scale, -12, -3), (cache.v_scale, -60, 5)):
        e = torch.randint(lo, hi, scale.shape, generator=g, device=cuda).float()
        scale.copy_(torch.where(scale.isnan(), scale, torch.exp2(e)))
    cache.k[0, :, 1] = torch.ones_like(cache.k[0, :, 1].float()).to(CT[ct])    # flat
    cache.v_scale[0, cache.table[1, :22].long(), 0] = 2.0 ** -100
    q = _queries(g, cuda, 2, 4, hd, qt)
    rows = torch.tensor([0, 1], dtype=torch.int32, device=cuda)
    pos = torch.full((2,), L - 1, dtype=torch.int32, device=cuda) if prefix else None
    got = _attend(cache, q, rows, pos, prefix)
    want, bound = _reference(q, cache, [0, 1], [L, L], hd ** -0.5, split=PREFIX_SPLIT[qt] if prefix else None)
    # (weights below 2^-126 of their largest times a value's scale may be flushed: 2^-120 of that scale's values)
    _close(got, want, bound + 2.0 ** -100, DT[qt])


@pytest.mark.parametrize("prefix", [False, True, "wide"])
def test_attention_of_codes_that_are_nan(cuda, prefix):
    """An e4m3 NaN makes the heads that read it NaN, and no others; past a query's positions, in absent
    pages and behind the length none is reached."""
    lens = [40, 100, 17]
    cache, g = _filled(cuda, 2, 64, 32, lens, "e4m3", 7)
    nan = torch.tensor(float("nan")).to(torch.float8_e4m3fn).to(cuda)
    rows = torch.tensor([0, 1, 2], dtype=torch.int32, device=cuda)
    pos = torch.tensor([n - 1 for n in lens], dtype=torch.int32, device=cuda) if prefix else None
    for qt in ("f32", "bf16", "f16"):
        q = _queries(g, cuda, 3, 4, 64, qt)
        clean = _attend(cache, q, rows, pos, prefix).clone()
        assert bool(clean.isfinite().all())
        t = cache.table.tolist()
        was = cache.k[0, t[1][1], 0, 3, 5].clone(), cache.v[0, t[0][1], 1, 7, 9].clone()
        cache.k[0, t[1][1], 0, 3, 5] = nan
        cache.v[0, t[0][1], 1, 7, 9] = nan  # request 0's last position, column 9
        got = _attend(cache, q, rows, pos, prefix)
        assert bool(got[1, :2].isnan().all()) and torch.equal(got[1, 2:], clean[1, 2:])
        assert torch.equal(got[0, :2], clean[0, :2]) and torch.equal(got[2], clean[2])
        assert bool(got[0, 2:, 9].isnan().all())
        cols = [c for c in range(64) if c != 9]
        assert torch.equal(got[0, 2:][:, cols], clean[0, 2:][:, cols])
        if prefix:  # queries that do not see them, beside others that do
            both = torch.cat([q, q]).view(2, 3, 4, 64).transpose(0, 1).reshape(6, 4, 64).contiguous()
            two = torch.tensor([0, 0, 1, 1, 2, 2], dtype=torch.int32, device=cuda)
            got = _attend(cache, both, two, torch.tensor([38, 39, 34, 99, 16, 16], dtype=torch.int32, device=cuda), prefix)
            assert bool(got[0::2].isfinite().all()) and torch.equal(got[5], clean[2])
            got = _attend(cache, q, rows, torch.tensor([38, 34, 16], dtype=torch.int32, device=cuda), prefix)
            assert bool(got.isfinite().all())
        cache.k[0, t[1][1], 0, 3, 5], cache.v[0, t[0][1], 1, 7, 9] = was


@pytest.mark.parametrize("prefix", [False, True, "wide"])
@pytest.mark.parametrize("ct", ["i8", "e4m3"])
def test_attention_over_absent_pages(cuda, ct, prefix):
    cache, g = _filled(cuda, 2, 64, 16, [200, 33, 64], ct, 11)
    for r, b, bad in ((0, 0, -1), (0, 5, -2**31), (0, 12, 2**31 - 1), (1, 2, cache.n_pages), (2, 0, -7), (2, 1, -7), (2, 2, 1 << 20),
                      (2, 3, -1)):
        cache.table[r, b] = bad
    q = _queries(g, cuda, 3, 4, 64, "bf16")
    rows = torch.arange(3, dtype=torch.int32, device=cuda)
    pos = torch.tensor([199, 32, 63], dtype=torch.int32, device=cuda) if prefix else None
    want, bound = _reference(q, cache, range(3), [200, 33, 64], 0.125, split=PREFIX_SPLIT["bf16"])
    got = _attend(cache, q, rows, pos, prefix)
    _close(got, want, bound, torch.bfloat16)
    assert not bool(got[2].any())
    # lengths outside the table's width: negative is empty, too long its whole width
    cache.lens.copy_(torch.tensor([-3, 2**31 - 1, 64], dtype=torch.int32))
    if prefix:
        got = _attend(cache, q, rows, torch.full_like(pos, 2**31 - 1), prefix)
    else:
        got = cache.attend(0, q, rows=rows)
    assert not bool(got[0].any()) and not bool(got[2].any())


@pytest.mark.parametrize("form", [True, "wide"])
def test_prefix_positions_past_the_end(cuda, form):
    """A position past the request's length, up to the largest there is, sees what the request has."""
    cache, g = _filled(cuda, 2, 64, 32, [77, 300], "i8", 5)
    q = _queries(g, cuda, 4, 4, 64, "f32")
    rows = torch.tensor([0, 0, 1, 1], dtype=torch.int32, device=cuda)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=cuda)  # noqa: E731
    want = _attend(cache, q, rows, i32(76, 76, 299, 299), form)
    assert torch.equal(_attend(cache, q, rows, i32(77, 2**31 - 1, 2**31 - 1, 2**31 - 2), form), want)
    assert not bool(_attend(cache, q, rows, i32(-1, -2**31, -2**31, -1), form).any())


@pytest.mark.parametrize("prefix", [True, "wide"])
def test_prefix_queries_before_a_nan(cuda, prefix):
    """Queries of one tile before and after a NaN key and a NaN value: those that do not see it are as
    without it, the others NaN (of the value: in its column)."""
    cache, g = _filled(cuda, 2, 64, 16, [300], "e4m3", 3)
    nan = torch.tensor(float("nan")).to(torch.float8_e4m3fn).to(cuda)
    rows = torch.zeros(300, dtype=torch.int32, device=cuda)
    pos = torch.arange(300, dtype=torch.int32, device=cuda)
    for qt in ("f32", "bf16", "f16"):
        q = _queries(g, cuda, 300, 4, 64, qt)
        clean = _attend(cache, q, rows, pos, prefix).clone()
        at_v, at_k = int(cache.table[0, 70 // 16]), int(cache.table[0, 200 // 16])
        was = cache.v[0, at_v, 1, 70 % 16, 9].clone(), cache.k[0, at_k, 0, 200 % 16, 0].clone()
        cache.v[0, at_v, 1, 70 % 16, 9] = nan
        cache.k[0, at_k, 0, 200 % 16, 0] = nan
        got = _attend(cache, q, rows, pos, prefix)
        cols = [c for c in range(64) if c != 9]
        assert torch.equal(got[:70], clean[:70]) and torch.equal(got[:200, :2], clean[:200, :2])
        assert bool(got[70:, 2:, 9].isnan().all()) and bool(got[200:, :2].isnan().all())
        want, bound = _reference(q, cache, [0] * 300, list(range(1, 301)), 0.125, split=PREFIX_SPLIT[qt])
        _close(got[70:, 2:][:, :, cols], want[70:, 2:][:, :, cols], bound[70:, 2:][:, :, cols], DT[qt])
        cache.v[0, at_v, 1, 70 % 16, 9], cache.k[0, at_k, 0, 200 % 16, 0] = was


def test_offsets_past_32_bits(cuda):
    """Pages whose byte offsets pass 2^32, written by append and seen by read and both attentions."""
    nkv, hd, page, n_pages = 8, 128, 16, 300000  # 4.9e9 bytes a pool
    cache = _cache(cuda, nkv, hd, "e4m3", n_pages=n_pages, page=page, rows=2, max_len=64)
    cache.free.copy_(torch.arange(n_pages, dtype=torch.int32))  # the last page on top
    m = cache.reserve([50, 20])
    assert int(m.slots.min()) > (n_pages - 10) * page
    g = torch.Generator(device=cuda).manual_seed(1)
    x = torch.randn((70, 48 * hd), generator=g, device=cuda).bfloat16()
    q = cache.append(0, x, m, n_heads=32).view(70, 32, hd)
    k, v = cache.read(0, torch.tensor([0, 50, 70], dtype=torch.int32, device=cuda), 70, dtype=torch.float32)
    kv = x.view(70, 48, hd)[:, 32:].float()
    assert float((k - kv[:, :8]).abs().max()) <= 2.0 ** -4 * 6 and float((v - kv[:, 8:]).abs().max()) <= 2.0 ** -4 * 6
    for r, n, at in ((0, 50, 0), (1, 20, 50)):
        G = 4
        for h in range(nkv):
            qq = q[at + n - 1, h * G:(h + 1) * G].to(F64)
            w = torch.softmax(qq @ k[at:at + n, h].to(F64).t().contiguous() * hd ** -0.5, -1) @ v[at:at + n, h].to(F64)
            rows = torch.tensor([r], dtype=torch.int32, device=cuda)
            for pos in (None, torch.tensor([n - 1], dtype=torch.int32, device=cuda)):
                got = cache.attend(0, q[at + n - 1:at + n].contiguous(), rows=rows, pos=pos)[0, h * G:(h + 1) * G]
                # a weight off by 2^-8, the output's rounding: of values below 6
                assert float((got.to(F64) - w).abs().max()) <= 6 * (2 * 2.0 ** -8 + 2.0 ** -8)


def test_pools_of_other_strides(cuda):
    """Position-major pages, keys and values of one tensor, scales of one tensor, q and out as columns of
    wider rows, through the C-ABI."""
    import ctypes

    from syrinx_amd import lib
    from syrinx_amd._lib import check
    from syrinx_amd.paged import KvPages

    nh, nkv, hd, page, lens, n_pages = 6, 2, 80, 32, [5, 100, 33], 14
    g = torch.Generator(device=cuda).manual_seed(3)
    for ct, code in (("i8", 24), ("e4m3", 0x101)):
        both = torch.zeros((n_pages, page, 2, nkv, hd + 16), dtype=torch.uint8, device=cuda)
        sc = torch.full((n_pages, 2, nkv, page // B + 1), 5.0, device=cuda)
        k, v = both[:, :, 0, :, :hd], both[:, :, 1, :, :hd]
        pages = KvPages(code, nkv, hd, page, n_pages, k.data_ptr(), v.data_ptr(), k.stride(0), k.stride(2), k.stride(1),
                        sc[:, 0].data_ptr(), sc[:, 1].data_ptr(), sc.stride(0), sc.stride(2))
        plain = _cache(cuda, nkv, hd, ct, n_pages=n_pages, page=page, rows=3, max_len=128)
        m = plain.reserve(lens)
        T, width = sum(lens), (nh + 2 * nkv) * hd
        wide = torch.randn((T, width + 8), generator=g, device=cuda).bfloat16()
        q = plain.append(0, wide[:, :width], m, n_heads=nh)
        s = torch.cuda.current_stream().cuda_stream
        check(lib().sxq_kv_append(0, ctypes.byref(pages), 30, wide.data_ptr(), wide.stride(0), T, nh, None, None, 1e-6, None, None, 0, 0,
                                  None, m.slots.data_ptr(), None, s))
        ids, off = m.slots.long() // page, m.slots.long() % page
        for mine, other in ((k, plain.k[0]), (v, plain.v[0])):
            assert torch.equal(mine[ids, off], other.view(torch.uint8)[ids, :, off])
        assert torch.equal(sc[ids, 0][:, :, :2][torch.arange(T, device=cuda), :, off // B], plain.k_scale[0][ids, :, off // B])
        assert bool((both[:, :, :, :, hd:] == 0).all()) and bool((sc[..., -1] == 5).all())
        # attention and read through the same strides
        qw = torch.randn((T, (nh + 4) * hd), generator=g, device=cuda).bfloat16()
        qv = qw.as_strided((T, nh, hd), (qw.stride(0), hd, 1))
        buf = torch.full((T, (nh + 1) * hd), 3.0, device=cuda, dtype=torch.bfloat16)
        size = ctypes.c_size_t()
        check(lib().sxq_kv_prefix_attention_workspace(ctypes.byref(pages), T, nh, ctypes.byref(size)))
        ws = torch.full((size.value,), 0xA5, dtype=torch.uint8, device=cuda)  # (a workspace needs to hold nothing)
        check(lib().sxq_kv_prefix_attention(0, ctypes.byref(pages), 30, qv.data_ptr(), qv.stride(0), T, nh, m.rows.data_ptr(),
                                            m.pos.data_ptr(), plain.lens.data_ptr(), 3, plain.table.data_ptr(), plain.max_blocks,
                                            plain.max_blocks, 0.2, buf.data_ptr(), buf.stride(0), ws.data_ptr(), size.value, s))
        want = plain.attend(0, qv.contiguous(), rows=m.rows, pos=m.pos, scale=0.2)
        assert torch.equal(buf[:, :nh * hd].reshape(T, nh, hd), want) and bool((buf[:, nh * hd:] == 3).all())
        last = [4, 104, 137]
        ql = qw[last].as_strided((3, nh, hd), (qw.stride(0), hd, 1))
        check(lib().sxq_kv_attention_workspace(ctypes.byref(pages), 3, nh, ctypes.byref(size)))
        ws = torch.zeros(size.value, dtype=torch.uint8, device=cuda)
        buf.fill_(3.0)
        check(lib().sxq_kv_attention(0, ctypes.byref(pages), 30, ql.data_ptr(), ql.stride(0), 3, nh, None, plain.lens.data_ptr(), 3,
                                     plain.table.data_ptr(), plain.max_blocks, plain.max_blocks, 0.2, buf.data_ptr(), buf.stride(0),
                                     ws.data_ptr(), size.value, s))
        assert torch.equal(buf[:3, :nh * hd].reshape(3, nh, hd), plain.attend(0, ql.contiguous(), scale=0.2))
        assert bool((buf[:, nh * hd:] == 3).all())


# ---- refusals -------------------------------------------------------------------------

def test_python_refusals(cuda):
    with pytest.raises(SxqError):
        _cache(cuda, 2, 72, "i8", n_pages=4, page=16, rows=2, max_len=64)
    cache = _cache(cuda, 2, 64, "i8", n_pages=4, page=16, rows=2, max_len=64)
    half = PagedKvCache(1, 2, 64, n_pages=4, page_size=16, max_rows=2, max_len=64, dtype=torch.bfloat16, device=cuda)
    q = torch.zeros((2, 4, 64), dtype=torch.bfloat16, device=cuda)
    rows = torch.zeros(2, dtype=torch.int32, device=cuda)
    for c, kw in ((half, dict(rows=rows, pos=rows)), (cache, dict(pos=rows)), (cache, dict(rows=rows, pos=rows[:1])),
                  (cache, dict(rows=rows, pos=rows.long())), (cache, dict(rows=rows, pos=rows.cpu()))):
        with pytest.raises(ValueError):
            c.attend(0, q, **kw)
    with pytest.raises(ValueError):
        cache.attend(0, q.to(torch.float8_e4m3fn))
    with pytest.raises(SxqError):
        cache.attend(0, q, rows=rows, pos=rows, workspace=torch.zeros(256, dtype=torch.uint8, device=cuda)[:0])
    with pytest.raises(ValueError):
        cache.append(0, torch.zeros((2, 8 * 64), device=cuda).to(torch.int8), SlotMap(rows, rows, None), n_heads=4)
    cu = torch.tensor([0, 2], dtype=torch.int32, device=cuda)
    bf = torch.zeros((2, 2, 64), dtype=torch.bfloat16, device=cuda)
    for kw in (dict(cu=cu.long()), dict(cu=cu.cpu()), dict(total=-1), dict(dtype=torch.int8), dict(rows=rows), dict(start=rows[:1].long()),
               dict(out=(bf, bf.float())), dict(out=(bf, bf[:1])), dict(out=(bf.transpose(1, 2), bf.transpose(1, 2))),
               dict(out=(bf.cpu(), bf.cpu())), dict(cu=cu[:0], total=0), dict(layer=1),
               dict(out=(bf, torch.zeros((4, 2, 64), dtype=torch.bfloat16, device=cuda)[::2]))):
        args = dict(layer=0, cu=cu, total=2)
        args.update(kw)
        with pytest.raises(ValueError):
            cache.read(**args)


# ---- the operators together -----------------------------------------------------------

@pytest.mark.parametrize("it", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("ct", ["i8", "e4m3"])
def test_steps_of_ragged_requests(cuda, it, ct):
    """Prompts admitted in chunks, drafts appended, verified and rewound, requests leaving and others in
    their pages: every step's queries over what `read` says that the cache holds, in 64 bits."""
    rows, nh, nkv, hd, page = 6, 8, 2, 64, 16
    cache = _cache(cuda, nkv, hd, ct, n_pages=40, page=page, rows=rows, max_len=120)
    _junk(cache, 2)
    tables = _tables(cache.max_len, hd, cuda, 1e4)
    w = 1 + 0.1 * torch.randn(hd, device=cuda)
    g = torch.Generator(device=cuda).manual_seed(17)
    steps = [[30, 0, 17, 1, 0, 0], [1, 0, 1, 1, 0, 0], [5, 45, 0, 1, 0, 0], [-3, 0, 0, 0, 0, 0], [1, 1, 1, 1, 100, 0],
             [RELEASE, 1, 1, 1, 1, 0], [16, 1, RELEASE, 1, 1, 64], [1, 1, 31, 1, 1, 1], [1, -20, 1, 1, 1, 1], [1, 4, 4, 4, 1, 1]]
    for add in steps:
        m = cache.reserve(add)
        assert not bool(m.status.any())
        T = m.slots.numel()
        if T == 0:
            continue
        qkv = torch.randn((T, (nh + 2 * nkv) * hd), generator=g, device=cuda).to(DT[it])
        before = _state(cache)
        q = cache.append(0, qkv, m, n_heads=nh, q_norm=w, k_norm=w, rope=tables).view(T, nh, hd)
        ref, err = _rows64(qkv, nh, nkv, hd, w, w, 1e-6, tables, m.pos.long(), False)
        _check_append(cache, ct, before, ref[:, nh:], err[:, nh:], m.slots.tolist(), str(add))
        ctx = cache.attend(0, q, rows=m.rows, pos=m.pos)
        lens = cache.lens.tolist()
        cu = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device=cuda)
        k, v = cache.read(0, cu, sum(lens), dtype=torch.float32)
        want, bound = _reference(q, cache, m.rows.tolist(), [p + 1 for p in m.pos.tolist()], hd ** -0.5, split=PREFIX_SPLIT[it])
        _close(ctx, want, bound, DT[it], str(add))
        r, p = m.rows.tolist()[-1], m.pos.tolist()[-1]
        kk, vv = (x[int(cu[r]):int(cu[r]) + p + 1].to(F64) for x in (k, v))
        for h in range(nkv):
            a = torch.softmax(q[-1, 4 * h:4 * h + 4].to(F64) @ kk[:, h].t().contiguous() * hd ** -0.5, -1) @ vv[:, h]
            assert torch.allclose(a, want[-1, 4 * h:4 * h + 4], rtol=1e-9, atol=1e-9)
        last = [int(c) - 1 for c, a in zip(m.cu.tolist()[1:], add) if a > 0]
        want, bound = _reference(q[last], cache, m.rows[last].tolist(), [1 << 30] * len(last), hd ** -0.5)
        _close(cache.attend(0, q[last].contiguous(), rows=m.rows[last].contiguous()), want, bound, DT[it])


def _loop(cache, add, qkv, m, tables, q, out, out1, back, cu, ws):
    cache.reserve(add, out=m)
    cache.append(0, qkv, m, n_heads=8, rope=tables, out=q)
    cache.attend(0, q.view(-1, 8, 64), rows=m.rows, pos=m.pos, out=out, workspace=ws[0])
    cache.attend(0, q.view(-1, 8, 64), rows=m.rows, out=out1, workspace=ws[1])
    cache.read(0, cu, back[0].shape[0], out=back)


@pytest.mark.parametrize("own_ws", [True, False])
@pytest.mark.parametrize("ct", ["i8", "e4m3"])
def test_a_captured_step_replays_with_eager_work_between(cuda, ct, own_ws):
    """All the operators captured at a fixed capacity: the requests that take part change on the GPU;
    every replay equals the eager step on a second cache."""
    rows, cap = 5, 12

    def fresh():
        c = _cache(cuda, 2, 64, ct, n_pages=60, page=16, rows=rows, max_len=400)
        _junk(c, 4)
        c.reserve([300, 3, 17, 0, 90])
        return c

    a, b = fresh(), fresh()
    tables = _tables(400, 64, cuda)
    add = torch.zeros(rows, dtype=torch.int32, device=cuda)
    cu = torch.tensor([0, 100, 120, 160, 160, 200], dtype=torch.int32, device=cuda)
    qkv = torch.zeros((cap, 12 * 64), dtype=torch.bfloat16, device=cuda)
    ma, mb = a.reserve(add, cap), b.reserve(add, cap)
    outs = [[torch.zeros((cap, 8 * 64), dtype=torch.bfloat16, device=cuda)]
            + [torch.zeros((cap, 8, 64), dtype=torch.bfloat16, device=cuda) for _ in range(2)]
            + [tuple(torch.zeros((200, 2, 64), device=cuda) for _ in range(2))] for _ in range(2)]
    ws = (a.workspace(cap, 8, prefix=True), a.workspace(cap, 8)) if own_ws else (None, None)

    def step(cache, m, o, w):
        _loop(cache, add, qkv, m, tables, o[0], o[1], o[2], o[3], cu, w)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(a, ma, outs[0], ws)
        step(b, mb, outs[1], (None, None))
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(a, ma, outs[0], ws)
    g = torch.Generator(device=cuda).manual_seed(8)
    for turn in range(6):
        add.copy_(torch.tensor([[1, 1, 1, 1, 1], [1, 0, 5, 0, 1], [0, 12, 0, 0, 0], [1, 1, RELEASE, 1, 1], [4, 4, 3, 0, -40],
                                [1, 1, 1, 1, 1]][turn], dtype=torch.int32))
        qkv.copy_(torch.randn(qkv.shape, generator=g, device=cuda) * 2.0 ** turn)
        graph.replay()
        step(b, mb, outs[1], (None, None))
        if turn % 2:
            torch.cuda.synchronize()
        other = a.attend(0, outs[0][0].view(-1, 8, 64), rows=ma.rows, pos=ma.pos)  # eager, its own workspace
        live = ma.rows >= 0
        assert torch.equal(other[live], outs[0][1][live]), turn
        for x, y in zip(outs[0][:3] + list(outs[0][3]), outs[1][:3] + list(outs[1][3])):
            assert torch.equal(x, y), turn
        for x, y in zip(_state(a), _state(b)):
            assert torch.equal(x[0].view(torch.uint8), y[0].view(torch.uint8)) and torch.equal(x[1], y[1]), turn


def test_two_graphs_and_two_streams_at_once(cuda):
    """Graphs captured on one stream and replayed on two at once, and eager calls on two streams:
    each has a workspace of its own."""
    cache, g = _filled(cuda, 2, 64, 16, [5000, 3000, 700], "i8", 2)
    rows = torch.tensor([0] * 20 + [1, 2, 2], dtype=torch.int32, device=cuda)
    pos = torch.tensor(list(range(4980, 5000)) + [2999, 698, 699], dtype=torch.int32, device=cuda)
    qs = [_queries(g, cuda, 23, 8, 64, "bf16") for _ in range(2)]

    def both(q, outs=(None, None)):
        return (cache.attend(0, q, rows=rows, pos=pos, out=outs[0]), cache.attend(0, q, rows=rows, out=outs[1]))

    want = [tuple(x.clone() for x in both(q)) for q in qs]
    outs = [(torch.zeros_like(q), torch.zeros_like(q)) for q in qs]
    graphs = []
    for q, o in zip(qs, outs):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            both(q, o)
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert all(torch.equal(x, y) for x, y in zip(o, w))
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(both(qs[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, y) for o in got[i] for x, y in zip(o, want[i]))
