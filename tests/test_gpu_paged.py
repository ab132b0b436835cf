"""The paged key/value cache on the GPU against plain 64-bit statements of the same operators:
page allocation (integers, equal), append and attention (bounds derived from the f32 arithmetic
at each value), their edges, and a decode loop of the three together, eager and captured."""
import ctypes
import math

import numpy as np
import pytest
import torch

from syrinx_amd import SxqError, lib
from syrinx_amd._lib import check
from syrinx_amd.paged import RELEASE, KvPages, PagedKvCache, SlotMap

pytestmark = pytest.mark.gpu

F64 = torch.float64
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
U32 = 2.0 ** -24  # half a step of f32, relative


def _half_step(dtype):
    return torch.finfo(dtype).eps / 2


@pytest.fixture(scope="module")
def cuda():
    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a ROCm GPU")
    return torch.device("cuda:0")


# ---- reserve --------------------------------------------------------------------------

class Pages:
    """The page allocator request by request: what sxq_kv_reserve has to leave behind."""

    def __init__(self, n_rows, width, page, n_pages):
        self.page, self.width = page, width
        self.lens = [0] * n_rows
        self.table = np.full((n_rows, width), -1, np.int64)
        self.free = list(range(n_pages - 1, -1, -1))
        self.count = n_pages

    def blocks(self, n):
        return -(-n // self.page)

    def step(self, add, cap):
        back = []
        for r, a in enumerate(add):
            if a < 0:
                new = max(0, self.lens[r] + a)
                for b in range(self.blocks(new), self.blocks(self.lens[r])):
                    back.append(int(self.table[r, b]))
                    self.table[r, b] = -1
                self.lens[r] = new
        for p in reversed(back):
            self.free[self.count] = p
            self.count += 1
        avail, asked, room = self.count, 0, 0
        cu, status, toks = [0], [], []
        for r, a in enumerate(add):
            st, got = 0, 0
            if a >= 0:
                have, need = self.blocks(self.lens[r]), self.blocks(self.lens[r] + a)
                if self.lens[r] + a > self.width * self.page:
                    st = 2
                else:
                    asked += need - have
                    room += a
                    if need > have and asked > avail:
                        st = 1
                    elif a and room > cap:
                        st = 3
                    else:
                        for b in range(have, need):
                            self.count -= 1
                            self.table[r, b] = self.free[self.count]
                        for p in range(self.lens[r], self.lens[r] + a):
                            toks.append((self.table[r, p // self.page] * self.page + p % self.page, p, r))
                        self.lens[r] += a
                        got = a
            status.append(st)
            cu.append(cu[-1] + got)
        toks += [(-1, -1, -1)] * (cap - len(toks))
        slots, pos, rows = (np.array([t[i] for t in toks], np.int64).reshape(-1) for i in range(3))
        return np.array(cu), slots, pos, rows, np.array(status)


def _same(got, want, what):
    got = got.cpu().numpy()
    assert np.array_equal(got, np.asarray(want)), f"{what}: {got} instead of {want}"


def _check_state(cache, model, what):
    _same(cache.lens, model.lens, what + " lens")
    _same(cache.table, model.table, what + " table")
    _same(cache.free_count, [model.count], what + " free_count")
    _same(cache.free, model.free, what + " free")


def _small_cache(rows, max_len, page, n_pages, **kw):
    return PagedKvCache(1, 1, 8, n_pages=n_pages, page_size=page, max_rows=rows, max_len=max_len, device="cuda:0", **kw)


RESERVE = [(1, 100, 16, 9), (3, 64, 16, 7), (16, 300, 64, 40), (63, 128, 32, 100), (64, 128, 32, 150), (65, 200, 16, 500),
           (500, 90, 16, 1500), (1024, 70, 64, 1100), (1025, 40, 16, 2000), (2500, 60, 32, 3100)]


@pytest.mark.parametrize("rows,max_len,page,n_pages", RESERVE)
def test_reserve_steps_equal_the_sequential_allocator(cuda, rows, max_len, page, n_pages):
    rng = np.random.default_rng(rows)
    cache = _small_cache(rows, max_len, page, n_pages)
    model = Pages(rows, cache.max_blocks, page, n_pages)
    seen = set()
    for step in range(12):
        kind = rng.integers(0, 6, rows)
        add = np.where(kind < 2, 1, np.where(kind == 2, 0, rng.integers(0, max_len, rows)))
        add = np.where(kind == 4, -rng.integers(0, max_len, rows), add)
        add = np.where((kind == 5) & (rng.random(rows) < 0.5), RELEASE if step % 2 else max_len + page + 1, add)
        if step == 7:
            add = np.full(rows, RELEASE)
        if step in (3, 8):
            add = np.ones(rows, np.int64)
        total = int(add[(add > 0) & (add <= max_len)].sum())
        cap = [total + 5, max(0, total // 2), 0][0 if step % 4 else step // 4 % 3]
        m = cache.reserve(torch.tensor(add, dtype=torch.int32, device=cuda), cap)
        cu, slots, pos, rws, status = model.step([int(a) for a in add], cap)
        what = f"step {step}"
        _same(m.cu, cu, what + " cu")
        _same(m.status, status, what + " status")
        for name, want in (("slots", slots), ("pos", pos), ("rows", rws)):
            _same(getattr(m, name), want, f"{what} {name}")
        _check_state(cache, model, what)
        seen |= set(status.tolist())
    assert seen >= {0, 2, 3} and (1 in seen) == (rows in (3, 63, 1024, 2500))  # the rows short of pages


@pytest.mark.parametrize("rows,page", [(16, 64), (300, 16), (1500, 32)])
def test_reserve_of_many_tokens_and_its_exact_inverse(cuda, rows, page):
    cache = _small_cache(rows, 2000, page, rows * (2000 // page + 1))
    model = Pages(rows, cache.max_blocks, page, cache.n_pages)
    rng = np.random.default_rng(page)
    first = rng.integers(0, 900, rows)
    m = cache.reserve(first.tolist())
    want = model.step(first.tolist(), int(first.sum()))
    for name, w in zip(("cu", "slots", "pos", "rows", "status"), want):
        _same(getattr(m, name), w, name)
    before = [t.clone() for t in (cache.lens, cache.table, cache.free, cache.free_count)]
    add = rng.integers(0, 1000, rows)
    add[::3] = -np.minimum(first[::3], rng.integers(0, 900, len(first[::3])))
    cap = int(add[add > 0].sum()) + 3
    cache.reserve(torch.tensor(add, dtype=torch.int32, device=cuda), cap)
    cache.reserve(torch.tensor(-add, dtype=torch.int32, device=cuda), int(-add[add < 0].sum()))
    live = int(before[3])
    for name, t, b in zip(("lens", "table", "free", "free_count"), (cache.lens, cache.table, cache.free, cache.free_count),
                          before):
        if name == "free":
            t, b = t[:live], b[:live]
        assert torch.equal(t, b), name


def test_reserve_reads_no_index_it_has_not_checked(cuda):
    """Lengths, page ids and the free count outside their ranges: nothing is read or written out
    of bounds (guard elements around every array keep their values), ids that are no page give
    slot -1."""
    rows, width, page, n_pages = 5, 4, 16, 6
    guard = 64

    def guarded(values):
        t = torch.full((len(values) + 2 * guard,), 77, dtype=torch.int32, device=cuda)
        t[guard:-guard] = torch.tensor(values, dtype=torch.int32)
        return t, t[guard:-guard]

    names = {
        "add": [1, 1, RELEASE, 3, 1], "lens": [-5, 1 << 30, 2**31 - 1, 15, 63],
        "table": [-1] * width + [99] * width + [2**31 - 1] * width + [-7, 3, -1, -1] + [0, 1, 2, 12345],
        "free": [4, -9, 88, 1, 0, 2], "count": [1 << 20], "cu": [0] * (rows + 1), "slots": [0] * 8, "pos": [0] * 8,
        "rows": [0] * 8, "status": [0] * rows,
    }
    whole, part = {}, {}
    for k, v in names.items():
        whole[k], part[k] = guarded(v)
    p = {k: ctypes.c_void_p(t.data_ptr()) for k, t in part.items()}
    check(lib().sxq_kv_reserve(0, page, n_pages, rows, width, p["add"], p["lens"], p["table"], width, p["free"], p["count"],
                               8, p["cu"], p["slots"], p["pos"], p["rows"], p["status"],
                               torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    for k, t in whole.items():
        assert bool((t[:guard] == 77).all()) and bool((t[-guard:] == 77).all()), k
    assert part["lens"].tolist() == [1, 64, 0, 18, 64]
    assert part["status"].tolist() == [0, 2, 0, 0, 0]
    slots = part["slots"].tolist()
    assert all(s == -1 or 0 <= s < n_pages * page for s in slots) and part["cu"].tolist() == [0, 1, 1, 1, 4, 5]
    assert slots[1] == -1 and slots[4] == -1  # the pages of lengths 15 and 63 are ids -7 and 12345


@pytest.mark.parametrize("rows,cap", [(70, 100), (300, 5000), (1500, 9000)])
def test_reserve_of_a_corrupted_state_stays_inside_its_arrays(cuda, rows, cap):
    """Any lengths, page ids, free pages and free count, through every way the call is split into
    launches: guard elements keep their values, slots lie in the pool or are -1."""
    width, page, n_pages, guard = 7, 16, 400, 256
    rng = np.random.default_rng(rows)
    bad = np.array([-2**31, -7, -1, 0, 3, 90, 112, 113, 400, 5000, 2**31 - 1])

    def guarded(n, values=None):
        t = torch.full((n + 2 * guard,), 77, dtype=torch.int32, device=cuda)
        if values is not None:
            t[guard:guard + n] = torch.from_numpy(values.astype(np.int32)).to(cuda)
        return t, t[guard:guard + n]

    for count in (2**31 - 1, 350, -5):
        arrays = {
            "add": guarded(rows, rng.choice([1, 1, 5, 60, 112, -3, -2**31, 2**31 - 1], rows)),
            "lens": guarded(rows, rng.choice(bad, rows)), "table": guarded(rows * width, rng.choice(bad, rows * width)),
            "free": guarded(n_pages, rng.choice(bad, n_pages)), "count": guarded(1, np.array([count])),
            "cu": guarded(rows + 1), "slots": guarded(cap), "pos": guarded(cap), "rows": guarded(cap), "status": guarded(rows)}
        p = {k: ctypes.c_void_p(v[1].data_ptr()) for k, v in arrays.items()}
        check(lib().sxq_kv_reserve(0, page, n_pages, rows, width, p["add"], p["lens"], p["table"], width, p["free"],
                                   p["count"], cap, p["cu"], p["slots"], p["pos"], p["rows"], p["status"],
                                   torch.cuda.current_stream().cuda_stream))
        torch.cuda.synchronize()
        for k, (whole, _) in arrays.items():
            assert bool((whole[:guard] == 77).all()) and bool((whole[-guard:] == 77).all()), k
        got = {k: v[1].cpu().numpy() for k, v in arrays.items()}
        assert ((got["lens"] >= 0) & (got["lens"] <= width * page)).all() and 0 <= got["count"][0] <= n_pages
        assert ((got["slots"] >= -1) & (got["slots"] < n_pages * page)).all() and got["cu"][-1] <= cap
        assert (np.diff(got["cu"]) >= 0).all() and (got["rows"][got["cu"][-1]:] == -1).all()


def test_reserve_python_refusals(cuda):
    cache = _small_cache(4, 64, 16, 8)
    with pytest.raises(ValueError):
        cache.reserve([1] * 5)
    with pytest.raises(ValueError):
        cache.reserve(torch.zeros(4, dtype=torch.int32, device=cuda))  # no capacity
    with pytest.raises(ValueError):
        cache.reserve(torch.zeros(4, dtype=torch.int64, device=cuda), 4)
    with pytest.raises(ValueError):
        cache.reserve(torch.zeros(3, dtype=torch.int32, device=cuda), 4)
    with pytest.raises(ValueError):
        cache.reserve(torch.zeros(4, dtype=torch.int32), 4)
    with pytest.raises(ValueError):
        cache.reserve([1], -1)
    m = cache.reserve([1, 2], 6)
    with pytest.raises(ValueError):
        cache.reserve([1], 5, out=m)
    with pytest.raises(ValueError):
        cache.reserve([1], out=SlotMap(m.slots, m.pos, m.rows))
    assert cache.reserve([1], out=m) is m and cache.lens.tolist() == [2, 2, 0, 0]


# ---- append ---------------------------------------------------------------------------

def _append_reference(x, nh, nkv, hd, qn, kn, eps, rope, pos, interleaved):
    """Roped heads [T, nh + 2 nkv, hd] in 64 bits and, per element, the magnitude that the f32
    arithmetic's error is relative to (|a c| + |b s| of the normalised pair)."""
    h = x.to(F64).view(-1, nh + 2 * nkv, hd)
    for w, sl in ((qn, slice(0, nh)), (kn, slice(nh, nh + nkv))):
        if w is not None:
            part = h[:, sl]
            h = h.clone()
            h[:, sl] = part / torch.sqrt(part.square().mean(-1, keepdim=True) + eps) * w.to(F64)
    mag = h.abs()
    if rope is not None:
        c, s = (t.to(F64)[pos][:, None] for t in rope)
        rot, r = h[:, :nh + nkv], h.clone()
        mag = mag.clone()
        ia, ib = (slice(0, None, 2), slice(1, None, 2)) if interleaved else (slice(0, hd // 2), slice(hd // 2, None))
        a, b = rot[..., ia], rot[..., ib]
        r[:, :nh + nkv, ia], r[:, :nh + nkv, ib] = a * c - b * s, b * c + a * s
        mag[:, :nh + nkv, ia], mag[:, :nh + nkv, ib] = (a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()
        h = r
    return h, mag


def _tables(n, hd, dev, theta=1e6):
    ang = torch.arange(n, dtype=F64)[:, None] * theta ** (-2.0 * torch.arange(hd // 2, dtype=F64) / hd)
    return ang.cos().float().to(dev), ang.sin().float().to(dev)


APPEND = [
    # T, nh, nkv, hd, page, in, cache, norms, rope, interleaved, padding of the row
    (1, 14, 2, 64, 16, "f32", "f32", "", True, False, 0),
    (5, 32, 8, 128, 64, "f32", "bf16", "qk", True, True, 0),
    (37, 4, 4, 80, 16, "f16", "f16", "qk", True, False, 8),
    (64, 6, 3, 96, 32, "bf16", "bf16", "k", True, True, 0),
    (19, 7, 1, 256, 128, "bf16", "f32", "q", True, False, 24),
    (3, 2, 2, 8, 16, "f32", "f16", "qk", True, True, 1),
    (33, 5, 5, 24, 16, "f16", "bf16", "", False, False, 0),
    (300, 16, 2, 64, 32, "bf16", "f16", "qk", False, False, 0),
    (130, 3, 1, 40, 1024, "f32", "f32", "qk", True, False, 3),
    (4097, 8, 2, 64, 16, "bf16", "bf16", "qk", True, True, 0),
    (1, 1, 1, 248, 16, "f16", "f32", "qk", True, True, 5),
]


@pytest.mark.parametrize("T,nh,nkv,hd,page,it,ct,norms,rope,inter,pad", APPEND)
def test_append_against_64_bits(cuda, T, nh, nkv, hd, page, it, ct, norms, rope, inter, pad):
    g = torch.Generator(device=cuda).manual_seed(T * 131 + hd)
    n_pages, width, eps = -(-T // page) + 3, (nh + 2 * nkv) * hd, 1e-5
    cache = PagedKvCache(2, nkv, hd, n_pages=n_pages, page_size=page, max_rows=1, max_len=page, dtype=DT[ct], device=cuda)
    for pool in (cache.k, cache.v):
        pool.copy_(torch.randn(pool.shape, generator=g, device=cuda))
    k0, v0 = cache.k.clone(), cache.v.clone()
    qkv = (torch.randn((T, width + pad), generator=g, device=cuda) * 1.7).to(DT[it])[:, :width]
    top = 500
    pos = torch.randint(0, top, (T,), generator=g, device=cuda).int()
    slots = torch.randperm(n_pages * page, generator=g, device=cuda)[:T].int()
    drop = torch.arange(T, device=cuda) % 7 == 3
    slots[drop] = torch.tensor([-1, n_pages * page, 2**31 - 1, -2**31], dtype=torch.int32,
                               device=cuda).repeat(T)[:int(drop.sum())]
    qn, kn = ((1 + 0.2 * torch.randn(hd, generator=g, device=cuda)) if c in norms else None for c in "qk")
    tables = _tables(top, hd, cuda) if rope else None
    out = torch.full((T, nh * hd), 55.0, dtype=DT[it], device=cuda)
    got = cache.append(1, qkv, SlotMap(slots, pos, None), n_heads=nh, q_norm=qn, k_norm=kn, eps=eps, rope=tables,
                       interleaved=inter, out=out)
    assert got.data_ptr() == out.data_ptr()
    want, mag = _append_reference(qkv.contiguous(), nh, nkv, hd, qn, kn, eps, tables, pos.long(), inter)
    # the norm: hd products summed (each sum rounded at most hd times over, halved by the
    # square root), the division by hd, + eps, the root, the division and the weight; the
    # rotation: two products and their sum
    rel = (hd / 2 + 9) * U32

    def close(a, w, m, dt, what):
        bound = rel * m + _half_step(dt) * (w.abs() + rel * m) + torch.finfo(dt).smallest_normal * torch.finfo(dt).eps
        bad = (a.to(F64) - w).abs() > bound
        assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} beyond the bound"

    live = ~drop
    close(out[live].view(-1, nh, hd), want[live, :nh], mag[live, :nh], DT[it], "q")
    assert bool((out[drop] == 55).all())
    flat = slots[live].long()
    touched = torch.zeros(n_pages * page, dtype=torch.bool, device=cuda)
    touched[flat] = True
    for pool, old, lo, what in ((cache.k, k0, nh, "k"), (cache.v, v0, nh + nkv, "v")):
        assert torch.equal(pool[0], old[0])
        rows = pool[1].transpose(1, 2).reshape(-1, nkv, hd)  # by slot
        close(rows[flat], want[live, lo:lo + nkv], mag[live, lo:lo + nkv], DT[ct], what)
        assert torch.equal(rows[~touched], old[1].transpose(1, 2).reshape(-1, nkv, hd)[~touched]), what


def test_append_rows_of_any_values(cuda):
    """A zero row under a norm stays zero, infinities and NaN stay in their own head, positions
    outside the tables take the nearest row."""
    nh, nkv, hd = 2, 1, 64
    cache = PagedKvCache(1, nkv, hd, n_pages=2, page_size=16, max_rows=1, max_len=16, dtype=torch.float32, device=cuda)
    x = torch.randn((5, 4, hd), device=cuda)
    x[0] = 0
    x[1, 0, 5] = float("inf")
    x[2, 2, 7] = float("nan")
    w = torch.ones(hd, device=cuda)
    tables = _tables(10, hd, cuda)
    pos = torch.tensor([3, 3, 3, 99, -4], dtype=torch.int32, device=cuda)
    m = SlotMap(torch.arange(5, dtype=torch.int32, device=cuda), pos, None)
    q = cache.append(0, x.view(5, -1), m, n_heads=nh, q_norm=w, k_norm=w, rope=tables).view(5, nh, hd)
    k, v = cache.k[0, 0, 0, :5], cache.v[0, 0, 0, :5]
    assert not bool(q[0].any()) and not bool(k[0].any()) and not bool(v[0].any())
    assert bool(q[1, 0].isnan().any()) and bool(q[1, 1].isfinite().all()) and bool(k[1].isfinite().all())
    assert bool(k[2].isnan().all()) and bool(q[2].isfinite().all()) and bool(v[2].isfinite().all())
    want, mag = _append_reference(x[3:].reshape(2, -1), nh, nkv, hd, w, w, 1e-6, tables,
                                  torch.tensor([9, 0], device=cuda), False)
    assert bool(((q[3:].to(F64) - want[:, :2]).abs() <= (hd / 2 + 10) * U32 * mag[:, :2]).all())


def test_append_python_refusals(cuda):
    cache = PagedKvCache(1, 2, 64, n_pages=4, page_size=16, max_rows=1, max_len=64, dtype=torch.bfloat16, device=cuda)
    m = cache.reserve([3])
    x = torch.zeros((3, 8 * 64), device=cuda)
    ok = dict(n_heads=4)
    bad = [(dict(layer=1), ok), (dict(qkv=x.cpu()), ok), (dict(qkv=x[:, :-1]), ok), (dict(qkv=x.double()), ok),
           (dict(qkv=torch.zeros((4, 512), device=cuda)), ok),  # more tokens than the map
           (dict(qkv=x.t().contiguous().t()), ok), (dict(qkv=x[:1].expand(3, 512)), ok),
           (dict(), dict(n_heads=4, q_norm=torch.ones(32, device=cuda))),
           (dict(), dict(n_heads=4, k_norm=torch.ones(64, device=cuda).half())),
           (dict(), dict(n_heads=4, rope=(torch.ones(8, 64, device=cuda),) * 2)),
           (dict(), dict(n_heads=4, rope=(torch.ones(8, 32, device=cuda), torch.ones(9, 32, device=cuda)))),
           (dict(), dict(n_heads=4, out=torch.zeros((3, 255), device=cuda))),
           (dict(), dict(n_heads=4, out=torch.zeros((3, 256), device=cuda).half())),
           (dict(slot_map=SlotMap(m.slots.long(), m.pos, None)), ok)]
    for pos_kw, kw in bad:
        args = dict(layer=0, qkv=x, slot_map=m)
        args.update(pos_kw)
        with pytest.raises(ValueError):
            cache.append(args["layer"], args["qkv"], args["slot_map"], **kw)


# ---- attend ---------------------------------------------------------------------------

def _attend_reference(q, k_pool, v_pool, table, lens, rows, scale):
    """Outputs [n, nh, hd] in 64 bits, and an element's error bound of f32 arithmetic (before
    the output's rounding).  With u = 2^-24 and, per head, S = max_j scale sum_d |q_d k_jd|: a
    score is off by (hd + 3) u S (hd products and sums, the scale; splitting f32 into 16-bit
    parts adds less than u per product), so a weight exp(s_j - m) by twice that relative, plus
    the argument's own rounding |s_j - m| u <= 2 S u and 4 u for exp and its rescaling at each
    of the ceil(len / 16) tiles and at the join; a weight carried in two f16 parts, or three of
    bf16, is off by 4 u (2^-22), in two bf16 parts (bf16 queries) by 2^-18.  Weighted and plain
    sums of len terms: len u each."""
    n, nh, hd = q.shape
    split = 2.0 ** -18 if q.dtype == torch.bfloat16 else 4 * U32
    page, nkv = k_pool.shape[2], k_pool.shape[1]
    out, bound = torch.zeros((n, nh, hd), dtype=F64, device=q.device), torch.zeros((n, nh, hd), dtype=F64, device=q.device)
    for i in range(n):
        r = int(rows[i])
        if not 0 <= r < table.shape[0]:
            continue
        L = min(max(int(lens[r]), 0), table.shape[1] * page)
        p = torch.arange(L, device=q.device)
        ids = table[r].long()[p // page]
        p = p[(ids >= 0) & (ids < k_pool.shape[0])]
        if p.numel() == 0:
            continue
        ids = table[r].long()[p // page]
        G = nh // nkv
        for h in range(nkv):
            k, v = k_pool[ids, h, p % page].to(F64), v_pool[ids, h, p % page].to(F64)
            qq = q[i, h * G:(h + 1) * G].to(F64)
            s = (qq @ k.t().contiguous()) * scale
            w = torch.softmax(s, -1)
            S = ((qq.abs() @ k.abs().t().contiguous()) * abs(scale)).amax(-1, keepdim=True)
            out[i, h * G:(h + 1) * G] = w @ v
            rel = 2 * (hd + 3) * U32 * S + 2 * S * U32 + split + (4 + 4 * (L / 16 + 2) + 2 * L) * U32
            bound[i, h * G:(h + 1) * G] = 2 * rel * (w @ v.abs())
    return out, bound


def _filled(cuda, nkv, hd, page, lens, dt, seed, extra=3, layers=1, layer=0, max_len=None):
    g = torch.Generator(device=cuda).manual_seed(seed)
    max_len = max_len or max(1, max(lens))
    n_pages = sum(-(-n // page) for n in lens) + extra
    cache = PagedKvCache(layers, nkv, hd, n_pages=n_pages, page_size=page, max_rows=len(lens), max_len=max_len, dtype=DT[dt],
                         device=cuda)
    cache.k.fill_(float("nan"))  # what no request holds must not matter
    cache.v.fill_(float("nan"))
    order = torch.randperm(n_pages, generator=g, device=cuda).int()
    at = 0
    for r, n in enumerate(lens):
        b = -(-n // page)
        cache.table[r, :b] = order[at:at + b]
        for j in range(b):
            m = min(page, n - j * page)
            for pool in (cache.k, cache.v):
                pool[layer, int(order[at + j]), :, :m] = torch.randn((nkv, m, hd), generator=g, device=cuda).to(DT[dt])
        at += b
    cache.lens.copy_(torch.tensor(lens, dtype=torch.int32))
    return cache, g


def _close(got, want, bound, dt, what=""):
    tol = bound + _half_step(dt) * (want.abs() + bound) + torch.finfo(dt).smallest_normal * torch.finfo(dt).eps
    err = (got.to(F64) - want).abs()
    bad = ~(err <= tol)
    assert not bool(bad.any()), f"{what} {int(bad.sum())} of {bad.numel()} beyond the bound, worst {float((err / tol).max()):.2f}"


TYPES = [("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16"), ("f16", "f16")]
EDGES = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 300, 511, 513, 1000]


@pytest.mark.parametrize("qt,ct", TYPES)
@pytest.mark.parametrize("nh,nkv,hd,page", [(8, 2, 64, 16), (32, 8, 128, 32), (7, 1, 128, 64), (16, 1, 256, 16), (5, 5, 80, 32),
                                            (6, 3, 96, 128), (40, 2, 64, 32), (3, 1, 8, 16), (33, 1, 40, 1024), (2, 2, 136, 16)])
def test_attend_lengths_beside_tiles_and_pages(cuda, qt, ct, nh, nkv, hd, page):
    cache, g = _filled(cuda, nkv, hd, page, EDGES, ct, nh * 1000 + hd)
    q = (2 * torch.randn((len(EDGES), nh, hd), generator=g, device=cuda)).to(DT[qt])
    got = cache.attend(0, q)
    want, bound = _attend_reference(q, cache.k[0], cache.v[0], cache.table, cache.lens, range(len(EDGES)), hd ** -0.5)
    _close(got, want, bound, DT[qt], f"{nh}/{nkv}x{hd}")
    assert not bool(got[0].any())
    assert torch.equal(cache.attend(0, q), got)  # the same call, the same bits


@pytest.mark.parametrize("qt,ct", TYPES)
@pytest.mark.parametrize("lens,nh,nkv,hd,page", [
    ([9001], 14, 2, 64, 16), ([20000, 3, 0, 777], 32, 8, 128, 32), ([70001], 4, 1, 128, 16), ([4096, 4097], 16, 16, 64, 256),
    ([12345], 48, 2, 96, 64)])
def test_attend_long_caches(cuda, qt, ct, lens, nh, nkv, hd, page):
    cache, g = _filled(cuda, nkv, hd, page, lens, ct, sum(lens))
    q = (2 * torch.randn((len(lens), nh, hd), generator=g, device=cuda)).to(DT[qt])
    want, bound = _attend_reference(q, cache.k[0], cache.v[0], cache.table, cache.lens, range(len(lens)), hd ** -0.5)
    _close(cache.attend(0, q), want, bound, DT[qt])


def test_attend_more_heads_than_the_card_has_places(cuda):
    """900 KV heads of 18 query heads (two tiles of 16 each): more workgroups a piece than split
    queries have counters for."""
    cache, g = _filled(cuda, 900, 8, 16, [1500, 400, 0, 33], "bf16", 12)
    q = torch.randn((4, 900 * 18, 8), generator=g, device=cuda).bfloat16()
    want, bound = _attend_reference(q, cache.k[0], cache.v[0], cache.table, cache.lens, range(4), 8 ** -0.5)
    for _ in range(2):
        _close(cache.attend(0, q), want, bound, torch.bfloat16)


@pytest.mark.parametrize("n,long", [(129, 0), (1025, 40000), (2600, 9000)])
def test_attend_thousands_of_queries(cuda, n, long):
    """More queries than a workgroup walks over by itself, one of them far longer than the rest,
    idle and repeated rows; twice, the second time on another order."""
    rng = np.random.default_rng(n)
    lens = [int(v) for v in np.exp(rng.uniform(0, math.log(90), n))]
    lens[n // 3] = max(long, 1)
    lens[n // 2] = 0
    cache, g = _filled(cuda, 1, 16, 16, lens, "bf16", n)
    for turn in range(2):
        rows = torch.tensor(rng.integers(-1, n, 2 * n), dtype=torch.int32, device=cuda)
        rows[7] = n // 3
        rows[11] = n + 5
        q = torch.randn((2 * n, 3, 16), generator=g, device=cuda).bfloat16()
        out = torch.full_like(q, 9.0)
        got = cache.attend(0, q, rows=rows, out=out)
        live = (rows >= 0) & (rows < n)
        assert bool((got[~live] == 9).all())
        some = torch.cat([torch.tensor([7]), torch.from_numpy(rng.permutation(2 * n)[:400])])
        some = some[live[some.to(cuda)].cpu()]
        want, bound = _attend_reference(q[some], cache.k[0], cache.v[0], cache.table, cache.lens, rows[some].tolist(), 0.25)
        _close(got[some], want, bound, torch.bfloat16)
        few = some[:40]  # the same queries in a call of their own
        _close(cache.attend(0, q[few].contiguous(), rows=rows[few].contiguous()), want[:40], bound[:40], torch.bfloat16)


@pytest.mark.parametrize("n", [100, 300])
def test_attend_many_requests(cuda, n):
    rng = np.random.default_rng(n)
    lens = [int(v) for v in np.exp(rng.uniform(0, math.log(700), n))]
    cache, g = _filled(cuda, 2, 64, 16, lens, "bf16", n)
    q = torch.randn((n, 8, 64), generator=g, device=cuda).bfloat16()
    rows = torch.tensor(rng.integers(-1, n, 2 * n), dtype=torch.int32, device=cuda)  # repeated, reordered, idle
    qq = torch.cat([q, q])
    out = torch.full_like(qq, 9.0)
    got = cache.attend(0, qq, rows=rows, out=out)
    want, bound = _attend_reference(qq, cache.k[0], cache.v[0], cache.table, cache.lens, rows.tolist(), 0.125)
    live = rows >= 0
    _close(got[live], want[live], bound[live], torch.bfloat16)
    assert bool((got[~live] == 9).all())


def test_attend_peaked_and_flat_rows(cuda):
    """Scores of hundreds apart (all but one weight underflow), equal scores, and a running
    maximum that rises at every position."""
    L, hd = 3000, 64
    for ct in ("f32", "bf16", "f16"):
        cache, g = _filled(cuda, 3, hd, 16, [L], ct, 5)
        k = torch.zeros((3, L, hd), device=cuda)
        k[0, :, 0] = torch.arange(L, device=cuda) * 0.25 - 300
        k[1] = 1.0
        k[2, 1234, 3] = 200.0
        ids = cache.table[0].long()[torch.arange(L, device=cuda) // 16]
        cache.k[0, ids, :, torch.arange(L, device=cuda) % 16] = k.transpose(0, 1).to(DT[ct])
        q = torch.zeros((1, 3, hd), device=cuda, dtype=DT[ct])
        q[0, 0, 0], q[0, 1], q[0, 2, 3] = 8.0, 1.0, 16.0
        want, bound = _attend_reference(q, cache.k[0], cache.v[0], cache.table, cache.lens, [0], 1.0)
        _close(cache.attend(0, q, scale=1.0), want, bound, DT[ct], ct)


def test_attend_values_that_are_not_finite(cuda):
    """A NaN or infinity makes the heads that read it not finite, and no other; one behind the length, in
    an absent page or in a page's unused end reaches none."""
    lens = [40, 100, 17]
    for ct in ("f32", "bf16", "f16"):
        cache, g = _filled(cuda, 2, 64, 32, lens, ct, 7)  # unused positions are NaN already
        q = torch.randn((3, 4, 64), generator=g, device=cuda).to(DT[ct])
        clean = cache.attend(0, q).clone()
        assert bool(clean.isfinite().all())
        t = cache.table.tolist()
        cache.k[0, t[1][1], 0, 3, 5] = float("nan")     # request 1, KV head 0
        cache.v[0, t[0][1], 1, 7, 9] = float("inf")     # request 0, KV head 1, position 39 (the last), column 9
        got = cache.attend(0, q)
        assert bool(got[1, :2].isnan().all()) and torch.equal(got[1, 2:], clean[1, 2:])
        assert torch.equal(got[0, :2], clean[0, :2]) and torch.equal(got[2], clean[2])
        assert not bool(got[0, 2:, 9].isfinite().any())
        cols = [c for c in range(64) if c != 9]
        assert torch.equal(got[0, 2:][:, cols], clean[0, 2:][:, cols])
        # keys of -inf: weight zero; all of them: no weight at all
        cache.k[0, t[2][0], 0, :, :] = float("-inf")
        one = torch.ones((3, 4, 64), device=cuda, dtype=DT[ct])
        assert not bool(cache.attend(0, one)[2, :2].any())


def test_attend_absent_pages(cuda):
    """Page ids outside the pool count as absent: no address is formed from them."""
    cache, g = _filled(cuda, 2, 64, 16, [200, 33, 64], "bf16", 11)
    for r, b, bad in ((0, 0, -1), (0, 5, -2**31), (0, 12, 2**31 - 1), (1, 2, cache.n_pages), (2, 0, -7), (2, 1, -7), (2, 2, 1 << 20),
                      (2, 3, -1)):
        cache.table[r, b] = bad
    q = torch.randn((3, 4, 64), generator=g, device=cuda).bfloat16()
    want, bound = _attend_reference(q, cache.k[0], cache.v[0], cache.table, cache.lens, range(3), 0.125)
    got = cache.attend(0, q)
    _close(got, want, bound, torch.bfloat16)
    assert not bool(got[2].any())
    # lengths outside the table's width: negative is empty, too long is its whole width
    cache.lens.copy_(torch.tensor([-3, 2**31 - 1, 64], dtype=torch.int32))
    cache.table[1] = cache.table[0].clamp(0, cache.n_pages - 1)
    cache.k.nan_to_num_()
    cache.v.nan_to_num_()
    want, bound = _attend_reference(q, cache.k[0], cache.v[0], cache.table, cache.lens, range(3), 0.125)
    got = cache.attend(0, q)
    _close(got, want, bound, torch.bfloat16)
    assert not bool(got[0].any())


def _raw_attend(pages, q, lens, table, out, scale, dev):
    n, nh, hd = q.shape
    size = ctypes.c_size_t()
    check(lib().sxq_kv_attention_workspace(ctypes.byref(pages), n, nh, ctypes.byref(size)))
    ws = torch.zeros(size.value, dtype=torch.uint8, device=dev)
    check(lib().sxq_kv_attention(0, ctypes.byref(pages), {torch.float32: 0, torch.float16: 1, torch.bfloat16: 30}[q.dtype],
                                 q.data_ptr(), q.stride(0), n, nh, None, lens.data_ptr(), n, table.data_ptr(),
                                 table.stride(0), table.shape[1], scale, out.data_ptr(), out.stride(0), ws.data_ptr(),
                                 size.value, torch.cuda.current_stream().cuda_stream))


@pytest.mark.parametrize("ct", ["f32", "bf16", "f16"])
def test_attend_pools_of_other_strides(cuda, ct):
    """Position-major pages, keys and values of one tensor, a wider table, q and out as columns
    of wider rows."""
    dt, nh, nkv, hd, page, lens = DT[ct], 6, 2, 80, 16, [5, 100, 33]
    g = torch.Generator(device=cuda).manual_seed(3)
    both = torch.randn((30, page, 2, nkv, hd + 8), generator=g, device=cuda).to(dt)  # [page][pos][k|v][head][hd + pad]
    k, v = both[:, :, 0, :, :hd], both[:, :, 1, :, :hd]
    code = {"f32": 0, "f16": 1, "bf16": 30}[ct]
    pages = KvPages(code, nkv, hd, page, 30, k.data_ptr(), v.data_ptr(), k.stride(0), k.stride(2), k.stride(1))
    table = torch.randperm(30, generator=g, device=cuda).int().view(3, 10)
    ln = torch.tensor(lens, dtype=torch.int32, device=cuda)
    wide = torch.randn((3, (nh + 4) * hd), generator=g, device=cuda).to(dt)
    q = wide.as_strided((3, nh, hd), (wide.stride(0), hd, 1))
    buf = torch.full((3, (nh + 1) * hd), 3.0, device=cuda, dtype=dt)
    out = buf.as_strided((3, nh, hd), (buf.stride(0), hd, 1))
    _raw_attend(pages, q, ln, table[:, :8], out, 0.3, cuda)
    want, bound = _attend_reference(q, k.transpose(1, 2), v.transpose(1, 2), table[:, :8], lens, range(3), 0.3)
    _close(out, want, bound, dt)
    assert bool((buf[:, nh * hd:] == 3).all())


def test_offsets_past_32_bits(cuda):
    """Pages whose element and byte offsets pass 2^32, written by append and read by attend."""
    nkv, hd, page, n_pages = 8, 128, 16, 300000  # 4.9e9 elements a pool
    cache = PagedKvCache(1, nkv, hd, n_pages=n_pages, page_size=page, max_rows=2, max_len=64, dtype=torch.bfloat16, device=cuda)
    cache.free.copy_(torch.arange(n_pages, dtype=torch.int32))  # the last page on top
    m = cache.reserve([50, 20])
    assert int(m.slots.min()) > (n_pages - 10) * page
    g = torch.Generator(device=cuda).manual_seed(1)
    x = torch.randn((70, 48 * hd), generator=g, device=cuda).bfloat16()
    cache.append(0, x, m, n_heads=32)
    kv = x.view(70, 48, hd)[:, 32:]
    ids = m.slots.long()
    assert torch.equal(cache.k[0, ids // page, :, ids % page], kv[:, :8])
    q = torch.randn((2, 32, hd), generator=g, device=cuda).bfloat16()
    want, bound = _attend_reference(q, cache.k[0], cache.v[0], cache.table, cache.lens, range(2), hd ** -0.5)
    _close(cache.attend(0, q), want, bound, torch.bfloat16)


def test_attend_python_refusals(cuda):
    cache = PagedKvCache(1, 2, 64, n_pages=4, page_size=16, max_rows=2, max_len=64, dtype=torch.bfloat16, device=cuda)
    q = torch.zeros((2, 4, 64), dtype=torch.bfloat16, device=cuda)
    for bad in (q.cpu(), q[..., :32], q.double(), q.view(-1), q.transpose(0, 1), q.view(2, 256)[:, :100]):
        with pytest.raises(ValueError):
            cache.attend(0, bad)
    for kw in (dict(layer=2), dict(rows=torch.zeros(3, dtype=torch.int32, device=cuda)), dict(rows=torch.zeros(2, device=cuda)),
               dict(out=torch.zeros((2, 4, 64), device=cuda)), dict(out=q[:1]),
               dict(workspace=torch.zeros(1 << 20, device=cuda))):
        args = dict(layer=0)
        args.update(kw)
        with pytest.raises(ValueError):
            cache.attend(args.pop("layer"), q, **args)
    for bad in (q.half(), q[:, :3].contiguous(), torch.zeros((3, 4, 64), dtype=torch.bfloat16, device=cuda)):
        with pytest.raises(SxqError):
            cache.attend(0, bad)
    with pytest.raises(SxqError):
        cache.attend(0, q, scale=float("inf"))
    with pytest.raises(SxqError):
        cache.attend(0, q, workspace=torch.zeros(256, dtype=torch.uint8, device=cuda)[:0])
    assert cache.attend(0, q[:0]).shape == (0, 4, 64)


# ---- the operators together -----------------------------------------------------------

class Dense:
    """The same cache as lists of 64-bit rows per request, as stored (rounded to the pages')."""

    def __init__(self, rows):
        self.k, self.v = [[] for _ in range(rows)], [[] for _ in range(rows)]

    def attend(self, r, q, nkv, scale):
        G = q.shape[0] // nkv
        k, v = torch.stack(self.k[r]).to(F64), torch.stack(self.v[r]).to(F64)
        out = torch.empty(q.shape, dtype=F64, device=q.device)
        for h in range(nkv):
            w = torch.softmax(q[h * G:(h + 1) * G].to(F64) @ k[:, h].t().contiguous() * scale, -1)
            out[h * G:(h + 1) * G] = w @ v[:, h]
        return out


@pytest.mark.parametrize("it,ct", TYPES)
def test_decode_steps_of_ragged_requests(cuda, it, ct):
    """Prompts admitted, decode steps with requests joining, pausing and leaving: every step's
    context against the dense cache in 64 bits."""
    rows, nh, nkv, hd, page = 6, 8, 2, 64, 16
    cache = PagedKvCache(1, nkv, hd, n_pages=40, page_size=page, max_rows=rows, max_len=120, dtype=DT[ct], device=cuda)
    dense = Dense(rows)
    tables = _tables(cache.max_len, hd, cuda, 1e4)
    w = 1 + 0.1 * torch.randn(hd, device=cuda)
    g = torch.Generator(device=cuda).manual_seed(17)
    steps = [[30, 0, 17, 1, 0, 0], [1, 0, 1, 1, 0, 0], [1, 45, 0, 1, 0, 0], [1, 1, 1, 1, 100, 0], [RELEASE, 1, 1, 1, 1, 0],
             [16, 1, RELEASE, 1, 1, 64], [1, 1, 31, 1, 1, 1], [1, -20, 1, 1, 1, 1], [1, 1, 1, 1, 1, 1]]
    for add in steps:
        m = cache.reserve(add)
        assert not bool(m.status.any())
        for r, a in enumerate(add):
            if a < 0:
                keep = max(0, len(dense.k[r]) + a)
                del dense.k[r][keep:], dense.v[r][keep:]
        T = m.slots.numel()
        qkv = torch.randn((T, (nh + 2 * nkv) * hd), generator=g, device=cuda).to(DT[it])
        q = cache.append(0, qkv, m, n_heads=nh, q_norm=w, k_norm=w, rope=tables)
        ref, _ = _append_reference(qkv, nh, nkv, hd, w, w, 1e-6, tables, m.pos.long(), False)
        for t, r in enumerate(m.rows.tolist()):
            dense.k[r].append(ref[t, nh:nh + nkv].to(DT[ct]))
            dense.v[r].append(ref[t, nh + nkv:].to(DT[ct]))
        assert cache.lens.tolist() == [len(k) for k in dense.k]
        last = [int(c) - 1 for c, a in zip(m.cu.tolist()[1:], add) if a > 0]
        qs = q.view(T, nh, hd)[last].contiguous()
        ctx = cache.attend(0, qs, rows=m.rows[last].contiguous())
        for i, r in enumerate(m.rows[last].tolist()):
            want = dense.attend(r, qs[i], nkv, hd ** -0.5)
            # a cached value rounded the other way (its f32 arithmetic's last bit) is one step of
            # the pages' type off: 2 half-steps of |k| in a score (|q . k| scale < 8 here), of |v] in the sum
            tol = (2 * 8 + 2) * 2 * _half_step(DT[ct]) * 4 if ct != "f32" else 2e-4
            err = (ctx[i].to(F64) - want).abs() - _half_step(DT[it]) * want.abs()
            assert float(err.max()) < tol, (add, r, float(err.max()))
    used = sum(-(-len(k) // page) for k in dense.k)
    assert int(cache.free_count) == 40 - used
    cache.reserve([RELEASE] * rows)
    assert int(cache.free_count) == 40 and sorted(cache.free.tolist()) == list(range(40))


def _loop(cache, add, qkv, m, tables, q, out, ws):
    cache.reserve(add, out=m)
    cache.append(0, qkv, m, n_heads=8, rope=tables, out=q)
    cache.attend(0, q.view(-1, 8, 64), rows=m.rows, out=out, workspace=ws)


@pytest.mark.parametrize("own_ws", [True, False])
def test_a_captured_step_replays_with_eager_work_between(cuda, own_ws):
    """One decode step captured at a fixed capacity: the requests that take part change on the
    GPU; every replay equals the eager step on a second cache, with eager calls and
    synchronizations between the replays."""
    rows, cap = 5, 6

    def fresh():
        c = PagedKvCache(1, 2, 64, n_pages=60, page_size=16, max_rows=rows, max_len=400, dtype=torch.bfloat16, device=cuda)
        c.reserve([300, 3, 17, 0, 90])
        torch.manual_seed(4)
        c.k.copy_(torch.randn_like(c.k))
        c.v.copy_(torch.randn_like(c.v))
        return c

    a, b = fresh(), fresh()
    tables = _tables(400, 64, cuda)
    add = torch.zeros(rows, dtype=torch.int32, device=cuda)
    qkv = torch.zeros((cap, 12 * 64), dtype=torch.bfloat16, device=cuda)
    ma, mb = a.reserve(add, cap), b.reserve(add, cap)
    qa, qb = (torch.zeros((cap, 8 * 64), dtype=torch.bfloat16, device=cuda) for _ in range(2))
    oa, ob = (torch.zeros((cap, 8, 64), dtype=torch.bfloat16, device=cuda) for _ in range(2))
    ws = a.workspace(cap, 8) if own_ws else None
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _loop(a, add, qkv, ma, tables, qa, oa, ws)
        _loop(b, add, qkv, mb, tables, qb, ob, None)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _loop(a, add, qkv, ma, tables, qa, oa, ws)
    g = torch.Generator(device=cuda).manual_seed(8)
    for step in range(6):
        add.copy_(torch.tensor([[1, 1, 1, 1, 1], [1, 0, 1, 0, 1], [0, 2, 0, 0, 0], [1, 1, RELEASE, 1, 1], [1, 1, 3, 0, -40],
                                [1, 1, 1, 1, 1]][step], dtype=torch.int32))
        qkv.copy_(torch.randn(qkv.shape, generator=g, device=cuda))
        graph.replay()
        _loop(b, add, qkv, mb, tables, qb, ob, None)
        if step % 2:
            torch.cuda.synchronize()
        other = a.attend(0, qa.view(-1, 8, 64), rows=ma.rows)  # eager, its own workspace
        live = ma.rows >= 0
        assert torch.equal(other[live], oa[live]), step
        assert torch.equal(oa, ob) and torch.equal(qa, qb) and torch.equal(ma.slots, mb.slots), step
        assert torch.equal(a.lens, b.lens) and torch.equal(a.table, b.table) and torch.equal(a.free_count, b.free_count)


def test_two_graphs_and_two_streams_at_once(cuda):
    """Graphs captured on one stream and replayed on two at once, and eager calls on two streams:
    each has a workspace of its own."""
    cache, g = _filled(cuda, 2, 64, 16, [5000, 3000, 700], "bf16", 2)
    qs = [torch.randn((3, 8, 64), generator=g, device=cuda).bfloat16() for _ in range(2)]
    want = [cache.attend(0, q).clone() for q in qs]
    outs = [torch.zeros_like(q) for q in qs]
    graphs = []
    for q, o in zip(qs, outs):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            cache.attend(0, q, out=o)
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert torch.equal(o, w)
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(cache.attend(0, qs[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in got[i])
