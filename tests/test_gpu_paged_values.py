"""What the paged attention does with keys, values and queries that are not finite, for every
pair of types, and a decode loop held to derived bounds at each of its steps."""
import pytest
import torch

from syrinx_amd.paged import RELEASE, PagedKvCache
from test_gpu_paged import (DT, F64, TYPES, U32, _append_reference, _attend_reference, _close, _filled, _half_step,
                            _tables)

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def cuda():
    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a ROCm GPU")
    return torch.device("cuda:0")


@pytest.mark.parametrize("nh,nkv,hd,page,L", [(4, 1, 64, 16, 50), (8, 2, 128, 32, 700), (3, 1, 80, 16, 33), (2, 2, 256, 64, 300)])
@pytest.mark.parametrize("qt,ct", TYPES)
def test_keys_with_infinities(cuda, qt, ct, nh, nkv, hd, page, L):
    """A score of -inf has no weight, one of +inf or NaN makes its head NaN, and where every score
    is -inf the output is zero: as the arithmetic has it, whatever the queries' type."""
    cache, g = _filled(cuda, nkv, hd, page, [L, L, L, L], ct, hd + L)
    q = torch.randn((4, nh, hd), generator=g, device=cuda)
    q[:, :, 3] = q[:, :, 3].abs() + 0.5      # f32 values with and without low parts
    q[:, :, 4] = 1.5                         # exact in 16 bits: the low parts are zero
    q[3, 0, 4] = 0.0
    q = q.to(DT[qt])
    clean = cache.attend(0, q).clone()

    def at(r, p, h, d):
        return (0, int(cache.table[r, p // page]), h, p % page, d)

    gone = sorted({0, 7, 15, 16, L // 2, L - 1})
    for p in gone:
        cache.k[at(0, p, 0, 3)] = float("-inf")
        cache.k[at(0, p, 0, 4)] = float("-inf")
    cache.k[at(1, L // 3, 0, 4)] = float("inf")
    for p in range(L):
        cache.k[at(2, p, 0, 3)] = float("-inf")
    cache.k[at(3, 5, 0, 4)] = float("-inf")
    got = cache.attend(0, q)
    G = nh // nkv
    assert torch.equal(got[:, G:], clean[:, G:])  # the other KV heads
    # request 0: the definition over the positions that have weight
    p = torch.tensor([i for i in range(L) if i not in gone], device=cuda)
    ids = cache.table[0].long()[p // page]
    k, v = (pool[0, ids, 0, p % page].to(F64) for pool in (cache.k, cache.v))
    qq = q[0, :G].to(F64)
    w = torch.softmax(qq @ k.t().contiguous() * hd ** -0.5, -1)
    S = (qq.abs() @ k.abs().t().contiguous()).amax(-1, keepdim=True) * hd ** -0.5
    split = 2.0 ** -18 if qt == "bf16" else 4 * U32
    rel = 2 * (hd + 3) * U32 * S + 2 * S * U32 + split + (4 + 4 * (L / 16 + 2) + 2 * L) * U32
    _close(got[0, :G], w @ v, 2 * rel * (w @ v.abs()), DT[qt], "without the keys of -inf")
    assert bool(got[1, :G].isnan().all())
    assert not bool(got[2, :G].any())
    assert bool(got[3, 0].isnan().all()) and bool(got[3, 1:G].isfinite().all())  # 0 * -inf; a weight of none


@pytest.mark.parametrize("qt,ct", TYPES)
def test_infinite_queries_and_values(cuda, qt, ct):
    cache, g = _filled(cuda, 1, 64, 16, [40, 40, 40], ct, 3)
    q = torch.randn((3, 2, 64), generator=g, device=cuda).to(DT[qt])
    clean = cache.attend(0, q).clone()
    q[0, 0, 9] = float("inf")   # scores of both signs: +inf among them
    q[1, 1, 9] = float("nan")
    cache.v[0, int(cache.table[2, 1]), 0, 3, 7] = float("-inf")
    got = cache.attend(0, q)
    assert bool(got[0, 0].isnan().all()) and torch.equal(got[0, 1], clean[0, 1])
    assert bool(got[1, 1].isnan().all()) and torch.equal(got[1, 0], clean[1, 0])
    assert not bool(got[2, :, 7].isfinite().any())
    cols = [c for c in range(64) if c != 7]
    assert torch.equal(got[2][:, cols], clean[2][:, cols])
    # a query of -inf over keys of one sign: every score -inf
    cache.k.copy_(cache.k.nan_to_num().abs() + 0.5)
    q = torch.zeros((3, 2, 64), device=cuda, dtype=DT[qt])
    q[:, :, :] = float("-inf")
    assert not bool(cache.attend(0, q)[:2].any())


class Stored:
    """Requests' rows in 64 bits as the definition gives them, before the pages' rounding, with the
    bound of the f32 arithmetic that made them."""

    def __init__(self, rows):
        self.k, self.v, self.kb = ([[] for _ in range(rows)] for _ in range(3))


@pytest.mark.parametrize("it,ct", TYPES)
def test_decode_loop_step_by_step(cuda, it, ct):
    """Prompts admitted, decode steps with requests joining, pausing, rewinding and leaving.  Each
    step is held to two derived bounds: every row that the pages hold, read through the table,
    against the row's own values (one rounding of the pages' type); and the context against
    64-bit attention over what is stored."""
    rows, nh, nkv, hd, page = 6, 8, 2, 64, 16
    cache = PagedKvCache(1, nkv, hd, n_pages=40, page_size=page, max_rows=rows, max_len=120, dtype=DT[ct], device=cuda)
    want = Stored(rows)
    tables = _tables(cache.max_len, hd, cuda, 1e4)
    g = torch.Generator(device=cuda).manual_seed(23)
    w = 1 + 0.1 * torch.randn(hd, generator=g, device=cuda)
    rel = (hd / 2 + 9) * U32  # as for the append alone
    tiny = torch.finfo(DT[ct]).smallest_normal * torch.finfo(DT[ct]).eps
    steps = [[30, 0, 17, 1, 0, 0], [1, 0, 1, 1, 0, 0], [1, 45, 0, 1, 0, 0], [1, 1, 1, 1, 100, 0], [RELEASE, 1, 1, 1, 1, 0],
             [16, 1, RELEASE, 1, 1, 64], [1, 1, 31, 1, 1, 1], [1, -20, 1, 1, 1, 1], [1, 1, 1, 1, 1, 1], [1, 12, 0, -3, 1, 1]]
    for step, add in enumerate(steps):
        m = cache.reserve(add)
        assert not bool(m.status.any())
        for r, a in enumerate(add):
            if a < 0:
                keep = max(0, len(want.k[r]) + a)
                for rows_of in (want.k, want.v, want.kb):
                    del rows_of[r][keep:]
        n = m.slots.numel()
        qkv = torch.randn((n, (nh + 2 * nkv) * hd), generator=g, device=cuda).to(DT[it])
        q = cache.append(0, qkv, m, n_heads=nh, q_norm=w, k_norm=w, rope=tables)
        ref, mag = _append_reference(qkv, nh, nkv, hd, w, w, 1e-6, tables, m.pos.long(), False)
        for t, r in enumerate(m.rows.tolist()):
            want.k[r].append(ref[t, nh:nh + nkv])
            want.kb[r].append(rel * mag[t, nh:nh + nkv])
            want.v[r].append(ref[t, nh + nkv:])
        assert cache.lens.tolist() == [len(k) for k in want.k]
        held = set()
        for r in range(rows):
            L = len(want.k[r])
            if L == 0:
                continue
            p = torch.arange(L, device=cuda)
            ids = cache.table[r].long()[p // page]
            mine = set(ids.tolist())
            assert not held & mine and min(mine) >= 0  # no page belongs to two
            held |= mine
            half = _half_step(DT[ct])
            k, v = (pool[0, ids, :, p % page].to(F64) for pool in (cache.k, cache.v))
            k64, kb = torch.stack(want.k[r]), torch.stack(want.kb[r])
            assert bool(((k - k64).abs() <= kb + half * (k64.abs() + kb) + tiny).all()), (step, r, "keys")
            v64 = torch.stack(want.v[r])
            assert bool(((v - v64).abs() <= half * v64.abs() + tiny).all()), (step, r, "values")
        last = [int(c) - 1 for c, a in zip(m.cu.tolist()[1:], add) if a > 0]
        qs, of = q.view(n, nh, hd)[last].contiguous(), m.rows[last].contiguous()
        ctx = cache.attend(0, qs, rows=of)
        exact, bound = _attend_reference(qs, cache.k[0], cache.v[0], cache.table, cache.lens, of.tolist(), hd ** -0.5)
        _close(ctx, exact, bound, DT[it], f"step {step}")


def test_every_query_sees_its_whole_request(cuda):
    """Maps with several tokens of a request: each query reads the request to its end, later tokens
    included, so that a decoder's attention is that of the last one; picked by cu, those equal
    the calls of one token."""
    nh, nkv, hd = 4, 2, 64
    cache = PagedKvCache(1, nkv, hd, n_pages=20, page_size=16, max_rows=3, max_len=100, dtype=torch.float32, device=cuda)
    g = torch.Generator(device=cuda).manual_seed(5)
    m = cache.reserve([40, 0, 3])
    q = cache.append(0, torch.randn((43, (nh + 2 * nkv) * hd), generator=g, device=cuda), m, n_heads=nh)
    q = q.view(43, nh, hd)
    got = cache.attend(0, q, rows=m.rows)
    want, bound = _attend_reference(q, cache.k[0], cache.v[0], cache.table, cache.lens, m.rows.tolist(), hd ** -0.5)
    _close(got, want, bound, torch.float32)
    grew = m.cu[1:] > m.cu[:-1]
    last = (m.cu[1:] - 1).clamp(min=0).long()
    rows = torch.where(grew, torch.arange(3, device=cuda), -1).int()
    out = torch.full((3, nh, hd), 7.0, device=cuda)
    cache.attend(0, q[last].contiguous(), rows=rows, out=out)
    assert bool((out[1] == 7).all())
    _close(out[[0, 2]], want[[39, 42]], bound[[39, 42]], torch.float32)
