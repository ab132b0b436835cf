"""What the paged attention does with keys, values and queries that are not finite, for every
pair of types."""
import pytest
import torch

from test_gpu_paged import DT, F64, TYPES, U32, _close, _filled

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
