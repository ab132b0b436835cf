"""Decode engines whose paged cache holds e4m3 codes: stored keys and values within half a step of the
step's own, the attention over what is stored, graphs, rewinds, and the loops that drive an engine."""
import numpy as np
import pytest
import torch

import test_gpu_decoder as T
from syrinx_amd import SxqError, _lib, dualar
from syrinx_amd import decoder as D
from test_gpu_paged_engine import _engine, _paged, _rope64

pytestmark = pytest.mark.gpu
E4M3 = torch.float8_e4m3fn


@pytest.fixture(scope="module")
def cuda():
    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a ROCm GPU")
    return torch.device("cuda:0")


@pytest.mark.parametrize("kind", ["fish", "cv2"])
def test_e4m3_pages(cuda, kind):
    """What is read back is within a code's half step (2^-4 of the value, or 2^-10 of a scale that is at
    most 2 / 448 of the largest value near it, twice where a block was rescaled) of the step's own keys
    and values, off by the f32 norm and rotation; the traced context is the attention over it."""
    if kind == "fish":
        cfg = T._fish_small(n_layers=2, max_batch=3)
    else:
        cfg = D.cosyvoice2_lm_config(n_layers=2, max_seq=96, max_batch=3)
    lm, W = T._build(cfg, cuda, 71, 3, cls=_paged(20, 16, E4M3))
    rng = np.random.default_rng(72)
    counts = [33, 5, 48]
    if kind == "fish":
        *_, tr = lm.prefill(prompts=[torch.from_numpy(T._frames(rng, c, cfg)) for c in counts], exact=True, trace=True)
    else:
        *_, tr = lm.prefill(embeds=[torch.from_numpy(rng.standard_normal((c, cfg.dim)).astype(np.float32)) for c in counts],
                            exact=True, trace=True)
    rows = [(s, i) for s in range(3) for i in range(counts[s])]
    nh, nkv, hd = cfg.n_heads, cfg.n_kv_heads, cfg.head_dim
    G = nh // nkv

    def check(tr, rows):
        for l, t in enumerate(tr["layers"]):
            for r, (s, p) in enumerate(rows):
                k = t["qkv"][r][nh * hd:(nh + nkv) * hd].reshape(nkv, hd).astype(np.float64)
                v = t["qkv"][r][(nh + nkv) * hd:].reshape(nkv, hd).astype(np.float64)
                if cfg.qk_norm:
                    k = k / np.sqrt((k * k).mean(-1, keepdims=True) + cfg.norm_eps) * W[("k_norm", l)]
                k = _rope64(cfg, k, p)
                for g in range(nkv):
                    last = lm.lengths(3)[s]
                    ks, vs = (x.cpu().numpy().astype(np.float64) for x in lm.read_kv(l, s, g, 0, last))
                    block = slice(p // 16 * 16, min(last, p // 16 * 16 + 16))
                    for got, want, f32 in ((ks, k[g], (hd + 8) * 2.0 ** -24 * 1.5), (vs, v[g], 0.0)):
                        top = np.abs(got[block]).max() * (1 + 2.0 ** -4)
                        tol = 2.0 ** -4 * np.abs(want) + 2 * 2.0 ** -10 * top * 2 / 448 + f32 * np.abs(want).max()
                        assert (np.abs(got[p] - want) <= tol).all(), (l, r, g)
                    ks, vs = ks[:p + 1], vs[:p + 1]
                    q = t["q"][r].reshape(nh, hd)[g * G:(g + 1) * G].astype(np.float64)
                    sc = q @ ks.T / np.sqrt(hd)
                    w = np.exp(sc - sc.max(-1, keepdims=True))
                    w /= w.sum(-1, keepdims=True)
                    T._glue_close(t["ctx"][r].reshape(nh, hd)[g * G:(g + 1) * G], w @ vs, f"layer {l} row {r} attention")

    check(tr, rows)
    lm.enable_trace()
    for step in range(2):
        # (a step may rescale its block's earlier codes, so what it read is what is there after it)
        if kind == "fish":
            lm.step(ids=torch.from_numpy(T._frames(rng, 3, cfg)))
        else:
            lm.step(embeds=torch.from_numpy(rng.standard_normal((3, cfg.dim)).astype(np.float32)))
        check(lm.trace(3), [(s, counts[s] + step) for s in range(3)])


def test_graph_replay_equals_eager(cuda):
    cfg = T._fish_small(n_layers=2, max_batch=3)
    a, b = (_engine(cfg, cuda, 18, kv_dtype=E4M3) for _ in range(2))
    rng = np.random.default_rng(9)
    prompts = [torch.from_numpy(T._frames(rng, c, cfg)) for c in (14, 31, 2)]
    for again in range(2):
        la, lb = a.prefill(prompts=prompts)[0], b.prefill(prompts=prompts)[0]
        assert torch.equal(la, lb)
        for step in range(6):
            n = 3 if step != 3 else 2
            fr = torch.from_numpy(T._frames(rng, n, cfg))
            x, nx = a.step(ids=fr, graph=True)
            y, ny = b.step(ids=fr, graph=False)
            if step % 2:
                torch.cuda.synchronize()
            assert torch.equal(x, y) and torch.equal(nx, ny), (again, step)
        assert a.lengths(3) == b.lengths(3) == [20, 37, 7] and a.free_pages() == b.free_pages() == 18 - 2 - 3 - 1
        a.reset()
        b.reset()


def test_a_reset_engine_repeats_a_prompt(cuda):
    """After a reset a stream's blocks begin anew, whatever scales its pages had: the same prompt and
    steps give the same bits, also in pages that other streams had."""
    cfg = T._fish_small(n_layers=1, max_batch=2)
    lm = _engine(cfg, cuda, 12, kv_dtype=E4M3)
    rng = np.random.default_rng(3)
    prompts = [torch.from_numpy(T._frames(rng, c, cfg)) for c in (30, 15)]
    frames = [torch.from_numpy(T._frames(rng, 2, cfg)) for _ in range(4)]
    first = None
    for turn in range(3):
        lm.kv_fill_random([90, 40], seed=turn)  # other codes and scales everywhere
        lm.reset()
        lm.prefill(prompts=prompts)
        out = [lm.step(ids=f, graph=True)[0].clone() for f in frames]
        first = first or out
        assert all(torch.equal(x, y) for x, y in zip(out, first))
        lm.reset()


def test_filled_cache_reads_as_normal_values(cuda):
    cfg = T._fish_small(n_layers=2, max_batch=2)
    lm = _engine(cfg, cuda, 12, kv_dtype=E4M3)
    lm.kv_fill_random([90, 17], seed=4)
    k, v = lm.read_kv(1, 0, 1, 0, 90)
    for x in (k, v):
        assert x.isfinite().all() and 0.9 < float(x.std()) < 1.1 and float(x.abs().max()) <= 7.0
    assert lm.step(ids=torch.from_numpy(T._frames(np.random.default_rng(1), 2, cfg)))[0].isfinite().all()


def test_create_refusals(cuda):
    cfg = T._fish_small(n_layers=1)
    with pytest.raises(SxqError) as e:
        D.DecoderLM(cfg, device=cuda, kv_pages=4, kv_dtype=torch.int8)
    assert e.value.code == _lib.ERR_DTYPE and "e4m3" in str(e.value)
    with pytest.raises(ValueError):
        D.DecoderLM(cfg, device=cuda, kv_dtype=E4M3)


def test_fish_frames_and_cosyvoice_tokens(cuda):
    from syrinx_amd.generate import CosyVoiceLm

    cfg = T._fish_small(n_layers=2, max_batch=3)
    slow = D.SlowAr(cfg, device=cuda, kv_pages=12, page_size=16, kv_dtype=E4M3)
    slow.init_random(seed=6)
    fast = D.FastAr(D.fish_s2_fast_ar_config(n_layers=1, num_codebooks=10, residual_size=64, max_batch=3), device=cuda)
    fast.init_random(seed=7)
    rng = np.random.default_rng(8)
    prompts = [T._frames(rng, c, cfg).T for c in (12, 30, 5)]
    params = dualar.DriveParams(max_new_frames=6)
    one = dualar.drive_batch(slow, fast, prompts, stop_id=4000, params=params)
    two = dualar.drive_batch(slow, fast, prompts, stop_id=4000, params=params)
    assert len(one) == 3 and all(torch.equal(x, y) for x, y in zip(one, two))
    cfg = D.cosyvoice2_lm_config(n_layers=2, max_seq=160)
    lm = D.Qwen2Lm(cfg, device=cuda, kv_pages=10, page_size=16, kv_dtype=E4M3)
    lm.init_random(seed=10)
    text = torch.randn((50, cfg.dim), device=cuda) * 0.5
    speech = torch.randn((cfg.embed_rows, cfg.dim), device=cuda) * 0.5
    lm.set_vector(-1, D.EMBED, speech)
    cv = CosyVoiceLm(lm, text, speech, torch.randn((2, cfg.dim), device=cuda))
    a = cv.generate([1, 2, 3, 4], [5, 6, 7], 8, 30, seed=11)
    b = cv.generate([1, 2, 3, 4], [5, 6, 7], 8, 30, seed=11)
    assert a == b and len(a) >= 8 and all(0 <= t < 6561 for t in a)
