"""The decode engine over a paged cache (sxq_lm_create_paged): every op of its steps and prompts
replayed by the CPU oracle exactly as for the contiguous engine (test_gpu_decoder's replays),
16-bit pages, the page accounting of its calls, graphs, and the Fish and CosyVoice loops on it."""
import functools

import numpy as np
import pytest
import torch

import test_gpu_decoder as T
from syrinx_amd import GgmlDType, SxqError
from syrinx_amd import _lib, dualar
from syrinx_amd import decoder as D

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def cuda():
    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a ROCm GPU")
    return torch.device("cuda:0")


def _paged(pages, page_size=16, kv_dtype=torch.float32, cls=D.DecoderLM):
    return functools.partial(cls, kv_pages=pages, page_size=page_size, kv_dtype=kv_dtype)


STEPS = {
    # name: (config, lengths, pages, page size)
    "fish_q4k": (lambda: T._fish_small(), [40], 6, 16),
    "fish_q8_0": (lambda: T._fish_small(dtype=GgmlDType.Q8_0), [31], 3, 32),
    "fish_bias": (lambda: T._fish_small(qkv_bias=1, o_bias=1), [40], 1, 64),
    "cv2_q8_0": (lambda: D.cosyvoice2_lm_config(n_layers=2, max_seq=96, dtype=GgmlDType.Q8_0), [70], 20, 16),
    "ragged": (lambda: T._fish_small(n_layers=1, max_batch=4), [5, 70, 17, 0], 12, 16),
    # a head width that no prompt kernel has, and lengths beyond the contiguous engine's limit
    "odd_width": (lambda: D.DecoderConfig(n_layers=1, dim=256, n_heads=16, n_kv_heads=2, head_dim=48, intermediate=256,
                                          vocab=64, max_seq=20000, weight_dtype=int(GgmlDType.Q8_0),
                                          tied_embedding=0), [16385], 320, 64),
}


@pytest.mark.parametrize("kind", list(STEPS))
def test_every_op_of_a_paged_step_matches_oracle(cuda, ora, kind):
    make, lengths, pages, page_size = STEPS[kind]
    cfg, n = make(), len(lengths)
    lm, W = T._build(cfg, cuda, 31, n, cls=_paged(pages, page_size))
    lm.kv_fill_random(lengths, seed=32)
    lm.enable_trace()
    rng = np.random.default_rng(33)
    for step in range(2):
        if cfg.n_codebooks:
            frames = list(T._frames(rng, n, cfg))
            logits, _ = lm.step(ids=torch.from_numpy(np.stack(frames)))
        else:
            frames = [None] * n
            logits, _ = lm.step(embeds=torch.from_numpy(rng.standard_normal((n, cfg.dim)).astype(np.float32)))
        tr, got = lm.trace(n), logits.cpu().numpy()
        for s in range(n):
            want = T._replay_step(ora, lm, cfg, W, tr, s, lengths[s] + step, frame=frames[s])
            T._bits_equal(got[s], want, f"{kind} stream {s} head projection")
    assert lm.lengths(n) == [v + 2 for v in lengths]
    assert lm.free_pages() == pages - sum(-(-(v + 2) // page_size) for v in lengths)


PROMPTS = {"fish_q4k_exact_1stream": (4, 16), "fish_q4k_gemm_after_cache": (2, 64), "fish_q8_0_ragged3": (9, 16),
           "cv2_q8_0_embeds": (3, 32), "cv2_q4_0_gemm_rows": (9, 16), "qwen3_4b_512_tokens": (17, 32)}


@pytest.mark.parametrize("kind", list(PROMPTS))
def test_every_op_of_a_paged_prompt_matches_oracle(cuda, ora, kind):
    make, plan, exact = T.PREFILL_KINDS[kind]
    cfg, n = make(), len(plan)
    lens0, counts = [p[0] for p in plan], [p[1] for p in plan]
    lm, W = T._build(cfg, cuda, 61, n, cls=_paged(*PROMPTS[kind]))
    lm.kv_fill_random(lens0, seed=62)
    rng = np.random.default_rng(63)
    if kind.startswith("cv2"):
        embs = [torch.from_numpy(rng.standard_normal((c, cfg.dim)).astype(np.float32)) for c in counts]
        logits, nxt, hidden, tr = lm.prefill(embeds=embs, exact=exact, trace=True)
        frames = None
    else:
        prompts = [T._frames(rng, c, cfg) for c in counts]
        logits, nxt, hidden, tr = lm.prefill(prompts=[torch.from_numpy(p) for p in prompts], exact=exact, trace=True)
        frames = np.concatenate(prompts)
    T._replay_prefill(ora, lm, cfg, W, tr, counts, lens0, frames, exact)
    assert lm.lengths(n) == [a + b for a, b in plan]


def _rope64(cfg, x, pos):
    half = cfg.head_dim // 2
    inv = (1.0 / np.power(np.float32(cfg.rope_theta), np.arange(half, dtype=np.float32) * 2 / cfg.head_dim)).astype(np.float32)
    a = (np.float32(pos) * inv).astype(np.float64)
    c, s = np.cos(a), np.sin(a)
    if cfg.rope_interleaved:
        y = np.empty_like(x)
        y[..., 0::2], y[..., 1::2] = x[..., 0::2] * c - x[..., 1::2] * s, x[..., 1::2] * c + x[..., 0::2] * s
        return y
    a_, b_ = x[..., :half], x[..., half:]
    return np.concatenate([a_ * c - b_ * s, b_ * c + a_ * s], -1)


def test_sixteen_bit_pages(cuda):
    """bf16 pages: the stored keys and values are the step's own rounded once, and the traced
    context is the attention over what is stored -- after a prompt, and after steps on it."""
    cfg = T._fish_small(n_layers=2, max_batch=3)
    lm, W = T._build(cfg, cuda, 71, 3, cls=_paged(20, 16, torch.bfloat16))
    rng = np.random.default_rng(72)
    counts = [33, 5, 48]
    prompts = [torch.from_numpy(T._frames(rng, c, cfg)) for c in counts]
    *_, tr = lm.prefill(prompts=prompts, exact=True, trace=True)
    rows = [(s, i) for s in range(3) for i in range(counts[s])]
    nh, nkv, hd = cfg.n_heads, cfg.n_kv_heads, cfg.head_dim
    G = nh // nkv

    def check(tr, rows):
        for l, t in enumerate(tr["layers"]):
            for r, (s, p) in enumerate(rows):
                k = t["qkv"][r][nh * hd:(nh + nkv) * hd].reshape(nkv, hd).astype(np.float64)
                v = torch.from_numpy(t["qkv"][r][(nh + nkv) * hd:].reshape(nkv, hd).copy())
                k = k / np.sqrt((k * k).mean(-1, keepdims=True) + cfg.norm_eps) * W[("k_norm", l)]
                k = _rope64(cfg, k, p)
                for g in range(nkv):
                    ks, vs = (x.cpu() for x in lm.read_kv(l, s, g, 0, p + 1))
                    assert torch.equal(vs[p], v[g].bfloat16().float())
                    # one rounding (2^-8) of a value off by the f32 norm and rotation (hd + 8 of
                    # 2^-24, relative to both terms of the rotation: at most 1.5 |k|max)
                    tol = 2.0 ** -8 * np.abs(k[g]) + (hd + 8) * 2.0 ** -24 * 1.5 * np.abs(k[g]).max()
                    assert (np.abs(ks[p].numpy() - k[g]) <= tol).all()
                    q = t["q"][r].reshape(nh, hd)[g * G:(g + 1) * G].astype(np.float64)
                    sc = q @ ks.numpy().astype(np.float64).T / np.sqrt(hd)
                    w = np.exp(sc - sc.max(-1, keepdims=True))
                    w /= w.sum(-1, keepdims=True)
                    T._glue_close(t["ctx"][r].reshape(nh, hd)[g * G:(g + 1) * G], w @ vs.numpy().astype(np.float64),
                                  f"layer {l} row {r} attention")

    check(tr, rows)
    lm.enable_trace()
    for step in range(2):
        lm.step(ids=torch.from_numpy(T._frames(rng, 3, cfg)))
        check(lm.trace(3), [(s, counts[s] + step) for s in range(3)])


def _engine(cfg, cuda, pages, page_size=16, seed=5, **kw):
    lm = D.DecoderLM(cfg, device=cuda, kv_pages=pages, page_size=page_size, **kw)
    lm.init_random(seed=seed)
    return lm


@pytest.mark.parametrize("kv_dtype", [torch.float32, torch.bfloat16])
def test_graph_replay_equals_eager(cuda, kv_dtype):
    """Steps of ragged streams across page ends, eager and as replayed graphs with eager work and
    synchronizations between, then a reset and another prompt: the same bits."""
    cfg = T._fish_small(n_layers=2, max_batch=3)
    a, b = (_engine(cfg, cuda, 18, kv_dtype=kv_dtype) for _ in range(2))
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
        assert a.free_pages() == 18 and a.lengths(3) == [0, 0, 0]


def test_rewinding_gives_pages_back_and_repeats_the_step(cuda):
    """A server that keeps a prompt and rewinds to it: the same steps give the same bits, however
    often, and the pages taken in between are there again."""
    cfg = T._fish_small(n_layers=1, max_batch=2)
    lm = _engine(cfg, cuda, 10)
    rng = np.random.default_rng(3)
    lm.prefill(prompts=[torch.from_numpy(T._frames(rng, c, cfg)) for c in (30, 15)])
    frames = [torch.from_numpy(T._frames(rng, 2, cfg)) for _ in range(5)]
    first = None
    for _ in range(3):
        out = [lm.step(ids=f, graph=True)[0].clone() for f in frames]
        assert lm.free_pages() == 10 - 3 - 2
        lm.set_lengths([30, 15])
        assert lm.free_pages() == 10 - 2 - 1
        first = first or out
        assert all(torch.equal(x, y) for x, y in zip(out, first))
    lm.set_lengths([0, 90])
    assert lm.free_pages() == 10 - 6 and lm.lengths(2) == [0, 90]


def test_out_of_pages_is_refused_before_anything_runs(cuda):
    cfg = T._fish_small(n_layers=1, max_batch=2)
    lm = _engine(cfg, cuda, 4)
    rng = np.random.default_rng(4)
    p = lambda c: torch.from_numpy(T._frames(rng, c, cfg))  # noqa: E731

    def refused(f):
        before = lm.lengths(2), lm.free_pages()
        with pytest.raises(SxqError) as e:
            f()
        assert e.value.code == _lib.ERR_OOM and "KV pages" in str(e.value)
        assert (lm.lengths(2), lm.free_pages()) == before

    refused(lambda: lm.prefill(prompts=[p(40), p(17)]))
    lm.prefill(prompts=[p(32), p(32)])
    refused(lambda: lm.step(ids=p(2)))
    refused(lambda: lm.set_lengths([65, 0]))
    lm.set_lengths([16, 32])
    x = lm.step(ids=p(1))[0]  # stream 0 takes the last page
    assert x.isfinite().all() and lm.free_pages() == 0 and lm.lengths(2) == [17, 32]
    refused(lambda: lm.step(ids=p(2)))


def test_create_refusals(cuda):
    cfg = T._fish_small(n_layers=1)
    for kw, code in ((dict(kv_pages=4, kv_dtype=torch.float16), _lib.ERR_DTYPE), (dict(kv_pages=4, kv_dtype=torch.int8), _lib.ERR_DTYPE),
                     (dict(kv_pages=0), _lib.ERR_INVALID), (dict(kv_pages=4, page_size=24), _lib.ERR_INVALID),
                     (dict(kv_pages=4, page_size=8), _lib.ERR_INVALID)):
        with pytest.raises(SxqError) as e:
            D.DecoderLM(cfg, device=cuda, **kw)
        assert e.value.code == code
    with pytest.raises(SxqError):  # max_seq
        D.DecoderLM(D.fish_s2_slow_ar_config(n_layers=1, max_seq=(1 << 20) + 1), device=cuda, kv_pages=4)
    with pytest.raises(SxqError):  # not a paged engine
        D.DecoderLM(cfg, device=cuda).free_pages()
    fast = D.FastAr(D.fish_s2_fast_ar_config(n_layers=1, residual_size=64, dtype=GgmlDType.Q8_0), device=cuda, kv_pages=4)
    from syrinx_amd.sampling import FishSampler
    with pytest.raises(SxqError) as e:
        fast.expand_batch(torch.zeros((1, 2560), device=cuda), torch.zeros(1, dtype=torch.int32, device=cuda),
                          FishSampler([1], semantic=(0, 63, -1), device=cuda))
    assert "paged" in str(e.value)


def test_fish_frames_on_a_paged_slow_ar(cuda):
    """drive_batch with its slow AR paged: the same call twice gives the same codes (the caches
    emptied and their pages taken again in between), frames of every stream."""
    cfg = T._fish_small(n_layers=2, max_batch=3)
    slow = D.SlowAr(cfg, device=cuda, kv_pages=12, page_size=16, kv_dtype=torch.bfloat16)
    slow.init_random(seed=6)
    fast = D.FastAr(D.fish_s2_fast_ar_config(n_layers=1, num_codebooks=10, residual_size=64, max_batch=3), device=cuda)
    fast.init_random(seed=7)
    rng = np.random.default_rng(8)
    prompts = [T._frames(rng, c, cfg).T for c in (12, 30, 5)]
    params = dualar.DriveParams(max_new_frames=6)
    one = dualar.drive_batch(slow, fast, prompts, stop_id=4000, params=params)
    two = dualar.drive_batch(slow, fast, prompts, stop_id=4000, params=params)
    assert len(one) == 3 and all(torch.equal(x, y) for x, y in zip(one, two))
    assert all(x.shape[0] == 10 and x.shape[1] >= 1 for x in one)


def test_cosyvoice_generate_on_a_paged_engine(cuda, tmp_path):
    from syrinx_amd.generate import CosyVoiceLm

    cfg = D.cosyvoice2_lm_config(n_layers=2, max_seq=160)
    lm = D.Qwen2Lm(cfg, device=cuda, kv_pages=10, page_size=16)
    lm.init_random(seed=10)
    text = torch.randn((50, cfg.dim), device=cuda) * 0.5
    speech = torch.randn((cfg.embed_rows, cfg.dim), device=cuda) * 0.5
    lm.set_vector(-1, D.EMBED, speech)
    cv = CosyVoiceLm(lm, text, speech, torch.randn((2, cfg.dim), device=cuda))
    a = cv.generate([1, 2, 3, 4], [5, 6, 7], 8, 30, seed=11)
    b = cv.generate([1, 2, 3, 4], [5, 6, 7], 8, 30, seed=11)
    assert a == b and len(a) >= 8 and all(0 <= t < 6561 for t in a)
