"""Serving loops on a paged decode engine: streams that have stopped, pages that run out in the
middle of a generation, long histories under a prompt."""
import dataclasses
import functools

import numpy as np
import pytest
import torch

import test_gpu_decoder as T
from syrinx_amd import SxqError, _lib, dualar
from syrinx_amd import decoder as D
from syrinx_amd.generate import COSYVOICE2, CosyVoiceLm
from syrinx_amd.sampling import RasSampler

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def cuda():
    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a ROCm GPU")
    return torch.device("cuda:0")


# ---- steps in which some streams sit out --------------------------------------------------

PATTERNS = [(1, 1, 1), (1, 0, 1), (0, 0, 1), (0, 1, 0), (1, 1, 1), (1, 0, 0)]


@pytest.mark.parametrize("page", [16, 32])
def test_every_op_of_the_streams_that_take_part_matches_oracle(cuda, ora, page):
    cfg, lengths = T._fish_small(n_layers=2, max_batch=3), [31, 5, 16]
    lm, W = T._build(cfg, cuda, 31, 3, cls=functools.partial(D.DecoderLM, kv_pages=12, page_size=page))
    lm.kv_fill_random(lengths, seed=32)
    lm.enable_trace()
    rng = np.random.default_rng(33)
    for active in PATTERNS:
        frames = list(T._frames(rng, 3, cfg))
        logits, _ = lm.step(ids=torch.from_numpy(np.stack(frames)), active=active)
        tr, got = lm.trace(3), logits.cpu().numpy()
        for s in range(3):
            if active[s]:
                want = T._replay_step(ora, lm, cfg, W, tr, s, lengths[s], frame=frames[s])
                T._bits_equal(got[s], want, f"{active} stream {s} head projection")
                lengths[s] += 1
        assert lm.lengths(3) == lengths and lm.free_pages() == 12 - sum(-(-n // page) for n in lengths)


def test_steps_of_some_streams_as_graphs(cuda):
    """Graph and eager steps of changing patterns, eager work and synchronizations between: the
    same bits for the streams that take part, the caches of the others as they were."""
    cfg = T._fish_small(n_layers=2, max_batch=3)
    a, b = (D.DecoderLM(cfg, device=cuda, kv_pages=18, page_size=16, kv_dtype=torch.bfloat16) for _ in range(2))
    rng = np.random.default_rng(5)
    prompts = [torch.from_numpy(T._frames(rng, n, cfg)) for n in (15, 30, 1)]
    for lm in (a, b):
        lm.init_random(seed=4)
        lm.prefill(prompts=prompts)
    for turn in range(18):
        active = PATTERNS[turn * 5 % len(PATTERNS)]
        ids = torch.from_numpy(T._frames(rng, 3, cfg))
        held = [s for s in range(3) if not active[s]]
        before = [[x.clone() for x in a.read_kv(1, s, 0, 0, a.lengths(3)[s])] for s in held]
        x, nx = a.step(ids=ids, graph=True, active=active)
        y, ny = b.step(ids=ids, graph=False, active=active)
        if turn % 3 == 1:
            torch.cuda.synchronize()
        live = [s for s in range(3) if active[s]]
        assert torch.equal(x[live], y[live]) and torch.equal(nx[live], ny[live]), (turn, active)
        assert x.isfinite().all() and a.lengths(3) == b.lengths(3)
        for s, old in zip(held, before):
            assert all(torch.equal(u, v) for u, v in zip(a.read_kv(1, s, 0, 0, a.lengths(3)[s]), old))
    for wrong in ([1, 0], [1, 1, 1, 1]):
        with pytest.raises(ValueError):
            a.step(ids=ids, active=wrong)
    with pytest.raises(SxqError) as e:
        D.DecoderLM(cfg, device=cuda).step(ids=ids, active=[1, 0, 1])
    assert e.value.code == _lib.ERR_INVALID


# ---- the Fish frame loop ----------------------------------------------------------------

class Scripted(dualar.FishSampler):
    """A sampler whose stream i stops at its pass stops[i] (from 0)."""

    def __init__(self, stops, semantic, device):
        super().__init__([1] * len(stops), semantic=semantic, device=device)
        self.stops, self.turn = stops, 0

    def sample_semantic(self, logits, out=None, out_stride=1, active=None):
        super().sample_semantic(logits, out=out, out_stride=out_stride, active=active)
        stop = torch.tensor([self.turn >= s for s in self.stops], device=active.device)
        active.masked_fill_(stop, 0)
        self.turn += 1


def _loop(cuda, pages, counts, stops, frames, page_size=16, **kw):
    """The frame loop over prompts of `counts` tokens; the slow engine, the number of passes, and
    the flags of every pass."""
    cfg = dataclasses.replace(T._fish_small(n_layers=1, max_batch=len(counts)), max_seq=400)
    slow = D.SlowAr(cfg, device=cuda, kv_pages=pages, page_size=page_size, **kw)
    slow.init_random(seed=6)
    fast = D.FastAr(D.fish_s2_fast_ar_config(n_layers=1, num_codebooks=10, residual_size=64, max_batch=len(counts)), device=cuda)
    fast.init_random(seed=7)
    rng = np.random.default_rng(8)
    logits, hidden = slow.prefill_batch([T._frames(rng, c, cfg).T for c in counts])
    sampler = Scripted(stops, (cfg.semantic_begin, cfg.semantic_end, -1), cuda)
    out, flags = dualar.generate_frames(slow, fast, sampler, logits, hidden, frames, max(counts))
    return slow, out, torch.stack(flags).cpu()


def test_streams_that_have_stopped_take_no_pages(cuda):
    """Three of four streams stop early: the pool holds the live tokens and no more."""
    stops, counts, frames = [3, 200, 7, 0], [20, 10, 31, 5], 120
    # stream 1 alone grows to 10 + 119; a stopped one may have had one step more than it needed
    pages = -(-(10 + 119) // 16) + sum(-(-(c + s + 1) // 16) for c, s in ((20, 3), (31, 7), (5, 0)))
    slow, out, flags = _loop(cuda, pages, counts, stops, frames)
    assert len(out) == frames and flags[:, 1].all()
    assert flags[:, 0].sum() == 3 and flags[:, 2].sum() == 7 and flags[:, 3].sum() == 0
    lens = slow.lengths(4)
    assert lens[1] == 10 + 119
    assert all(c + s <= n <= c + s + 1 for n, c, s in zip((lens[0], lens[2], lens[3]), (20, 31, 5), (3, 7, 0)))


def test_the_loop_ends_with_its_frames_when_pages_run_out(cuda):
    """Two live streams over a pool for 40 more tokens each: the frames up to there."""
    slow, out, flags = _loop(cuda, 2 * 3, [8, 8], [500, 500], 300)
    assert len(out) == 3 * 16 - 8 + 1 and flags.all()  # the last pass has no room for a step
    assert slow.lengths(2) == [48, 48] and slow.free_pages() == 0


def test_a_stream_that_stops_on_the_last_page_leaves_it_to_the_others(cuda):
    """The step that finds no pages comes before the host has seen who has stopped: it is made
    again for those that have not."""
    # both need a page at length 32; stream 0 stops in that very pass, one page is left
    slow, out, flags = _loop(cuda, 5, [16, 16], [16, 500], 40)
    assert len(out) == 33 and flags[:, 1].all() and flags[:, 0].sum() == 16
    assert slow.lengths(2) == [32, 48]


def test_every_stream_stopped_ends_the_loop(cuda):
    slow, out, flags = _loop(cuda, 8, [16, 20], [2, 5], 60)
    assert len(out) <= 7 and not flags[-1].any()


# ---- the CosyVoice loop -----------------------------------------------------------------

class ScriptedRas(RasSampler):
    """A sampler whose draw number `stop` (from 0) is a stop id."""

    def __init__(self, stop, variant, device):
        super().__init__([3], eos=(variant.stop_begin, variant.stop_end), device=device)
        self.stop, self.turn, self.first = stop, 0, variant.stop_begin

    def sample(self, logits, ignore_eos=False, out=None):
        super().sample(logits, ignore_eos=True, out=out)
        if self.turn == self.stop:
            out.fill_(self.first)
        self.turn += 1


@pytest.mark.parametrize("stop,ends", [(0, True), (6, True), (7, True), (8, False), (100, False)])
def test_a_token_that_stops_needs_no_page_for_the_step_after_it(cuda, stop, ends):
    """Nine prompt rows in a pool of one page of 16: seven steps have room.  The draw after them may
    be the stop, whose step (enqueued before the host looks) is not needed; another token's is."""
    cfg = D.cosyvoice2_lm_config(n_layers=1, max_seq=160)
    lm = D.Qwen2Lm(cfg, device=cuda, kv_pages=1, page_size=16)
    lm.init_random(seed=10)
    text = torch.randn((50, cfg.dim), device=cuda) * 0.5
    speech = torch.randn((cfg.embed_rows, cfg.dim), device=cuda) * 0.5
    lm.set_vector(-1, D.EMBED, speech)
    cv = CosyVoiceLm(lm, text, speech, torch.randn((2, cfg.dim), device=cuda))
    sampler = ScriptedRas(stop, COSYVOICE2, cuda)
    run = lambda: cv.generate([1, 2, 3, 4], [5, 6, 7], 0, 40, seed=0, sampler=sampler)  # noqa: E731
    if ends:
        assert len(run()) == stop
    else:
        with pytest.raises(SxqError) as e:
            run()
        assert e.value.code == _lib.ERR_OOM and "KV pages" in str(e.value)
    assert lm.lengths(1)[0] <= 16


# ---- prompts over long histories ----------------------------------------------------------

@pytest.mark.parametrize("kv_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("lens,counts,page", [([17000, 5, 300], [40, 33, 1], 32), ([0, 20000], [3, 70], 64),
                                              ([100, 0, 17], [1, 50, 130], 16)])
def test_a_prompt_attends_over_its_own_history(cuda, kv_dtype, lens, counts, page):
    """Streams of unlike lengths (past the contiguous engine's limit too): the traced context of a
    prompt's rows against 64-bit attention over what the pages hold of the row's own stream."""
    n, cfg = len(lens), dataclasses.replace(T._fish_small(n_layers=2, max_batch=len(lens)), max_seq=24000)
    pages = sum(-(-(a + b) // page) for a, b in zip(lens, counts))
    lm = D.DecoderLM(cfg, device=cuda, kv_pages=pages, page_size=page, kv_dtype=kv_dtype)
    lm.init_random(seed=11)
    lm.kv_fill_random(lens, seed=12)
    rng = np.random.default_rng(13)
    *_, tr = lm.prefill(prompts=[torch.from_numpy(T._frames(rng, c, cfg)) for c in counts], exact=True, trace=True)
    assert lm.free_pages() == 0
    nh, nkv, hd = cfg.n_heads, cfg.n_kv_heads, cfg.head_dim
    G, first, u = nh // nkv, 0, 2.0 ** -24
    for s in range(n):
        for i in sorted({0, counts[s] // 2, counts[s] - 1}):
            L = lens[s] + i + 1
            for l in range(2):
                q = torch.from_numpy(tr["layers"][l]["q"][first + i].copy()).to(cuda).view(nh, hd).double()
                got = torch.from_numpy(tr["layers"][l]["ctx"][first + i].copy()).to(cuda).view(nh, hd).double()
                for g in range(nkv):
                    k, v = (x.double() for x in lm.read_kv(l, s, g, 0, L))
                    qq = q[g * G:(g + 1) * G]
                    w = torch.softmax(qq @ k.t().contiguous() * hd ** -0.5, -1)
                    S = (qq.abs() @ k.abs().t().contiguous()).amax(-1, keepdim=True) * hd ** -0.5
                    # hd products and sums a score, exp of it and its rescalings, L weighted terms
                    rel = 2 * (hd + 3) * u * S + 2 * S * u + (8 + 4 * (L / 16 + 2) + 2 * L) * u
                    err = (got[g * G:(g + 1) * G] - w @ v).abs()
                    assert bool((err <= 2 * rel * (w @ v.abs())).all()), (s, i, l, g)
        first += counts[s]


def test_a_finished_batch_holds_no_pages(cuda):
    """A batch of three, then one stream that needs the pages of all: drive_batch gives back what
    its streams held."""
    cfg = T._fish_small(n_layers=1, max_batch=3)
    slow = D.SlowAr(cfg, device=cuda, kv_pages=6, page_size=16)
    slow.init_random(seed=6)
    fast = D.FastAr(D.fish_s2_fast_ar_config(n_layers=1, num_codebooks=10, residual_size=64, max_batch=3), device=cuda)
    fast.init_random(seed=7)
    rng = np.random.default_rng(8)
    prompts = [T._frames(rng, c, cfg).T for c in (12, 20, 5)]
    params = dualar.DriveParams(max_new_frames=6)
    first = dualar.drive_batch(slow, fast, prompts, stop_id=-1, params=params)
    assert slow.free_pages() == 6
    long = dualar.drive_batch(slow, fast, [T._frames(rng, 80, cfg).T], stop_id=-1, params=params)
    assert long[0].shape[1] == 6 and slow.free_pages() == 6
    again = dualar.drive_batch(slow, fast, prompts, stop_id=-1, params=params)
    assert all(torch.equal(x, y) for x, y in zip(first, again))
