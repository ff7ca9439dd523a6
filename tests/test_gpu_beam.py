"""The beam step against a plain 64-bit restatement: the selection over beams and vocabulary,
its state, the rings and the reordering of caches."""
import ctypes as C

import numpy as np
import pytest

import i8_beam_ref as ref
from vindexllm_b200 import abi

pytestmark = pytest.mark.gpu

# Scores: an fp32 store (2^-24 of the score) and the error of the log of the sum: the
# exponentials are off by 2^-22 and 2^-24 for each unit of distance to the maximum (weighted
# by themselves: below 1), a thread's fp32 sum of n terms by n 2^-24; n <= 64 here: 5e-6.
ATOL, RTOL = 5e-6, 2.0 ** -23


def _state(batch, beams, window, vocab, seed, fresh=False):
    rng = np.random.default_rng(seed)
    rows = batch * beams
    s = dict(scores=(-20 + 3 * rng.standard_normal(rows)).astype(np.float32),
             lengths=rng.integers(1, 30, rows).astype(np.int32),
             finished=(rng.random(rows) < 0.2).astype(np.int32))
    s["scores"][rng.random(rows) < 0.1] = -np.inf
    if window:
        s["hist"] = rng.integers(-2, vocab + 2, (rows, window)).astype(np.int32)
        s["count"] = rng.integers(0, window + 1, rows).astype(np.int32)
        s["pos"] = (s["count"] % window).astype(np.int32)
    return s


def _device(s, batch, beams, window):
    import torch
    from vindexllm_b200.sampler import BeamState
    t = {k: torch.as_tensor(v.copy(), device="cuda") for k, v in s.items()}
    return BeamState(batch, beams, window, **t)


def _check(got, want, batch, beams, exact=True):
    """got: (tokens, parents, BeamState); a pick may differ from the restatement's only where the
    two offers' ranks are nearer than the tolerance."""
    tokens, parents, state = got
    wt, wp, ws, ranks, offers = want
    t, p = tokens.cpu().numpy(), parents.cpu().numpy()
    same = (t == wt) & (p == wp)
    for g, k in zip(*np.nonzero(~same)):
        rank = offers[g].get((p[g, k], t[g, k]))
        assert rank is not None, f"prompt {g} slot {k}: ({p[g, k]}, {t[g, k]}) is no offer, want ({wp[g, k]}, {wt[g, k]})"
        near = 2 * (ATOL + RTOL * abs(rank))
        assert 0 < abs(rank - ranks[g, k]) <= near, f"prompt {g} slot {k}: rank {rank}, want {ranks[g, k]}"
    ok = same.reshape(-1)
    sc = state.scores.cpu().numpy()
    fin = np.isfinite(ws["scores"]) & ok
    assert np.array_equal(np.isfinite(sc), np.isfinite(ws["scores"]))
    assert (np.abs(sc[fin] - ws["scores"][fin]) <= ATOL + RTOL * np.abs(ws["scores"][fin])).all()
    names = {"lengths": state.lengths, "finished": state.finished}
    if state.window:
        names |= {"hist": state.hist, "pos": state.pos, "count": state.count}
    for name, v in names.items():
        assert np.array_equal(v.cpu().numpy()[ok], ws[name][ok]), name


def _bits(x, dtype):
    import torch
    t = torch.as_tensor(x, device="cuda")
    return t if dtype == "f32" else t.to(torch.bfloat16)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("vocab", [1, 2, 7, 33, 1000, 4096, 4097, 20011, 50257])
@pytest.mark.parametrize("batch,beams", [(1, 1), (3, 4), (2, 5), (1, 16), (1, 33), (1, 64)])
def test_step(gpu_ctx, dtype, vocab, batch, beams):
    """Odd vocabularies (rows off the 16-byte boundary), fewer tokens than beams, ties (values
    rounded to quarters), masks, finished and dead beams, all combinations of penalty and length."""
    from vindexllm_b200.sampler import BeamSearch
    rng = np.random.default_rng(vocab * 100 + beams)
    rows = batch * beams
    x = 3 * rng.standard_normal((rows, vocab)).astype(np.float32)
    x[rng.random(x.shape) < 0.05] = -np.inf
    x[::2] = np.round(x[::2] * 4) / 4
    lg = _bits(x, dtype)
    xf = lg.float().cpu().numpy()
    search = BeamSearch(gpu_ctx, batch, beams, vocab)
    for window, penalty, alpha in ((0, 1.0, 0.0), (20, 1.3, 0.6), (1, 0.8, 1.0)):
        s = _state(batch, beams, window, vocab, vocab + window)
        stop = np.unique(np.argmax(xf, 1))[:3].astype(np.int32)
        want = ref.beam_step(xf, batch, beams, s, stop, 9, penalty, alpha)
        state, out = _device(s, batch, beams, window), _device(s, batch, beams, window)
        import torch
        st = torch.as_tensor(stop, device="cuda")
        kw = dict(stop_ids=st, pad_token=9, repeat_penalty=penalty, length_alpha=alpha)
        got = search.step(state, lg, out=out, **kw)
        _check((*got, out), want, batch, beams)
        again = search.step(state, lg, **kw)  # in place: the same
        assert torch.equal(again[0], got[0]) and torch.equal(again[1], got[1])
        for name in ("scores", "lengths", "finished") + (("hist", "pos", "count") if window else ()):
            assert torch.equal(getattr(state, name), getattr(out, name)), name
    search.close()


@pytest.mark.parametrize("kind", ["rising", "falling", "constant", "two values", "one finite", "all masked", "lowest",
                                  "nan", "inf", "huge"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_rows_that_go_wrong(gpu_ctx, kind, dtype):
    """Orders in which every element enters the list, ties everywhere, masks that leave a row one
    token or none, the type's lowest value as a mask, NaN and infinities."""
    from vindexllm_b200.sampler import BeamSearch
    vocab = 30011
    ramp = np.arange(vocab, dtype=np.float32) * 1e-3
    for beams in (1, 4, 64):
        x = np.random.default_rng(beams).standard_normal((2 * beams, vocab)).astype(np.float32)
        row = {"rising": ramp, "falling": -ramp, "constant": np.full(vocab, 2.5, np.float32),
               "two values": (np.arange(vocab) % 2).astype(np.float32)}.get(kind, x[0].copy())
        if kind == "one finite":
            row[:] = -np.inf
            row[vocab - 2] = -700.0
        elif kind == "all masked":
            row[:] = -np.inf
        elif kind == "lowest":
            row[3:] = np.finfo(np.float32).min
        elif kind == "nan":
            row[vocab // 2] = np.nan
        elif kind == "inf":
            row[vocab - 1] = np.inf
        elif kind == "huge":
            row *= 1e30
        x[0] = row
        if beams > 1:
            x[beams] = row
        lg = _bits(x, dtype)
        xf = lg.float().cpu().numpy()
        s = _state(2, beams, 0, vocab, 5)
        s["scores"][:] = np.linspace(-1, -2, 2 * beams)
        s["finished"][:] = 0
        want = ref.beam_step(xf, 2, beams, s)
        search, out = BeamSearch(gpu_ctx, 2, beams, vocab), _device(s, 2, beams, 0)
        got = search.step(_device(s, 2, beams, 0), lg, out=out)
        _check((*got, out), want, 2, beams)
        search.close()


def test_strides_and_offsets(gpu_ctx):
    """A row stride beyond the vocabulary with NaN between the rows, a base at every element offset."""
    import torch
    from vindexllm_b200.sampler import BeamSearch
    batch, beams, vocab = 2, 3, 5000
    for dtype in (torch.float32, torch.bfloat16):
        wide = torch.full((batch * beams, vocab + 21), float("nan"), device="cuda", dtype=dtype)
        for off in range(9):
            wide.fill_(float("nan"))
            view = wide[:, off:off + vocab]
            view.copy_(torch.randn(view.shape, device="cuda", generator=torch.Generator("cuda").manual_seed(off)))
            s = _state(batch, beams, 0, vocab, off)
            want = ref.beam_step(view.float().cpu().numpy(), batch, beams, s)
            search, out = BeamSearch(gpu_ctx, batch, beams, vocab), _device(s, batch, beams, 0)
            got = search.step(_device(s, batch, beams, 0), view, out=out)
            _check((*got, out), want, batch, beams)
            search.close()


def test_offsets_beyond_32_bits(gpu_ctx):
    """Rows of logits and of a cache that lie more than 2^31 elements apart from first to last."""
    import torch
    from vindexllm_b200.sampler import BeamSearch
    vocab, beams = 5001, 9
    wide = torch.empty(beams, 1 << 28, dtype=torch.bfloat16, device="cuda")
    view = wide[:, 3:3 + vocab]
    view.copy_(torch.randn(view.shape, device="cuda", generator=torch.Generator("cuda").manual_seed(1)))
    cache = wide[:, 1 << 27:(1 << 27) + 777]
    cache.copy_(torch.randn(cache.shape, device="cuda", generator=torch.Generator("cuda").manual_seed(2)))
    before = cache.clone()
    s = _state(1, beams, 0, vocab, 3)
    s["scores"][:] = np.linspace(-2, -2.4, beams)
    want = ref.beam_step(view.float().cpu().numpy(), 1, beams, s)
    search, out = BeamSearch(gpu_ctx, 1, beams, vocab), _device(s, 1, beams, 0)
    got = search.step(_device(s, 1, beams, 0), view, out=out, caches=[cache])
    _check((*got, out), want, 1, beams)
    assert torch.equal(cache, before[got[1][0].long()])
    search.close()


def test_finished_rows_are_not_read(gpu_ctx):
    """Logits of finished and dead beams may hold anything."""
    import torch
    from vindexllm_b200.sampler import BeamSearch
    s = _state(1, 4, 0, 1000, 1)
    s["scores"][:] = [-3.0, -np.inf, -1.0, np.nan]
    s["finished"][:] = [0, 0, 1, 0]
    x = np.random.default_rng(0).standard_normal((4, 1000)).astype(np.float32)
    want = ref.beam_step(x, 1, 4, s)
    x[1:] = np.nan
    search, out = BeamSearch(gpu_ctx, 1, 4, 1000), _device(s, 1, 4, 0)
    got = search.step(_device(s, 1, 4, 0), torch.as_tensor(x, device="cuda"), out=out)
    _check((*got, out), want, 1, 4)


def test_full_vocabulary(gpu_ctx):
    """262144 tokens: many rows with long chunks, few rows with short ones. A thread sums at most
    512 terms: its fp32 sum is off by at most 512 * 2^-24 = 3e-5 of the sum."""
    import torch
    from vindexllm_b200.sampler import BeamSearch
    vocab = 262144
    for batch, beams, dtype in ((1, 4, torch.bfloat16), (40, 8, torch.float32)):
        rows = batch * beams
        x = torch.randn(rows, vocab, device="cuda", generator=torch.Generator("cuda").manual_seed(3)).mul_(3.0).to(dtype)
        s = _state(batch, beams, 0, vocab, 7)
        search, out = BeamSearch(gpu_ctx, batch, beams, vocab), _device(s, batch, beams, 0)
        tokens, parents = search.step(_device(s, batch, beams, 0), x, out=out, length_alpha=0.7)
        logp = torch.log_softmax(x.double(), 1)
        top = logp.topk(beams, 1).values.cpu().numpy()
        t, p, sc = tokens.cpu().numpy(), parents.cpu().numpy(), out.scores.cpu().numpy().reshape(batch, beams)
        for g in range(batch):
            r = slice(g * beams, (g + 1) * beams)
            done, score, length = s["finished"][r], s["scores"][r].astype(np.float64), s["lengths"][r]
            ranks = np.concatenate([[score[b] / length[b] ** 0.7] if done[b] else
                                    (score[b] + top[g * beams + b]) / (length[b] + 1) ** 0.7 for b in range(beams)])
            want = np.sort(ranks[ranks > -np.inf])[::-1][:beams]
            for k in range(len(want)):
                b = p[g, k]
                mine = score[b] if done[b] else score[b] + logp[g * beams + b, t[g, k]].item()
                assert abs(mine / (length[b] + (not done[b])) ** 0.7 - want[k]) <= 4e-5
                assert abs(sc[g, k] - mine) <= 4e-5 + RTOL * abs(mine)
        search.close()
        del logp


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("batch,beams,vocab", [(1, 2, 70000), (40, 4, 70000), (23, 7, 140000), (5, 40, 33000),
                                               (1, 3, 1000003), (111, 4, 4100)])
def test_chunk_shapes(gpu_ctx, dtype, batch, beams, vocab):
    """Chunks of one tile to the longest, odd numbers of tiles, a last chunk with a few elements or
    none. A thread sums at most 512 terms: ATOL + 512 * 2^-24 = 4e-5 of the sum."""
    import torch
    from vindexllm_b200.sampler import BeamSearch
    rows = batch * beams
    g = torch.Generator("cuda").manual_seed(vocab)
    x = (3 * torch.randn(rows, vocab, device="cuda", generator=g)).to(torch.float32 if dtype == "f32" else torch.bfloat16)
    s = _state(batch, beams, 0, vocab, 3)
    search, out = BeamSearch(gpu_ctx, batch, beams, vocab), _device(s, batch, beams, 0)
    tokens, parents = search.step(_device(s, batch, beams, 0), x, out=out)
    logp = torch.log_softmax(x.double(), 1)
    done, score = torch.as_tensor(s["finished"], device="cuda") != 0, torch.as_tensor(s["scores"], device="cuda").double()
    offers = torch.where(done[:, None], -torch.inf, score[:, None] + logp.topk(beams, 1).values)
    offers[:, 0] = torch.where(done, score, offers[:, 0])
    want = offers.view(batch, -1).sort(1, descending=True).values[:, :beams]
    src = (parents + beams * torch.arange(batch, device="cuda")[:, None]).long()
    mine = torch.where(done[src], score[src], score[src] + logp.view(-1)[src * vocab + tokens.clamp(min=0)])
    ok = want > -torch.inf
    assert ((mine - want).abs()[ok] <= 4e-5).all()
    assert ((out.scores.view(batch, beams).double() - mine).abs()[ok] <= 4e-5 + RTOL * mine.abs()[ok]).all()
    assert (out.scores.view(batch, beams)[~ok] == -torch.inf).all()
    flat = src * vocab + tokens  # no offer is taken twice
    assert all(len(set(f.tolist())) == beams for f, k in zip(flat, ok.all(1)) if k)
    search.close()


@pytest.mark.parametrize("vocab,window,held", [(300, 8192, 8192), (300, 8192, 7000), (20000, 2000, 2000), (5000, 700, 699),
                                               (9000, 257, 257)])
@pytest.mark.parametrize("kind", ["random", "top", "constant"])
def test_long_rings(gpu_ctx, vocab, window, held, kind):
    """Rings of up to 8192 tokens: most of a vocabulary, many times each; the rows' best tokens
    (more of them than a list takes at once); rows of equal logits, where every group is read
    again. The penalty is a power of two, so that repeating it is exact."""
    from vindexllm_b200.sampler import BeamSearch
    for beams in (1, 5, 64):
        rng = np.random.default_rng(vocab + beams)
        x = rng.standard_normal((beams, vocab)).astype(np.float32)
        if kind == "constant":
            x[:] = 1.5
        s = _state(1, beams, window, vocab, 7)
        s["finished"][:] = 0
        s["scores"][:] = np.linspace(-1, -3, beams)
        s["hist"] = rng.integers(0, vocab, (beams, window)).astype(np.int32)
        if kind == "top":
            best = np.argsort(-x, 1)[:, :min(window, vocab // 2)]
            s["hist"][:, :best.shape[1]] = best
        s["count"][:] = held
        s["pos"][:] = held % window
        want = ref.beam_step(x, 1, beams, s, (), 0, 0.5 if kind == "top" else 2.0, 0.0)
        search, out = BeamSearch(gpu_ctx, 1, beams, vocab), _device(s, 1, beams, window)
        import torch
        got = search.step(_device(s, 1, beams, window), torch.as_tensor(x, device="cuda"), out=out,
                          repeat_penalty=0.5 if kind == "top" else 2.0)
        _check((*got, out), want, 1, beams)
        search.close()


def test_the_same_bits_every_time(gpu_ctx):
    """Penalised tokens reach threads in the order of atomics: scores are the same bits all the same, and
    so are the offers next to one another."""
    import torch
    from vindexllm_b200.sampler import BeamSearch
    vocab, beams, window = 30000, 8, 600
    x = torch.randn(3 * beams, vocab, device="cuda", generator=torch.Generator("cuda").manual_seed(5))
    s = _state(3, beams, window, vocab, 11)
    s["hist"] = np.random.default_rng(1).integers(0, 700, s["hist"].shape).astype(np.int32)
    s["count"][:] = window
    search, first = BeamSearch(gpu_ctx, 3, beams, vocab), None
    for _ in range(20):
        out = _device(s, 3, beams, window)
        tokens, parents = search.step(_device(s, 3, beams, window), x, out=out, repeat_penalty=1.3, length_alpha=0.5)
        now = [tokens, parents, out.scores, out.hist]
        first = first or now
        assert all(torch.equal(a, b) for a, b in zip(now, first))
    search.close()


def test_penalised_values_that_go_wrong(gpu_ctx):
    """NaN, infinities and masks among the penalised tokens: as anywhere in the row."""
    import torch
    from vindexllm_b200.sampler import BeamSearch
    vocab, beams = 9000, 4
    for value in (np.nan, np.inf, -np.inf, np.finfo(np.float32).min, 3e38):
        x = np.random.default_rng(3).standard_normal((beams, vocab)).astype(np.float32)
        s = _state(1, beams, 6, vocab, 5)
        s["finished"][:] = 0
        s["scores"][:] = [-1, -1.5, -2, -2.5]
        s["hist"][:] = [5, 17, 5, 8999, -3, vocab]
        s["count"][:] = 6
        x[1, [5, 8999]] = value
        want = ref.beam_step(x, 1, beams, s, (), 0, 1.5, 0.0)
        search, out = BeamSearch(gpu_ctx, 1, beams, vocab), _device(s, 1, beams, 6)
        got = search.step(_device(s, 1, beams, 6), torch.as_tensor(x, device="cuda"), out=out, repeat_penalty=1.5)
        _check((*got, out), want, 1, beams)
        search.close()


@pytest.mark.parametrize("alpha", [0.0, 0.7, -1e6])
def test_scores_that_go_wrong(gpu_ctx, alpha):
    """Beams with a score of NaN or -infinity, finished or not, are never a parent, nor are those
    whose quotient is (alpha -1e6: a length above 1 divides by 0); slots without an offer keep
    their length."""
    import torch
    from vindexllm_b200.sampler import BeamSearch
    batch, beams, vocab = 4, 5, 700
    s = _state(batch, beams, 0, vocab, 21)
    sc, done = s["scores"].reshape(batch, beams), s["finished"].reshape(batch, beams)
    done[:] = [0, 1, 0, 1, 0]
    sc[:] = -3.0
    sc[0, :2] = np.nan
    sc[1, 2:] = -np.inf
    sc[2] = np.nan
    sc[3] = -np.inf
    search = BeamSearch(gpu_ctx, batch, beams, vocab)
    x = torch.as_tensor(np.random.default_rng(22).standard_normal((batch * beams, vocab)).astype(np.float32), device="cuda")
    tokens, parents = search.step(now := _device(s, batch, beams, 0), x, length_alpha=alpha, pad_token=9)
    t, p, out = tokens.cpu().numpy(), parents.cpu().numpy(), now.scores.reshape(batch, beams).cpu().numpy()
    length = s["lengths"].reshape(batch, beams)
    assert not np.isnan(out).any()
    for g in range(batch):
        fine = [b for b in range(beams) if sc[g, b] > -np.inf and (alpha > -1e6 or length[g, b] + 1 - done[g, b] < 2)]
        offers = sum(1 if done[g, b] else beams for b in fine)
        for k in range(beams):
            if k < offers:
                assert p[g, k] in fine and np.isfinite(out[g, k])
            else:
                assert p[g, k] == k and t[g, k] == 9 and out[g, k] == -np.inf
                assert now.finished.reshape(batch, beams)[g, k] == 0
                assert now.lengths.reshape(batch, beams)[g, k] == length[g, k]
    search.close()


@pytest.mark.parametrize("batch,beams,vocab", [(2, 12, 1000), (1, 4, 32000), (1, 30, 700), (3, 64, 300)])
@pytest.mark.parametrize("alpha", [-306.0, -305.5, 306.0])
def test_quotients_of_every_magnitude(gpu_ctx, batch, beams, vocab, alpha):
    """More than 96 offers whose quotients reach 2e307 or down to 1e-305: finite, so none is lost, and
    in their order. The scores stand far enough apart (checked here) that rounding cannot
    exchange two picks."""
    import torch
    from vindexllm_b200.sampler import BeamSearch
    rows = batch * beams
    rng = np.random.default_rng(beams)
    x = (2 * rng.standard_normal((rows, vocab))).astype(np.float32)
    s = dict(scores=rng.permutation(np.linspace(-16, -12, rows)).astype(np.float32),
             lengths=np.full(rows, 9, np.int32), finished=np.zeros(rows, np.int32))
    s["lengths"][1], s["finished"][1] = 10, 1
    want = ref.beam_step(x, batch, beams, s, (), 5, 1.0, alpha)
    for g in range(batch):
        best = np.sort(list(want[4][g].values()))[::-1][:beams + 1] * 10.0 ** alpha
        assert len(best) == beams + 1 and np.isfinite(best).all() and np.diff(-best).min() > 2 * (ATOL + 16 * RTOL)
    search, out = BeamSearch(gpu_ctx, batch, beams, vocab), _device(s, batch, beams, 0)
    tokens, parents = search.step(_device(s, batch, beams, 0), torch.as_tensor(x, device="cuda"), out=out, pad_token=5,
                                  length_alpha=alpha)
    assert np.array_equal(tokens.cpu().numpy(), want[0]) and np.array_equal(parents.cpu().numpy(), want[1])
    assert torch.isfinite(out.scores).all()
    search.close()


def test_quotients_next_to_zero(gpu_ctx):
    """Finished beams whose quotients are subnormal and negative: they stay, in their order."""
    import torch
    from vindexllm_b200.sampler import BeamSearch
    beams = 12
    order = np.random.default_rng(1).permutation(beams)
    s = dict(scores=(-1e-9 * (1 + order)).astype(np.float32), lengths=np.full(beams, 10, np.int32),
             finished=np.ones(beams, np.int32))
    search, out = BeamSearch(gpu_ctx, 1, beams, 500), _device(s, 1, beams, 0)
    tokens, parents = search.step(_device(s, 1, beams, 0), torch.zeros(beams, 500, device="cuda"), out=out, pad_token=5,
                                  length_alpha=306.0)
    assert (tokens == 5).all() and parents.cpu().numpy().tolist() == [np.argsort(order).tolist()]
    assert np.array_equal(out.scores.cpu().numpy(), np.sort(s["scores"])[::-1])
    search.close()

def test_many_stop_ids(gpu_ctx):
    import torch
    from vindexllm_b200.sampler import BeamSearch
    vocab, beams = 1000, 8
    x = np.random.default_rng(0).standard_normal((beams, vocab)).astype(np.float32)
    s = _state(1, beams, 0, vocab, 2)
    for n in (1, 64, 65, 400):
        stop = np.random.default_rng(n).permutation(vocab)[:n].astype(np.int32)
        want = ref.beam_step(x, 1, beams, s, set(stop.tolist()))
        search, out = BeamSearch(gpu_ctx, 1, beams, vocab), _device(s, 1, beams, 0)
        got = search.step(_device(s, 1, beams, 0), torch.as_tensor(x, device="cuda"), out=out,
                          stop_ids=torch.as_tensor(stop, device="cuda"))
        _check((*got, out), want, 1, beams)
        search.close()


def test_search_of_many_steps(gpu_ctx):
    """A whole search from its start (beam 0 alone is alive), in place, with rings, a token list as
    a cache, and a stop token: the tokens follow the parents, step by step."""
    import torch
    from vindexllm_b200.sampler import BeamSearch, BeamState
    batch, beams, vocab, window, steps = 3, 4, 501, 6, 12
    rng = np.random.default_rng(11)
    search = BeamSearch(gpu_ctx, batch, beams, vocab)
    state = BeamState(batch, beams, window)
    lists = torch.zeros(batch * beams, steps, dtype=torch.int32, device="cuda")
    host = dict(scores=state.scores.cpu().numpy(), lengths=np.zeros(batch * beams, np.int32),
                finished=np.zeros(batch * beams, np.int32), hist=np.zeros((batch * beams, window), np.int32),
                pos=np.zeros(batch * beams, np.int32), count=np.zeros(batch * beams, np.int32))
    hl = np.zeros((batch * beams, steps), np.int32)
    stop = torch.tensor([3, 77], dtype=torch.int32, device="cuda")
    for i in range(steps):
        x = 2 * rng.standard_normal((batch * beams, vocab)).astype(np.float32)
        x[:, 77] += 6
        want = ref.beam_step(x, batch, beams, host, (3, 77), 0, 1.4, 0.8)
        tokens, parents = search.step(state, torch.as_tensor(x, device="cuda"), stop_ids=stop, repeat_penalty=1.4,
                                      length_alpha=0.8, caches=[lists[:, :i]] if i else [])
        lists[:, i] = tokens.view(-1)
        _check((tokens, parents, state), want, batch, beams)
        assert np.array_equal(tokens.cpu().numpy(), want[0]) and np.array_equal(parents.cpu().numpy(), want[1])
        src = (want[1] + beams * np.arange(batch)[:, None]).reshape(-1)
        hl[:, :i] = hl[src, :i]
        hl[:, i] = want[0].reshape(-1)
        host = want[2]
        host["scores"] = state.scores.cpu().numpy()  # one step's rounding at a time
    assert np.array_equal(lists.cpu().numpy(), hl)
    assert state.finished.any()


PARENTS = [[0, 1, 2, 3], [3, 2, 1, 0], [0, 0, 0, 0], [1, 2, 3, 3], [-1, 4, 2, 1 << 30]]


@pytest.mark.parametrize("dtype,width", [("uint8", 1), ("uint8", 7), ("int16", 9), ("int32", 5), ("int64", 3),
                                         ("float16", 8), ("float32", 64), ("float32", 1000)])
def test_reorder(gpu_ctx, dtype, width):
    """Words of every size, in place and to another buffer, the filled part of a cache, more
    caches than one launch takes, parents out of range (their rows stay)."""
    import torch
    from vindexllm_b200.sampler import BeamSearch
    batch, beams = len(PARENTS), 4
    parents = torch.tensor(PARENTS, dtype=torch.int32, device="cuda")
    src = np.array([[b if 0 <= b < beams else k for k, b in enumerate(p)] for p in PARENTS])
    rows = torch.as_tensor((src + beams * np.arange(batch)[:, None]).reshape(-1), device="cuda")
    search = BeamSearch(gpu_ctx, batch, beams, 10)
    dt = getattr(torch, dtype)
    make = lambda i: torch.randint(0, 100, (batch * beams, 3, 11, width), device="cuda",  # noqa: E731
                                   generator=torch.Generator("cuda").manual_seed(i)).to(dt)
    a = [make(i) for i in range(40)]
    want, b = [t.clone() for t in a], [make(100 + i) for i in range(40)]
    left = [t.clone() for t in b]
    used = [(i % 11) + 1 for i in range(40)]
    search.reorder(parents, [(x[:, :, :u], y[:, :, :u]) for x, y, u in zip(a, b, used)])
    for x, y, l, w, u in zip(a, b, left, want, used):
        assert torch.equal(x, w)
        assert torch.equal(y[:, :, :u], w[rows, :, :u]) and torch.equal(y[:, :, u:], l[:, :, u:])
    search.reorder(parents, [x[:, 1:, u - 1:u] for x, u in zip(a, used)])
    for x, w, u in zip(a, want, used):
        w2 = w.clone()
        w2[:, 1:, u - 1:u] = w[rows, 1:, u - 1:u]
        assert torch.equal(x, w2)
    # Pieces of different shapes, rows inside the segments' gaps, empty views.
    e, f = make(7), torch.zeros(3, batch * beams, 11, width, dtype=dt, device="cuda").transpose(0, 1)
    search.reorder(parents, [(e, f), e[:, :0]])
    assert torch.equal(f, e[rows])
    search.reorder(parents, [f])
    assert torch.equal(f, e[rows][rows])
    search.close()


def test_a_cache_listed_twice_is_refused(gpu_ctx):
    """A cache that two layers share is listed once: twice, or as a source beside its being a target, is
    refused and moves nothing. Caches whose bytes lie between one another's are moved."""
    import torch
    from vindexllm_b200.sampler import BeamSearch, VdxsError
    batch, beams = 2, 3
    rows = batch * beams
    parents = torch.tensor([[2, 0, 1], [1, 1, 0]], dtype=torch.int32, device="cuda")
    src = (parents + beams * torch.arange(batch, device="cuda")[:, None]).view(-1).long()
    search = BeamSearch(gpu_ctx, batch, beams, 10)
    a, b = (torch.randn(rows, 4, 16, device="cuda") for _ in range(2))
    keep = [a.clone(), b.clone()]
    for caches in ([a, a], [a, b, a.view(rows, 64)], [(a, b), b], [(a, b), (b, a)], [a] + [torch.zeros_like(b) for _ in
                                                                                      range(40)] + [a[:, :2]]):
        with pytest.raises(VdxsError, match="another cache"):
            search.reorder(parents, caches)
    torch.cuda.synchronize()
    assert torch.equal(a, keep[0]) and torch.equal(b, keep[1])
    both = torch.randn(rows, 2, 4, 16, device="cuda")
    want = both[src]
    search.reorder(parents, [both[:, 0], both[:, 1], b[:, :0], b[:, :0]])
    assert torch.equal(both, want)
    search.reorder(parents, [(a, both[:, 0]), (a, both[:, 1])])  # one source, two targets
    assert torch.equal(both[:, 0], a[src]) and torch.equal(both[:, 1], a[src])
    search.close()

@pytest.mark.parametrize("beams", [1, 2, 9, 17, 64])
def test_reorder_other_beam_counts(gpu_ctx, beams):
    import torch
    from vindexllm_b200.sampler import BeamSearch
    batch = 3
    g = torch.Generator("cuda").manual_seed(beams)
    parents = torch.randint(0, beams, (batch, beams), device="cuda", generator=g).int()
    rows = (parents + beams * torch.arange(batch, device="cuda")[:, None]).view(-1).long()
    x = torch.randn(batch * beams, 2, 300, 8, device="cuda", generator=g)
    want = x[rows]
    search = BeamSearch(gpu_ctx, batch, beams, 10)
    search.reorder(parents, [x])
    assert torch.equal(x, want)
    search.close()


def test_graph_and_side_stream(gpu_ctx):
    """Captured without a warm-up call and replayed: each replay advances the state as an eager step
    of another search does."""
    import torch
    from vindexllm_b200.sampler import BeamSearch, BeamState
    batch, beams, vocab = 2, 4, 3000
    one, two = BeamSearch(gpu_ctx, batch, beams, vocab), BeamSearch(gpu_ctx, batch, beams, vocab)
    x = torch.randn(batch * beams, vocab, device="cuda")
    s1, s2 = BeamState(batch, beams, 4), BeamState(batch, beams, 4)
    c1 = torch.arange(batch * beams * 20, device="cuda").view(batch * beams, 20)
    c2 = c1.clone()
    t1 = torch.empty(batch, beams, dtype=torch.int32, device="cuda")
    p1 = torch.empty_like(t1)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        one.step(s1, x, repeat_penalty=1.2, caches=[c1], tokens=t1, parents=p1)
    side = torch.cuda.Stream()
    for i in range(4):
        x.normal_()
        side.wait_stream(torch.cuda.current_stream())
        t2, p2 = two.step(s2, x, repeat_penalty=1.2, caches=[c2], stream=side)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(t1, t2) and torch.equal(p1, p2) and torch.equal(c1, c2)
        assert torch.equal(s1.scores, s2.scores) and torch.equal(s1.hist, s2.hist) and torch.equal(s1.count, s2.count)


def test_two_host_threads(gpu_ctx):
    """A context for each host thread: searches of different rings, beams and chunks step at once, each as it
    does alone."""
    import threading

    import torch
    from vindexllm_b200.sampler import BeamSearch, SamplerContext
    shapes = [(1, 30, 9000, 700), (1, 64, 3000, 8192), (2, 5, 140000, 100), (1, 40, 70000, 3000)]

    def steps(ctx, batch, beams, vocab, window, stream):
        with torch.cuda.stream(stream):
            g = torch.Generator("cuda").manual_seed(vocab)
            x = torch.randn(batch * beams, vocab, device="cuda", generator=g)
            search, out = BeamSearch(ctx, batch, beams, vocab), _device(_state(batch, beams, window, vocab, 9), batch, beams,
                                                                        window)
            cache = torch.arange(batch * beams * 64, device="cuda").view(batch * beams, 64)
            got = []
            for _ in range(5):
                t, p = search.step(out, x, repeat_penalty=1.2, caches=[cache])
                got += [t, p, out.scores.clone(), out.hist.clone(), cache.clone()]
        torch.cuda.synchronize()
        search.close()
        return got

    results, failures = [None] * len(shapes), []
    gate = threading.Barrier(len(shapes))

    def work(i):
        try:
            ctx, stream = SamplerContext(0), torch.cuda.Stream()
            gate.wait(60)
            results[i] = steps(ctx, *shapes[i], stream)
            ctx.close()
        except BaseException as e:  # noqa: BLE001
            failures.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(shapes))]
    for t in threads:
        t.start()
    for t in threads:
        t.join(120)
    assert not failures, failures
    for got, shape in zip(results, shapes):
        want = steps(gpu_ctx, *shape, torch.cuda.Stream())
        assert all(torch.equal(a, b) for a, b in zip(got, want))

def test_norm_product_beam_run(gpu_ctx):
    """The tail of a decode step as a search runs it: norm, product and beam step, the step held to the
    restatement on the logits that the product gave."""
    import torch
    from vindexllm_b200.sampler import BeamSearch, BeamState, I8Weights
    batch, beams, vocab, k = 2, 5, 4099, 320
    gen = torch.Generator("cuda").manual_seed(4)
    w = I8Weights(gpu_ctx, 0.1 * torch.randn(vocab, k, device="cuda", generator=gen))
    nw = torch.ones(k, device="cuda")
    search, state = BeamSearch(gpu_ctx, batch, beams, vocab), BeamState(batch, beams, 8)
    hidden = torch.randn(batch * beams, k, device="cuda", generator=gen).bfloat16()
    for i in range(4):
        x = torch.randn(batch * beams, k, device="cuda", generator=gen).bfloat16()
        host = {n: getattr(state, n).cpu().numpy().copy() for n in ("scores", "lengths", "finished", "hist", "pos", "count")}
        q, scale, _ = gpu_ctx.rms_norm_i8(x, nw, residual=hidden, out_hidden=hidden)
        logits = w.unembed(q, scale, dtype=torch.bfloat16 if i % 2 else torch.float32)
        before = hidden.clone()
        tokens, parents = search.step(state, logits, repeat_penalty=1.1, caches=[hidden])
        want = ref.beam_step(logits.float().cpu().numpy(), batch, beams, host, (), 0, 1.1, 0.0)
        _check((tokens, parents, state), want, batch, beams)
        src = (parents + beams * torch.arange(batch, device="cuda")[:, None]).view(-1).long()
        assert torch.equal(hidden, before[src])
    w.close()
    search.close()


def test_refusals(gpu_ctx):
    import torch
    from vindexllm_b200.sampler import BeamSearch, BeamState
    lib = gpu_ctx.lib
    out = C.c_void_p()
    for b, k, v, code in ((0, 4, 10, abi.E_INVALID_ARG), (1, 0, 10, abi.E_INVALID_ARG), (1, 4, 0, abi.E_INVALID_ARG),
                          (1, 65, 10, abi.E_UNSUPPORTED), (2000, 64, 10, abi.E_UNSUPPORTED),
                          (1, 4, 1 << 25, abi.E_UNSUPPORTED)):
        assert lib.vdxs_beam_create(gpu_ctx.handle, b, k, v, C.byref(out)) == code and not out.value
    search, state = BeamSearch(gpu_ctx, 2, 3, 100), BeamState(2, 3, 4)
    x = torch.zeros(6, 100, device="cuda")
    tok = torch.zeros(2, 3, dtype=torch.int32, device="cuda")
    p = lambda t: C.c_void_p(t.data_ptr())  # noqa: E731

    def step(cfg=(0.0, 1.0, 4, 0, 0), xp=p(x), dt=0, stride=100, drop=None, stop=None, n_stop=0, cache=None, n=0,
             tp=p(tok), rows=state):
        a = rows.rows()
        if drop:
            setattr(a, drop, None)
        c = abi.VdxsBeamConfig(*cfg)
        return lib.vdxs_beam_step(search._h, C.byref(c), xp, dt, stride, C.byref(a), C.byref(a), stop, n_stop, cache, n,
                                  tp, p(tok), None)

    assert step() == abi.OK
    nan = float("nan")
    for bad in (dict(xp=None), dict(dt=2), dict(stride=99), dict(tp=None), dict(drop="scores"), dict(drop="finished"),
                dict(drop="hist"), dict(drop="hist_count"), dict(n_stop=1), dict(n_stop=-1), dict(n=1), dict(n=-1),
                dict(cfg=(nan, 1.0, 4, 0, 0)), dict(cfg=(0.0, 0.0, 4, 0, 0)), dict(cfg=(0.0, nan, 4, 0, 0)),
                dict(cfg=(0.0, 1.0, -1, 0, 0)), dict(cfg=(0.0, 1.0, 9000, 0, 0)), dict(cfg=(0.0, 1.0, 4, 0, 1)),
                dict(xp=C.c_void_p(x.data_ptr() + 2))):
        assert step(**bad) == abi.E_INVALID_ARG, bad
    buf = torch.zeros(6, 64, dtype=torch.uint8, device="cuda")
    at = buf.data_ptr()
    for c in ((at, at, 64, 0, 32, 0, 16, 1),      # in place with other strides
              (at, at + 8, 64, 0, 64, 0, 16, 1),  # overlap
              (at, at, 8, 0, 8, 0, 16, 1),        # rows overlap
              (at, at, 64, 8, 64, 8, 16, 2),      # segments overlap
              (at, at, -64, 0, -64, 0, 16, 1), (0, at, 64, 0, 64, 0, 16, 1), (at, at, 64, 0, 64, 0, -1, 1)):
        one = (abi.VdxsBeamCache * 1)(abi.VdxsBeamCache(*c))
        assert step(cache=one, n=1) == abi.E_INVALID_ARG, c
        assert lib.vdxs_beam_reorder(search._h, p(tok), one, 1, None) == abi.E_INVALID_ARG, c
    with pytest.raises(ValueError):
        search.step(state, x[:5])
    with pytest.raises(ValueError):
        search.step(BeamState(2, 4, 4), x)
    with pytest.raises(ValueError):
        search.step(state, x, out=BeamState(2, 3, 5))
    with pytest.raises(ValueError):
        search.reorder(tok, [torch.zeros(5, 3, device="cuda")])
    with pytest.raises(TypeError):
        search.step(state, x.half())
    search.close()


def test_unaligned_pointers_are_refused(gpu_ctx):
    from vindexllm_b200.sampler import BeamSearch, BeamState
    import torch
    lib, search, state = gpu_ctx.lib, BeamSearch(gpu_ctx, 2, 3, 100), BeamState(2, 3, 4)
    x, tok = torch.zeros(6, 100, device="cuda"), torch.zeros(2, 3, dtype=torch.int32, device="cuda")
    before = [getattr(state, n).clone() for n in ("scores", "lengths", "finished", "hist", "pos", "count")]

    def step(off=None, side=0, tp=0, pp=0, stop=None):
        rows = [state.rows(), state.rows()]
        if off:
            setattr(rows[side], off, getattr(rows[side], off) + 2)
        cfg = abi.VdxsBeamConfig(0.0, 1.0, 4, 0, 0)
        return lib.vdxs_beam_step(search._h, C.byref(cfg), x.data_ptr(), 0, 100, C.byref(rows[0]), C.byref(rows[1]), stop,
                                  1 if stop else 0, None, 0, tok.data_ptr() + tp, tok.data_ptr() + pp, None)

    for name, _ in abi.VdxsBeamRows._fields_:
        for side in (0, 1):
            assert step(name, side) == abi.E_INVALID_ARG, (name, side)
    assert step(tp=1) == step(pp=2) == step(stop=tok.data_ptr() + 2) == abi.E_INVALID_ARG
    assert lib.vdxs_beam_reorder(search._h, tok.data_ptr() + 2, None, 0, None) == abi.E_INVALID_ARG
    assert b"aligned" in lib.vdxs_last_error(gpu_ctx.handle)
    torch.cuda.synchronize()
    assert all(torch.equal(a, getattr(state, n)) for a, n in
               zip(before, ("scores", "lengths", "finished", "hist", "pos", "count")))
    assert step() == abi.OK
    search.close()
